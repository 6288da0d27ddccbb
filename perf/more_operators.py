"""Differential attention, norms on both sides of a sublayer with its gate and residual
scale, and orthogonalised updates of weight matrices: the timed workloads, their plain
form and their values in 64 bits.

Each case is a dict of plain values.  ``prepare`` makes what a user's program holds
before the call, ``run`` is one pass: the operators' formulas in elementary torch
operations where ``own`` is false, this package's calls where it is true.  ``exact``
gives the same outputs from the definitions in float64.

Kinds:
  diff_fwd    differential attention without gradients, (b, l, H, 64) tensors: the heads
              2p and 2p + 1 are the two maps of pair p, the value heads 2p and 2p + 1
              side by side its 128 value channels;
              o = (softmax(q1 k1^T / 8) - lam softmax(q2 k2^T / 8)) v
  diff_train  the same with the gradients of q, k, v and lam
  norm_fwd    y = x + scale * gate * w_post * a / rms(a), n = w_pre * y / rms(y)
  norm_train  the same with the gradients of everything
  ortho       Newton-Schulz products: X = G / |G|, five times
              X <- a X + (b A + c A^2) X with A = X X^T
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
D = 64
EPS = 1e-6
STEPS, COEFFS = 5, (3.4445, -4.7750, 2.0315)
CHUNK = 1 << 30  # scores of one map in one chunk of the plain form (4 GiB in fp32)


def listed():
    return [
        # A block of the unit tests' geometry (4 video tiles and an 18-token prefix)
        # without gradients: launches and host work decide.
        dict(name="diff_fwd_274", kind="diff_fwd", dtype="bf16", B=1, H=4, Hkv=4, Lq=274, Lk=274,
             causal=False, ragged=False),
        # One new token against a whole clip's keys, two clips, the second shorter.
        dict(name="diff_fwd_1q", kind="diff_fwd", dtype="bf16", B=2, H=8, Hkv=8, Lq=1, Lk=29952,
             causal=True, ragged=True),
        # The attention sublayer of the sampler at full video length (12 x 48 x 52).
        dict(name="diff_fwd_30k", kind="diff_fwd", dtype="bf16", B=1, H=8, Hkv=8, Lq=29952,
             Lk=29952, causal=False, ragged=False),
        # A training step of the unit tests' geometry, one clip of a padded batch empty.
        dict(name="diff_train_274", kind="diff_train", dtype="fp16", B=2, H=4, Hkv=4, Lq=274,
             Lk=274, causal=False, ragged=True),
        # A padded batch of three clips in causal order with grouped key heads.
        dict(name="diff_train_4159", kind="diff_train", dtype="fp16", B=3, H=8, Hkv=4, Lq=4159,
             Lk=4159, causal=True, ragged=True),
        # A training step of the sublayer at full video length.
        dict(name="diff_train_30k", kind="diff_train", dtype="bf16", B=1, H=8, Hkv=8, Lq=29952,
             Lk=29952, causal=False, ragged=False),
        # One token of the 512-wide block on its way between two sublayers.
        dict(name="norm_fwd_1", kind="norm_fwd", dtype="bf16", B=1, L=1, D=512, gate=False,
             pre=True, consumers=2),
        # A training step of a short padded batch of two clips with gates of their own.
        dict(name="norm_train_521", kind="norm_train", dtype="fp16", B=2, L=521, D=512, gate=True,
             pre=True, consumers=3),
        # The training benchmark's block: two clips of 29,952 tokens, between its sublayers.
        dict(name="norm_train_60k", kind="norm_train", dtype="bf16", B=2, L=29952, D=512,
             gate=False, pre=True, consumers=2),
        # The key/value down projection's gradient alone.
        dict(name="ortho_160x512", kind="ortho", dtype="fp32", n=1, R=160, C=512),
        # The output projections of eight blocks, gradients in 16 bits.
        dict(name="ortho_8x512", kind="ortho", dtype="bf16", n=8, R=512, C=512),
        # The MLPs of eight blocks of the training benchmark (ratio 4).
        dict(name="ortho_24x2048", kind="ortho", dtype="fp32", n=24, R=2048, C=512),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for key in ("bytes", "flops"):
            most[c["kind"], key] = max(most.get((c["kind"], key), 0), w[key])
    # one token is the listed call without gradients; longer ones go with the training cases
    for key in ("bytes", "flops"):
        most["norm_fwd", key] = most["norm_train", key]
    while True:
        kind = rng.choice(["diff_fwd", "diff_fwd", "diff_train", "diff_train", "norm_fwd",
                           "norm_train", "ortho", "ortho"])
        c = dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]))
        if kind.startswith("diff"):
            Hkv = rng.choice([2, 4, 6, 8])
            Lq = _logint(rng, 1, 29952)
            Lk = rng.choice([Lq, _logint(rng, 1, 29952)])
            c.update(B=rng.choice([1, 1, 2, 3]), H=Hkv * rng.choice([1, 1, 2, 4]), Hkv=Hkv, Lq=Lq,
                     Lk=Lk, causal=rng.random() < 0.4, ragged=rng.random() < 0.4)
        elif kind.startswith("norm"):
            c.update(B=rng.choice([1, 2, 3]), L=_logint(rng, 1, 29952), D=_logint(rng, 32, 2048),
                     gate=rng.random() < 0.5, pre=rng.random() < 0.8, consumers=rng.choice([1, 2, 3]))
        else:
            c.update(dtype=rng.choice(["bf16", "fp32"]), n=_logint(rng, 1, 24),
                     R=_logint(rng, 16, 2048), C=_logint(rng, 16, 2048))
        w = work(c)
        if all(w[key] <= most[kind, key] for key in w):
            return c


# ---------------------------------------------------------------------------
# Sizes of a case
# ---------------------------------------------------------------------------
def lengths(c):
    """(query lengths, key lengths) of the clips of a batch.  A ragged batch holds
    a full clip first and shorter ones after it; the last of two is empty in
    training, in inference its keys are five eighths of the others'."""
    B, Lq, Lk = c["B"], c["Lq"], c["Lk"]
    if not c["ragged"]:
        return [Lq] * B, [Lk] * B
    if c["kind"] == "diff_fwd":
        return [Lq] * B, [Lk - (3 * Lk * b) // (8 * max(1, B - 1)) for b in range(B)]
    part = [1.0 - b / max(1, B - 1) * (1.0 if B == 2 else 0.7) for b in range(B)]
    return [int(Lq * p) for p in part], [int(Lk * p) for p in part]


def _pairs(c):
    """(query, key) pairs that attend, over the batch, for one head."""
    n = 0
    for lq, lk in zip(*lengths(c)):
        if not c["causal"]:
            n += lq * lk
        else:  # query i sees the keys up to i + lk - lq
            rows = min(lq, lk)
            n += rows * lk - rows * (rows - 1) // 2
    return n


def work(c):
    """Bytes: inputs read once and outputs written once.  flops: two per multiply-add.
    Attention: the two score products and the combined map's product with the values, 128
    multiply-adds each; the backward's five (scores again, dA, dv, dq, dk).  Norms: about
    10 per element and norm each way.  Newton-Schulz products on the shorter side r: A and
    its square, symmetric, at half their products."""
    if c["kind"].startswith("diff"):
        ql, kl = lengths(c)
        q = sum(ql) * c["H"] * D * 2
        kv = sum(kl) * c["Hkv"] * D * 2
        out = c["B"] * c["Lq"] * c["H"] * D * 2
        gemm = 2 * _pairs(c) * (c["H"] // 2) * 2 * D
        if c["kind"] == "diff_fwd":
            return dict(bytes=q + 2 * kv + out, flops=2 * gemm)
        dkv = c["B"] * c["Lk"] * c["Hkv"] * D * 2
        # q, k, v, do in; o, dq, dk, dv out
        return dict(bytes=2 * q + 2 * kv + 2 * out + 2 * dkv, flops=7 * gemm)
    if c["kind"].startswith("norm"):
        n = c["B"] * c["L"] * c["D"]
        norms = 2 if c["pre"] else 1
        fwd = n * (4 + 2 + 4 + (2 if c["pre"] else 0))  # x, a in; y, n out
        if c["kind"] == "norm_fwd":
            return dict(bytes=fwd, flops=10 * norms * n)
        # y's and n's gradients in; those of x and a out
        bwd = n * (4 + (2 * c["consumers"] if c["pre"] else 0) + 4 + 2)
        return dict(bytes=fwd + bwd, flops=30 * norms * n)
    r, m, n = min(c["R"], c["C"]), max(c["R"], c["C"]), c["n"]
    size = DTYPES[c["dtype"]].itemsize
    return dict(bytes=2 * n * r * m * size, flops=STEPS * n * (3 * r * r * m + r * r * r))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _inputs(c, seed):
    """What both forms and the exact values start from."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    if c["kind"].startswith("diff"):
        B, H, Hkv, Lq, Lk = (c[x] for x in ("B", "H", "Hkv", "Lq", "Lk"))
        # q and k come normalised per head, with a gain on q that sharpens the scores
        # to a standard deviation of two; v is a band of the kv projection, its channels
        # with means of their own
        q = rn(B, Lq, H, D)
        q = (2.0 * q * torch.rsqrt(q.pow(2).mean(-1, keepdim=True) + EPS)).to(dt)
        k = rn(B, Lk, Hkv, D)
        k = (k * torch.rsqrt(k.pow(2).mean(-1, keepdim=True) + EPS)).to(dt)
        v = rn(B, Lk, Hkv, D + 32) + 0.5 * rn(Hkv, D + 32)
        x = dict(q=q, k=k, v=v.to(dt)[..., 32:], ql=None, kl=None)
        # the weight of the second map, a little apart from 0.8 - 0.6 exp(-0.3 layer)
        x["lam"] = (0.5 + 0.1 * rn(H // 2)).to(dt)
        if c["kind"] == "diff_train":
            x["do"] = (0.05 * rn(B, Lq, H, D) + 0.03 * rn(H, D)).to(dt)
        if c["ragged"]:
            ql, kl = lengths(c)
            if c["kind"] == "diff_train":
                x["ql"] = torch.tensor(ql, device=DEV, dtype=torch.int32)
            x["kl"] = torch.tensor(kl, device=DEV, dtype=torch.int32)
        return x
    if c["kind"].startswith("norm"):
        B, L, W = c["B"], c["L"], c["D"]
        # a residual stream a few layers deep with loud channels, a sublayer's output,
        # gains near one and scales that have left zero
        loud = 1.0 + 4.0 * (torch.rand(W, device=DEV, generator=g) < 0.02)
        x = dict(x=2.0 * rn(B, L, W) * loud, a=(0.7 * rn(B, L, W)).to(dt),
                 scale=0.3 + 0.1 * rn(W), post=1.0 + 0.1 * rn(W), pre=None, gate=None)
        if c["gate"]:
            x["gate"] = 1.0 + 0.2 * rn(B, W)
        if c["pre"]:
            x["pre"] = 1.0 + 0.1 * rn(W)
        if c["kind"] == "norm_train":
            x["dy"] = 0.02 * rn(B, L, W)
            x["dn"] = ([(0.02 * rn(B, L, W)).to(dt) for _ in range(c["consumers"])]
                       if c["pre"] else [])
        return x
    # momentum of gradients: noise over a decaying spectrum of common directions
    n, R, C = c["n"], c["R"], c["C"]
    k = max(1, min(R, C) // 8)
    decay = torch.exp(-4.0 * torch.arange(k, device=DEV) / k)
    G = 0.3 * rn(n, R, C) + torch.matmul(rn(n, R, k) * decay, rn(n, k, C))
    return dict(G=(1e-3 * G).to(dt))


def prepare(c, seed):
    x = _inputs(c, seed)
    st = dict(case=c, **x)
    if own:
        grads = dict(diff_train=("q", "k", "v", "lam"),
                     norm_train=("x", "a", "scale", "post", "pre", "gate")).get(c["kind"], ())
        for n in grads:
            if x[n] is not None:
                st[n] = x[n].detach().requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    c = st["case"]
    if c["kind"].startswith("diff"):
        from imfvideo_amd.imf_dit_video import diff_attention
        q, k, v, lam = st["q"], st["k"], st["v"], st["lam"]
        args = dict(causal=c["causal"], q_lens=st["ql"], k_lens=st["kl"])
        if c["kind"] == "diff_fwd":
            with torch.no_grad():
                return dict(o=diff_attention(q, k, v, lam, **args))
        o = diff_attention(q, k, v, lam, **args)
        dq, dk, dv, dlam = torch.autograd.grad(o, (q, k, v, lam), st["do"])
        return dict(o=o.detach(), dq=dq, dk=dk, dv=dv, dlam=dlam)
    if c["kind"].startswith("norm"):
        from imfvideo_amd.imf_dit_video import residual_norm
        args = dict(gate=st["gate"], pre_weight=st["pre"], eps=EPS, consumers=c["consumers"])
        if c["kind"] == "norm_fwd":
            with torch.no_grad():
                y, *n = residual_norm(st["x"], st["a"], st["scale"], st["post"], **args)
            return dict(y=y, n=n[0]) if n else dict(y=y)
        y, *n = residual_norm(st["x"], st["a"], st["scale"], st["post"], **args)
        leaves = {"d" + k: st[k] for k in ("x", "a", "scale", "post", "pre", "gate")
                  if st[k] is not None}
        grads = torch.autograd.grad([y, *n], list(leaves.values()), [st["dy"], *st["dn"]])
        out = dict(zip(leaves, grads), y=y.detach())
        return dict(out, n=n[0].detach()) if n else out
    from imfvideo_amd import ops
    return dict(X=ops.orthogonalize(st["G"], steps=STEPS, coeffs=COEFFS))


def _softmax(s, off):
    """Softmax of the last dimension in place; what `off` marks is 0, and so is a row
    with nothing left."""
    if off is None:
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        return s.div_(s.sum(-1, keepdim=True))
    s.masked_fill_(off, float("-inf"))
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == float("-inf"), torch.zeros_like(m), m)).exp_()
    z = s.sum(-1, keepdim=True)
    return s.mul_(torch.where(z > 0, 1.0 / z, torch.zeros_like(z)))


def _diff_plain(q, k, v, lam, ql, kl, causal, do=None):
    """Differential attention of (b, l, H, 64) tensors in fp32, the pairs of key heads of
    all clips beside each other, as many at a time as CHUNK has room for; with do also the
    gradients."""
    B, Lq, H, _ = q.shape
    Lk, P = k.shape[1], k.shape[2] // 2
    rep, scale, dev = H // k.shape[2], D ** -0.5, q.device
    off = None
    if ql is not None or kl is not None or causal:
        ql = torch.full((B,), Lq, device=dev) if ql is None else ql.long()
        kl = torch.full((B,), Lk, device=dev) if kl is None else kl.long()
        iq, ik = torch.arange(Lq, device=dev)[:, None], torch.arange(Lk, device=dev)[None, :]
        off = (iq >= ql[:, None, None]) | (ik >= kl[:, None, None])
        if causal:
            off = off | (ik > iq + (kl - ql)[:, None, None])
        off = off.repeat_interleave(P, 0)[:, None]  # (B P, 1, Lq, Lk)
    # (B P, rows, channels): a key pair's query pairs one after the other
    qm = q.float().reshape(B, Lq, P, rep, 2, D).permute(4, 0, 2, 3, 1, 5).reshape(2, B * P, rep * Lq, D)
    km = k.float().reshape(B, Lk, P, 2, D).permute(3, 0, 2, 1, 4).reshape(2, B * P, Lk, D)
    vm = v.float().reshape(B, Lk, P, 2 * D).permute(0, 2, 1, 3).reshape(B * P, Lk, 2 * D)
    lm = lam.float().reshape(P, rep).repeat(B, 1)[:, :, None, None]  # (B P, rep, 1, 1)
    o = torch.empty(B * P, rep * Lq, 2 * D, device=dev)
    if do is not None:
        dom = do.float().reshape(B, Lq, P, rep, 2 * D).permute(0, 2, 3, 1, 4)
        dom = dom.reshape(B * P, rep * Lq, 2 * D)
        dq, dk, dv = torch.empty_like(qm), torch.empty_like(km), torch.empty_like(vm)
        dl = torch.empty(B * P, rep, device=dev)
    step = max(1, min(B * P, CHUNK // (rep * Lq * Lk)))
    for g0 in range(0, B * P, step):
        g = slice(g0, g0 + step)
        n = vm[g].shape[0]
        a = []
        for m in range(2):
            s = torch.matmul(qm[m, g], km[m, g].transpose(1, 2)).mul_(scale)
            a.append(_softmax(s.reshape(n, rep, Lq, Lk), None if off is None else off[g]))
        both = torch.addcmul(a[0], a[1], lm[g], value=-1).reshape(n, rep * Lq, Lk)
        o[g] = torch.matmul(both, vm[g])
        if do is None:
            continue
        dv[g] = torch.matmul(both.transpose(1, 2), dom[g])
        del both
        da = torch.matmul(dom[g], vm[g].transpose(1, 2)).reshape(n, rep, Lq, Lk)
        for m in range(2):
            ad = a[m] * da
            delta = ad.sum(-1, keepdim=True)
            ds = ad.addcmul_(a[m], delta, value=-1).mul_(scale)
            if m == 1:
                dl[g] = -delta.double().sum((2, 3)).float()
                ds.mul_(-lm[g])
            ds = ds.reshape(n, rep * Lq, Lk)
            dq[m, g] = torch.matmul(ds, km[m, g])
            dk[m, g] = torch.matmul(ds.transpose(1, 2), qm[m, g])
    back = lambda t: t.reshape(B, P, rep, Lq, 2 * D).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)
    out = dict(o=back(o))
    if do is not None:
        two = lambda t, like, r, L: (t.reshape(2, B, P, r, L, D).permute(1, 4, 2, 3, 0, 5)
                                     .reshape(like.shape).to(like.dtype))
        out.update(dq=two(dq, q, rep, Lq), dk=two(dk, k, 1, Lk),
                   dv=dv.reshape(B, P, Lk, 2 * D).permute(0, 2, 1, 3).reshape(v.shape).to(v.dtype),
                   dlam=dl.reshape(B, P * rep).sum(0).to(lam.dtype))
    return out


def _norm_plain(st):
    c = st["case"]
    x, a, dt = st["x"], st["a"].float(), st["a"].dtype
    rows = (0, 1)
    ra = torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS)
    ah = a * ra
    k = st["scale"] * st["post"]
    k = k if st["gate"] is None else (k * st["gate"])[:, None]
    y = x + k * ah
    out = dict(y=y)
    if c["pre"]:
        ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        yh = y * ry
        out["n"] = (yh * st["pre"]).to(dt)
    if c["kind"] == "norm_fwd":
        return out
    dy = st["dy"]
    if c["pre"]:
        dn = st["dn"][0].float()
        for d in st["dn"][1:]:
            dn = dn + d.float()
        out["dpre"] = (dn * yh).sum(rows)
        u = dn * st["pre"]
        dy = dy + ry * (u - yh * (u * yh).mean(-1, keepdim=True))
    v = dy * k
    T = (dy * ah).sum(1)  # (B, D)
    gate = 1.0 if st["gate"] is None else st["gate"]
    out.update(dx=dy, da=(ra * (v - ah * (v * ah).mean(-1, keepdim=True))).to(dt),
               dscale=(gate * T).sum(0) * st["post"], dpost=(gate * T).sum(0) * st["scale"])
    if st["gate"] is not None:
        out["dgate"] = T * (st["scale"] * st["post"])
    return out


def _run_plain(st):
    c = st["case"]
    with torch.no_grad():
        if c["kind"].startswith("diff"):
            return _diff_plain(st["q"], st["k"], st["v"], st["lam"], st["ql"], st["kl"],
                               c["causal"], st.get("do"))
        if c["kind"].startswith("norm"):
            return _norm_plain(st)
        G = st["G"]
        X = G.float()
        if c["R"] > c["C"]:
            X = X.transpose(1, 2).contiguous()
        X = X / X.double().square().sum((1, 2), keepdim=True).sqrt().float()
        a, b, cc = COEFFS
        for _ in range(STEPS):
            A = torch.matmul(X, X.transpose(1, 2))
            B = torch.baddbmm(A, A, A, beta=b, alpha=cc)
            X = torch.baddbmm(X, B, X, beta=a)
        if c["R"] > c["C"]:
            X = X.transpose(1, 2).contiguous()
        return dict(X=X.to(G.dtype))


# ---------------------------------------------------------------------------
# The definitions in float64
# ---------------------------------------------------------------------------
def _diff_exact(x, c):
    """Block after block of the queries of one pair, its derivatives by autograd."""
    q, k, v, do = x["q"], x["k"], x["v"], x.get("do")
    rep = c["H"] // c["Hkv"]
    zeros = lambda t: torch.zeros(t.shape, device=t.device, dtype=torch.float64)
    out = dict(o=zeros(q))
    lam = x["lam"].double()
    if do is not None:
        out.update(dq=zeros(q), dk=zeros(k), dv=zeros(v), dlam=zeros(lam))
    for b, (lq, lk) in enumerate(zip(*lengths(c))):
        if lq == 0 or lk == 0:
            continue
        rows = max(1, min(lq, (1 << 27) // lk))
        for p in range(c["H"] // 2):
            kp = p // rep
            K = [k[b, :lk, 2 * kp + m].double().contiguous() for m in range(2)]
            V = torch.cat([v[b, :lk, 2 * kp], v[b, :lk, 2 * kp + 1]], -1).double()
            for i0 in range(0, lq, rows):
                i1 = min(lq, i0 + rows)
                Q = [q[b, i0:i1, 2 * p + m].double().contiguous() for m in range(2)]
                w = lam[p].clone()
                leaves = [*Q, *K, V, w]
                for t in leaves:
                    t.requires_grad_(do is not None)
                last = torch.arange(i0, i1, device=q.device) + (lk - lq if c["causal"] else lk)
                maps = []
                for m in range(2):
                    s = torch.matmul(Q[m], K[m].t()) / 8.0
                    if c["causal"]:
                        hid = torch.arange(lk, device=q.device)[None, :] > last[:, None]
                        s = torch.softmax(s.masked_fill(hid, -1e300), -1).masked_fill(hid, 0.0)
                    else:
                        s = torch.softmax(s, -1)
                    maps.append(s)
                O = torch.matmul(maps[0] - w * maps[1], V)
                out["o"][b, i0:i1, 2 * p:2 * p + 2] = O.detach().reshape(-1, 2, D)
                if do is None:
                    continue
                g = torch.autograd.grad(O, leaves,
                                        do[b, i0:i1, 2 * p:2 * p + 2].double().reshape(-1, 2 * D))
                for m in range(2):
                    out["dq"][b, i0:i1, 2 * p + m] = g[m]
                    out["dk"][b, :lk, 2 * kp + m] += g[2 + m]
                out["dv"][b, :lk, 2 * kp:2 * kp + 2] += g[4].reshape(-1, 2, D)
                out["dlam"][p] += g[5]
                del maps, O, g, leaves, s
    return out


def exact(c, seed):
    x = _inputs(c, seed)
    if c["kind"].startswith("diff"):
        return _diff_exact(x, c)
    if c["kind"] == "ortho":
        # on the other side: X (a + b G + c G^2) with G = X^T X
        X = x["G"].double()
        if c["R"] < c["C"]:
            X = X.transpose(1, 2)
        X = X / torch.linalg.matrix_norm(X)[:, None, None]
        a, b, cc = COEFFS
        eye = torch.eye(X.shape[2], device=X.device, dtype=torch.float64)
        for _ in range(STEPS):
            G = torch.matmul(X.transpose(1, 2).contiguous(), X)
            X = torch.matmul(X, a * eye + torch.matmul(G, b * eye + cc * G))
        return dict(X=X.transpose(1, 2) if c["R"] < c["C"] else X)
    t = {k: x[k].double().requires_grad_(c["kind"] == "norm_train")
         for k in ("x", "a", "scale", "post", "pre", "gate") if x[k] is not None}
    rms = lambda z: (z.square().mean(-1, keepdim=True) + EPS).sqrt()
    gate = t["gate"][:, None, :] if c["gate"] else 1.0
    y = t["x"] + gate * (t["a"] / rms(t["a"]) * t["post"]) * t["scale"]
    out, total = dict(y=y.detach()), [(y, x.get("dy"))]
    if c["pre"]:
        n = y / rms(y) * t["pre"]
        out["n"] = n.detach()
        total += [(n, d) for d in x.get("dn", ())]
    if c["kind"] == "norm_train":
        loss = sum((z * d.double()).sum() for z, d in total)
        out.update(zip(("d" + k for k in t), torch.autograd.grad(loss, list(t.values()))))
    return out

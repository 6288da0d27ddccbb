"""Dense attention, forward and backward, against float64 (tests/dense_attn_ref.py
derives the per-element bounds): types, head groups, one row to many, odd sizes, padded
batches, causal order, rows without a key, strides, and what memory holds behind a
sequence."""
from functools import partial

import pytest
import torch

from tests import dense_attn_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def inputs(seed, B, H, Hkv, Lq, Lk, dt, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    return [t.to(dt) for t in (gain * rn(B, H, Lq, 64), gain * rn(B, Hkv, Lk, 64),
                               rn(B, Hkv, Lk, 64), 0.3 * rn(B, H, Lq, 64))]


def run(q, k, v, do, lo=True, **kw):
    from imfvideo_amd import ops
    o, lse, *o_lo = ops.dense_attn_fwd(q, k, v, with_lo=lo, **kw)
    if lo:
        assert torch.equal(o, ops.dense_attn_fwd(q, k, v, **kw)[0])
        kw["o_lo"], = o_lo
    return dict(zip(("o", "lse", "dq", "dk", "dv"),
                    (o, lse, *ops.dense_attn_bwd(do, q, k, v, o, lse, **kw))))


def check_all(got, want, case):
    for n in ("o", "dq", "dk", "dv"):
        print("[ratio]", n, round(R.check(got[n], want[n], (case, n)), 3), flush=True)
    lse, ref = got["lse"].double().to(want["lse"][0].device), want["lse"][0]
    none = ref == float("-inf")
    assert torch.equal(none, lse == float("-inf")), (case, "lse of empty rows")
    assert ((lse - ref).abs()[~none] <= 1e-5 * (1 + ref.abs()[~none])).all(), (case, "lse")


# B, H, Hkv, Lq, Lk: one row and one key; edges of the 32- and 64-row tiles; odd ones;
# few queries over many keys (split keys, in both forms) and many over few (split queries); enough
# heads for the 128- and the 256-row forms; grouped key heads
SHAPES = [(1, 1, 1, 1, 1), (2, 2, 1, 1, 700), (1, 2, 2, 31, 33), (1, 2, 2, 64, 64),
          (2, 3, 3, 65, 63), (1, 4, 4, 274, 274), (2, 4, 2, 7, 1500), (1, 2, 1, 1333, 5),
          (1, 2, 2, 70, 1500), (2, 4, 2, 200, 2100), (3, 4, 1, 129, 130), (2, 64, 64, 200, 70),
          (2, 64, 32, 300, 97), (1, 128, 32, 257, 65)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "ragged", "both"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, mask, dt):
    B, H, Hkv, Lq, Lk = shape
    print("[case]", shape, mask, dt, flush=True)
    q, k, v, do = inputs(sum(shape), *shape, dt)
    causal = mask in ("causal", "both")
    ql = kl = None
    if mask in ("ragged", "both"):
        g = torch.Generator().manual_seed(B + Lq)
        ql = torch.randint(0, Lq + 1, (B,), generator=g)
        kl = torch.randint(0, Lk + 1, (B,), generator=g)
        ql[0], kl[B - 1] = Lq, Lk
    dev = "cuda" if H > 16 else "cpu"
    c = lambda t: None if t is None else t.cuda()
    for lo in (True, False):
        want = R.attention(q, k, v, causal, ql, kl, do=do, dev=dev, lo=lo)
        got = run(c(q), c(k), c(v), c(do), lo, causal=causal, q_lens=c(ql), k_lens=c(kl))
        torch.cuda.synchronize()
        check_all(got, want, (shape, mask, dt, lo))


@pytest.mark.parametrize("shape", [(1, 2, 2, 70, 90), (1, 2, 1, 3, 900), (2, 64, 64, 200, 70)])
@pytest.mark.parametrize("dt", DTYPES)
def test_what_the_rounding_lost(shape, dt):
    """o + o_lo is o before its rounding, to the rounding of o_lo: within the errors of P."""
    from imfvideo_amd import ops
    q, k, v, _ = inputs(7, *shape, dt)
    o, _, lo = ops.dense_attn_fwd(q.cuda(), k.cuda(), v.cuda(), with_lo=True)
    val, tol = R.attention(q, k, v, lo=True)["o"]
    u = torch.finfo(dt).eps / 2
    both = o.double().cpu() + lo.transpose(1, 2).double().cpu()
    assert ((both - val).abs() <= tol - u * (1 - u) * val.abs()).all()
    assert (lo.transpose(1, 2).double().abs().cpu() <= u * 1.01 * o.double().abs().cpu()
            + torch.finfo(dt).smallest_normal).all()


@pytest.mark.parametrize("shape", [(1, 2, 2, 70, 90), (2, 4, 2, 7, 500), (1, 2, 1, 250, 33),
                                   (1, 128, 128, 100, 70)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt", DTYPES)
def test_small_gradients_keep_what_rounding_loses(shape, causal, dt):
    """Few keys and rows: P and dS enter their products with the half that rounding them
    lost, so an element is off by its own rounding u |x| and second-order terms: dS's
    u^2 |dS|, and through delta P's u^2 P |v| and the u^2 |o| of the output's second half,
    each at most u^2 P mag with mag = |dout| . |v_j| + |dout| . P |v|; fp32 arithmetic T32 of
    the same sums for S, dP and delta."""
    q, k, v, do = inputs(7 + sum(shape), *shape, dt)
    B, H, Hkv, Lq, Lk = shape
    rep = H // Hkv
    got = run(*[t.cuda() for t in (q, k, v, do)], True, causal=causal)
    torch.cuda.synchronize()
    want = R.attention(q, k, v, causal, do=do)
    u, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    see = R.visible(B, Lq, Lk, causal, None, None)[:, None]
    K, V = (t.double().repeat_interleave(rep, 1) for t in (k, v))
    s = (q.double() @ K.transpose(-1, -2) / 8).masked_fill(~see, float("-inf"))
    P = torch.softmax(s, -1).nan_to_num(0.0)
    g = do.double().abs()
    mag = g @ V.abs().transpose(-1, -2) + (g * (P @ V.abs())).sum(-1, keepdim=True)
    E = (4 * u * u + 3 * R.T32) * P * mag + 2.0 ** -36 * see * mag.amax((-1, -2), keepdim=True)
    heads = lambda t: t.reshape(B, Hkv, rep, Lk, 64).sum(2)
    more = dict(dq=E @ K.abs() / 8, dk=heads(E.transpose(-1, -2) @ q.double().abs()) / 8,
                dv=heads(((2 * u * u + R.T32) * P + 2.0 ** -36 * see).transpose(-1, -2) @ g))
    for n in more:
        val = want[n][0]
        R.check(got[n], (val, u * val.abs() + more[n] + tiny), (shape, causal, dt, n))


@pytest.mark.parametrize("dt", DTYPES)
def test_one_key_has_no_score_gradient(dt):
    """The softmax of one key is 1 whatever its score: dq and dk are zero."""
    q, k, v, do = [t.cuda() for t in inputs(3, 2, 4, 2, 37, 5, dt)]
    lens = torch.tensor([1, 5], device="cuda")
    got = run(q, k, v, do, k_lens=lens)
    assert not got["dq"][0].any() and not got["dk"][0].any()
    assert got["dq"][1].any() and got["dk"][1].any()
    got = run(q, k[:, :, :1], v[:, :, :1], do, causal=True)
    assert not got["dq"].any() and not got["dk"].any() and got["dv"].any()


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_behind_a_sequence_are_not_used(dt):
    """NaN, infinities and the type's lowest value behind the sequences change nothing,
    bit for bit, and their rows come back as zeros."""
    B, H, Hkv, Lq, Lk = 4, 4, 2, 150, 170
    q, k, v, do = (t.cuda() for t in inputs(3, B, H, Hkv, Lq, Lk, dt))
    ql = torch.tensor([150, 77, 0, 1], device="cuda", dtype=torch.int32)
    kl = torch.tensor([65, 170, 9, 0], device="cuda", dtype=torch.int32)
    for causal in (False, True):
        base = None
        for junk in (0.0, float("nan"), float("inf"), torch.finfo(dt).min):
            print("[case]", dt, causal, junk, flush=True)
            x = [t.clone() for t in (q, k, v, do)]
            for b in range(B):
                x[0][b, :, int(ql[b]):] = junk
                x[1][b, :, int(kl[b]):] = junk
                x[2][b, :, int(kl[b]):] = junk
                x[3][b, :, int(ql[b]):] = junk
                empty = int(ql[b]) if kl[b] == 0 else max(0, int(ql[b] - kl[b])) * causal
                x[3][b, :, :empty] = junk  # rows without a key take no gradient
            got = run(*x, causal=causal, q_lens=ql, k_lens=kl)
            torch.cuda.synchronize()
            for b in range(B):
                assert not got["o"][b, :, int(ql[b]):].any()
                assert not got["dq"][b, :, int(ql[b]):].any()
                assert not got["dk"][b, :, int(kl[b]):].any()
                assert not got["dv"][b, :, int(kl[b]):].any()
            base = base or got
            for n in got:
                assert torch.equal(got[n], base[n]), (n, junk, causal)


def test_strides_and_layouts():
    """Token-major views, bands of a wider projection, broadcast heads, odd alignment
    and a wide row stride give what contiguous operands give, bit for bit."""
    B, H, L = 2, 4, 130
    q, k, v, do = (t.cuda() for t in inputs(5, B, H, H, L, L, torch.bfloat16))
    want = run(q, k, v, do)
    tok = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((B, L, H, 160), float("nan"), device="cuda", dtype=torch.bfloat16)

    def band(t, lo):
        w = wide.clone()
        w[..., lo:lo + 64] = t.transpose(1, 2)
        return w[..., lo:lo + 64].transpose(1, 2)

    def odd(t):
        flat = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    for name, f in (("token", tok), ("band", partial(band, lo=32)), ("odd band", partial(band, lo=3)),
                    ("odd", odd)):
        print("[case]", name, flush=True)
        got = run(f(q), f(k), f(v), f(do))
        for n in want:
            assert torch.equal(got[n], want[n]), (name, n)
    print("[case] broadcast", flush=True)
    kb, vb, qb = k[:, :1].expand(B, H, L, 64), v[:1].expand(B, H, L, 64), q[:, :, :1].expand_as(q)
    got = run(qb, kb, vb, do)
    ref = run(qb.contiguous(), kb.contiguous(), vb.contiguous(), do)
    for n in ref:
        assert torch.equal(got[n], ref[n]), n


def test_lengths_out_of_range_are_clamped():
    q, k, v, do = (t.cuda() for t in inputs(6, 3, 2, 2, 70, 90, torch.float16))
    lens = lambda *x: torch.tensor(x, device="cuda")
    got = run(q, k, v, do, causal=True, q_lens=lens(-5, 70, 2 ** 40), k_lens=lens(90, 1000, -1))
    want = run(q, k, v, do, causal=True, q_lens=lens(0, 70, 70), k_lens=lens(90, 90, 0))
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_lengths_of_zero():
    from imfvideo_amd.imf_dit_video import dense_attention
    z = lambda B, L: torch.zeros(B, L, 2, 64, device="cuda", dtype=torch.bfloat16,
                                 requires_grad=True)
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0), (2, 0, 0)):
        print("[case]", B, Lq, Lk, flush=True)
        q, k, v = z(B, Lq), z(B, Lk), z(B, Lk)
        o = dense_attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        o.sum().backward()
        assert all(t.grad.shape == t.shape and not t.grad.any() for t in (q, k, v))


def test_sharp_and_flat_rows_fp16():
    """Rows of one key, rows spread over many keys with probabilities below fp16's
    normal range, and gradients far from one (a loss scale)."""
    B, H, L = 1, 2, 2100
    q, k, v, do = inputs(8, B, H, H, L, L, torch.float16)
    q[:, 0] *= 4.0
    q[:, 1] = 0.0
    for mul in (2.0 ** 12, 2.0 ** -12):
        print("[case]", mul, flush=True)
        d = (do.float() * mul).half()
        want = R.attention(q, k, v, do=d, dev="cuda")
        got = run(q.cuda(), k.cuda(), v.cuda(), d.cuda())
        for n in ("o", "dk", "dv", "dq"):
            val, tol = want[n]
            ok = val.abs() < 6e4  # past fp16's range the gradient is an infinity
            err = (got[n].double() - val).abs()
            assert (err <= tol)[ok].all(), (n, mul, (err / tol)[ok].max().item())


def test_a_row_maximum_that_keeps_rising():
    """Keys in rising order of their score move the running bound at every tile."""
    L = 900
    for dt in DTYPES:
        q, k, v, do = inputs(9, 1, 1, 1, 40, L, dt)
        k = (k.float().abs() * torch.linspace(0.0, 4.0, L)[:, None]).to(dt)
        q = q.abs()
        check_all(run(q.cuda(), k.cuda(), v.cuda(), do.cuda()),
                  R.attention(q, k, v, do=do), ("rising", dt))


@pytest.mark.parametrize("dt", DTYPES)
def test_gradients_against_differences(dt):
    """<gradient, direction> against central differences of the float64 forward."""
    q, k, v, do = inputs(10, 1, 2, 1, 37, 45, dt, gain=1.0)
    got = run(q.cuda(), k.cuda(), v.cuda(), do.cuda(), causal=True)
    want = R.attention(q, k, v, causal=True, do=do)
    g = torch.Generator().manual_seed(1)

    def loss(q, k, v):
        see = R.visible(1, 37, 45, True, None, None)[:, None]
        s = (q @ k.repeat_interleave(2, 1).transpose(-1, -2) / 8).masked_fill(~see, float("-inf"))
        return ((torch.softmax(s, -1) @ v.repeat_interleave(2, 1)) * do.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        hi, lo = ([t + s * h * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        diff = ((loss(*hi) - loss(*lo)) / (2 * h)).item()
        mine = (got[n].cpu().double() * d).sum().item()
        assert abs(mine - diff) <= (want[n][1] * d.abs()).sum().item() + 1e-8, (n, mine, diff)


def test_long_cache_offsets_past_32_bits():
    """20 million keys of one head: 2.56 GB of keys, byte offsets past 2^31; the heavy
    keys sit at the far end."""
    from imfvideo_amd import ops
    L = 20_000_003
    g = torch.Generator(device="cuda").manual_seed(4)
    k = torch.empty(1, 1, L, 64, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    v = torch.empty_like(k).normal_(generator=g)
    q = torch.empty(1, 1, 2, 64, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    do = torch.empty_like(q).normal_(generator=g)
    k[..., -300:, :] += 2.0 * q[:, :, :1]  # row 0 attends the end
    print("[case] long forward", flush=True)
    o, lse = ops.dense_attn_fwd(q, k, v)
    print("[case] long backward", flush=True)
    dq, dk, dv = ops.dense_attn_bwd(do, q, k, v, o, lse)
    torch.cuda.synchronize()
    s = torch.cat([q[0, 0].double() @ c.double().t() for c in k[0, 0].split(1 << 22)], 1) / 8
    p = torch.softmax(s, -1)
    parts = list(zip(p.split(1 << 22, 1), v[0, 0].split(1 << 22)))
    ref = sum(a @ b.double() for a, b in parts)
    pv = sum(a @ b.double().abs() for a, b in parts)
    u = 2.0 ** -8
    assert ((o[0, 0].double() - ref).abs() <= u * ref.abs() + (u + 1e-4) * pv).all()
    tail = slice(L - 5000, L)
    dv_ref = p[:, tail].t() @ do[0, 0].double()
    bound = u * dv_ref.abs() + (u + 1e-4) * (p[:, tail].t() @ do[0, 0].double().abs()) + 1e-30
    assert ((dv[0, 0, tail].double() - dv_ref).abs() <= bound).all()
    dp = do[0, 0].double() @ v[0, 0, tail].double().t()
    delta = (do[0, 0].double() * ref).sum(-1, keepdim=True)
    ds = p[:, tail] * (dp - delta)
    dk_ref = ds.t() @ q[0, 0].double() / 8
    ed = (do[0, 0].double().abs() * (u * ref.abs() + (u + 1e-4) * pv)).sum(-1, keepdim=True)
    es = (u + 1e-4) * ds.abs() + p[:, tail] * (ed + 1e-4 * (dp.abs() + delta.abs()))
    bound = u * dk_ref.abs() + es.t() @ q[0, 0].double().abs() / 8 + 1e-30
    assert ((dk[0, 0, tail].double() - dk_ref).abs() <= bound).all()


def test_results_repeat_and_streams_do_not_mix():
    """Bit-identical results over repeated calls and on two streams at once."""
    shapes = [(1, 4, 2, 5, 3000), (2, 8, 8, 300, 300)]
    xs = [[t.cuda() for t in inputs(12 + i, *s, torch.bfloat16)] for i, s in enumerate(shapes)]
    want = [run(*x, causal=True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(5):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                outs.append(run(*x, causal=True))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        for n in got:
            assert torch.equal(got[n], want[i % 2][n]), (i, n)


@pytest.mark.parametrize("shape", [(1, 4, 4, 274, 274), (2, 2, 1, 3, 2000)])
def test_graph_replays_match_eager(shape):
    from imfvideo_amd import ops
    x = [t.cuda() for t in inputs(13, *shape, torch.float16)]
    lens = torch.tensor([shape[4] - 3] * shape[0], device="cuda", dtype=torch.int32)

    def step():
        q, k, v, do = x
        o, lse = ops.dense_attn_fwd(q, k, v, k_lens=lens)
        return [o, lse, *ops.dense_attn_bwd(do, q, k, v, o, lse, k_lens=lens)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    for r in range(4):
        for t in x:
            t.copy_(torch.randn(t.shape, device="cuda") * 0.5)
        lens.fill_(shape[4] - 5 * r)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_autograd_entry():
    """dense_attention: autograd's gradients are the op's; broadcast inputs and a shared
    key head collect theirs; autocast casts; no-grad gives the same output."""
    from imfvideo_amd.imf_dit_video import dense_attention
    q, k, v, do = (t.cuda().transpose(1, 2).contiguous()
                   for t in inputs(14, 2, 4, 2, 50, 60, torch.bfloat16))
    kl = torch.tensor([60, 41])
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = dense_attention(*x, causal=True, k_lens=kl.cuda())
    grads = torch.autograd.grad(o, x, do)
    ref = run(*(t.transpose(1, 2) for t in (q, k, v, do)), causal=True, k_lens=kl)
    assert torch.equal(o, ref["o"].transpose(1, 2))
    for a, n in zip(grads, ("dq", "dk", "dv")):
        assert torch.equal(a, ref[n].transpose(1, 2)), n
    with torch.no_grad():
        assert torch.equal(dense_attention(*x, causal=True, k_lens=[60, 41]), o)
    one = k[:, :1].clone().requires_grad_(True)  # one key row for every position
    o = dense_attention(q, one.expand(2, 60, 2, 64), v)
    g, = torch.autograd.grad(o, one, do)
    want = run(*(t.transpose(1, 2) for t in (q, one.detach().expand(2, 60, 2, 64), v, do)))
    assert torch.equal(g, want["dk"].transpose(1, 2).sum(1, keepdim=True))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        o32 = dense_attention(q.float(), k, v.float())
    assert o32.dtype == torch.bfloat16 and torch.equal(o32, dense_attention(q, k, v))


def test_only_the_gradients_asked_for():
    """Frozen keys or queries: the others' gradients are the same bits; an expanded output
    gradient (of a sum) is taken too."""
    from imfvideo_amd import ops
    from imfvideo_amd.imf_dit_video import dense_attention
    x = [t.cuda().transpose(1, 2).contiguous()
         for t in inputs(16, 2, 4, 2, 70, 90, torch.float16)[:3]]
    req = lambda *on: [t.clone().requires_grad_(r) for t, r in zip(x, on)]
    full = req(True, True, True)
    want = torch.autograd.grad(dense_attention(*full).sum(), full)
    for on in ((True, False, False), (False, True, True), (False, True, False), (False, False, True)):
        a = req(*on)
        leaves = [t for t, r in zip(a, on) if r]
        got = torch.autograd.grad(dense_attention(*a).sum(), leaves)
        for g, w in zip(got, [w for w, r in zip(want, on) if r]):
            assert torch.equal(g, w), on
    o, lse = ops.dense_attn_fwd(*x, tok=True)
    assert ops.dense_attn_bwd(o, *x, o, lse, tok=True, need_kv=False)[1:] == (None, None)


def test_autograd_in_a_graph():
    """Forward and backward of the autograd entry captured together, while an eager graph of
    other leaves lives; replays on refilled inputs match eager calls."""
    from imfvideo_amd.imf_dit_video import dense_attention
    x = [t.cuda().transpose(1, 2).contiguous() for t in inputs(17, 1, 2, 2, 130, 130,
                                                               torch.bfloat16)]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in x[:3]]
        o = dense_attention(*leaves, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, x[3])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    other = x[0].clone().requires_grad_(True)
    alive = dense_attention(other, x[1], x[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    for _ in range(4):
        for t in x:
            t.copy_(torch.randn(t.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    del alive


def test_infinite_scores():
    """A score of +inf makes its row NaN; a row whose scores are all -inf is NaN as the
    softmax of it is; other rows are not touched."""
    from imfvideo_amd import ops
    for L in (40, 300):
        q, k, v, _ = (t.cuda() for t in inputs(18, 1, 64, 64, L, L, torch.bfloat16))
        base, _ = ops.dense_attn_fwd(q, k, v)
        q2, k2 = q.clone(), k.abs()
        want, _ = ops.dense_attn_fwd(q2, k2, v)
        q2[:, :, 5] = float("inf")
        q2[:, :, 7] = float("-inf")
        o, lse = ops.dense_attn_fwd(q2, k2, v)
        assert torch.isnan(o[:, :, 5]).all() and torch.isnan(o[:, :, 7]).all()
        keep = [i for i in range(L) if i not in (5, 7)]
        assert torch.equal(o[:, :, keep], want[:, :, keep])
        assert torch.isfinite(base).all()


def test_autograd_refusals():
    from imfvideo_amd.imf_dit_video import dense_attention
    x = [torch.randn(1, 8, 2, 64, device="cuda").half().requires_grad_(True) for _ in range(3)]
    o = dense_attention(*x)
    g, = torch.autograd.grad(o.float().sum(), x[0], create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        torch.autograd.grad(g.float().sum(), x[0])
    o = dense_attention(*x)
    with pytest.raises(RuntimeError, match="one gradient at a time"):
        torch.autograd.grad(o, x, torch.ones(3, *o.shape, device="cuda").half(),
                            is_grads_batched=True)
    o = dense_attention(*x)
    with torch.no_grad():
        x[1].add_(1.0)  # an operand changed between forward and backward
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.float().sum().backward()
    with pytest.raises(TypeError):
        dense_attention(*(t.detach().float() for t in x))


def test_block_with_dense_attention():
    """A TransformerBlock over dense_attention under bf16 autocast: the output and the
    gradients of a block over the library's attention, within the roundings of the 16-bit
    path: two evaluations of one block that differ by a rounding of the attention's
    operands' type at a few places; every entry within eight steps of the tensor's largest."""
    from imfvideo_amd.imf_dit_video import (TransformerBlock, dense_attention,
                                            precompute_axial_rope_3d, sdpa_math_attention)
    torch.manual_seed(15)
    make = lambda f: TransformerBlock(128, 2, 64, 32, 32, 32, 64, mlp_ratio=2, attn_impl=f).cuda()
    a = make(dense_attention)
    with torch.no_grad():
        a.attn_scale.fill_(0.5), a.mlp_scale.fill_(0.5)
    b = make(sdpa_math_attention)
    b.load_state_dict(a.state_dict())
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(32, (2, 8, 8), 18))
    x = torch.randn(2, 146, 128, device="cuda")
    dy = torch.randn(2, 146, 128, device="cuda")
    res = []
    for m in (a, b):
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(xi, cos, sin)
        y.backward(dy)
        res.append([y.detach(), xi.grad] + [p.grad for p in m.parameters()])
    for s, t in zip(*res):
        assert torch.isfinite(s).all()
        assert (s - t).abs().max() <= 8 * 2.0 ** -8 * t.abs().max()

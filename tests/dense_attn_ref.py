"""Dense attention and its gradients in float64, with per-element bounds of the
rounding errors that the 16-bit kernels may make.

With u half a unit in the last place of the operands' type (eps / 2) and t a bound for fp32
arithmetic (products, hardware exp2 and log2, log-sum-exp, sums):
  P is rounded to 16 bits for P v:           |do| <= u |o| + (u + t) P |v|
  delta is taken from the rounded o, or, with its second half, from one that carries
  the errors before that rounding only: |ddelta| <= |dout| . (|do| (- u |o|)) + t |dout| . P|v|
  P and dS are rounded before the products:  |ddv| <= u |dv| + (u + t) P^T |dout|
    |ddS| <= (u + t) |dS| + P (|ddelta| + t |dout| |v|^T + t |delta|)
  |ddq| <= u |dq| + scale |ddS| |k| + t scale |dS| |k|,  dk alike.
Each also takes one step of the type's subnormals.
"""
import torch

T32 = 2e-5  # exponents up to 2^6 at 2^-23, the hardware exp2 / log2 and the sums


def visible(B, Lq, Lk, causal, ql, kl):
    """(B, Lq, Lk) bool: query i sees key j."""
    i, j = torch.arange(Lq)[:, None], torch.arange(Lk)[None, :]
    out = torch.empty(B, Lq, Lk, dtype=torch.bool)
    for b in range(B):
        n = Lq if ql is None else min(max(int(ql[b]), 0), Lq)
        m = Lk if kl is None else min(max(int(kl[b]), 0), Lk)
        out[b] = (i < n) & (j < m)
        if causal:
            out[b] &= j <= i + m - n
    return out


def attention(q, k, v, causal=False, ql=None, kl=None, scale=None, do=None, dev="cpu",
              lo=False):
    """(B, H, L, 64) operands -> dict of name -> (value, bound), float64 on dev; lse
    without a bound (-inf where no key is seen)."""
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    rep = H // Hkv
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Lq, Lk, causal, ql, kl).to(dev)[:, None]
    keep_q, keep_k = see.any(-1, keepdim=True), see.any(-2)[..., None]
    f = lambda t: t.to(dev).double()
    q, k, v = f(q), f(k), f(v)
    q = q.masked_fill(~keep_q, 0.0)
    k, v = k.masked_fill(~keep_k, 0.0), v.masked_fill(~keep_k, 0.0)
    K, V = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = (q @ K.transpose(-1, -2) * scale).masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(s, -1)
    P = torch.exp(s - lse.masked_fill(lse == float("-inf"), 0.0)[..., None])
    o = P @ V
    PV = P @ V.abs()
    eo = u * o.abs() + (u + T32) * PV + tiny
    out = dict(o=(o, eo), lse=(lse, None))
    if do is None:
        return out
    g = f(do).masked_fill(~keep_q, 0.0)
    delta = (g * o).sum(-1, keepdim=True)
    dP = g @ V.transpose(-1, -2)
    dS = P * (dP - delta)
    eo = eo - u * (1 - u) * o.abs() if lo else eo
    ed = (g.abs() * eo).sum(-1, keepdim=True) + T32 * (g.abs() * PV).sum(-1, keepdim=True)
    mag = g.abs() @ V.abs().transpose(-1, -2) + delta.abs()
    eS = (u + T32) * dS.abs() + P * (ed + T32 * mag) + 2.0 ** -36 * see * mag.amax((-1, -2),
                                                                              keepdim=True)
    heads = lambda t: t.reshape(B, Hkv, rep, Lk, D).sum(2)
    dq = scale * dS @ K
    dk = scale * heads(dS.transpose(-1, -2) @ q)
    dv = heads(P.transpose(-1, -2) @ g)
    eq = u * dq.abs() + scale * (eS + T32 * dS.abs()) @ K.abs() + tiny
    ek = u * dk.abs() + scale * heads((eS + T32 * dS.abs()).transpose(-1, -2) @ q.abs()) + tiny
    ev = u * dv.abs() + heads(((u + T32) * P + 2.0 ** -36 * see).transpose(-1, -2) @ g.abs()) + tiny
    out.update(dq=(dq, eq), dk=(dk, ek), dv=(dv, ev))
    return out


def check(got, want, what):
    """Every element of got within the bound of want = (value, bound)."""
    val, tol = want
    err = (got.to(val.device).double() - val).abs()
    ratio = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, "error over bound", ratio, "largest", err.max().item())
    return ratio

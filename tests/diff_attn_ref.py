"""Differential attention and its gradients in float64, with per-element bounds of the
rounding errors that the 16-bit kernels may make.

With u half a unit in the last place of the operands' type (eps / 2) and t a bound for fp32
arithmetic (dense_attn_ref.T32), A_m = P_m the two maps, C = P_1 - lam P_2, |C| = P_1 + |lam| P_2:
  P_m is rounded to 16 bits for P_m v:      |do| <= u |o| + (u + t) |C| |v|
  delta_m = dout . P_m v from fp32 sums of the rounded P_m: |ddelta_m| <= (u + t) |dout| . P_m |v|
  C and dS_m are rounded before the products: |ddv| <= u |dv| + (u + t) |C|^T |dout|
    |ddS_m| <= (u + t) |dS_m| + P_m (|ddelta_m| + t (|dout| |v|^T + |delta_m|)), times |lam| for m = 2
  |ddq_m| <= u |dq_m| + scale (|ddS_m| + t |dS_m|) |k_m|,  dk_m alike
  |ddlam| <= sum |ddelta_2| + t sum |delta_2|, and u |dlam| of a 16-bit lam.
Each also takes one step of the type's subnormals, and fp16's maps and dS, held with shared
powers of two, 2^-36 of the largest of their kind.
"""
import torch

from tests.dense_attn_ref import T32, check, visible  # noqa: F401


def attention(q, k, v, lam, causal=False, ql=None, kl=None, scale=None, do=None, dev="cpu"):
    """(B, L, H, 64) operands -> dict of name -> (value, bound), float64 on dev; lse without a
    bound."""
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    P, rep = H // 2, H // Hkv
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Lq, Lk, causal, ql, kl).to(dev)[:, None]
    keep_q, keep_k = see.any(-1, keepdim=True), see.any(-2)[..., None]
    heads = lambda t: t.to(dev).double().transpose(1, 2)
    wide = lambda t, n: (t.to(dev).double().reshape(B, -1, n, 2 * D).transpose(1, 2))
    q, k = heads(q).masked_fill(~keep_q, 0.0), heads(k).masked_fill(~keep_k, 0.0)
    qm = [q[:, m::2] for m in range(2)]
    km = [k[:, m::2].repeat_interleave(rep, 1) for m in range(2)]
    V = wide(v, Hkv // 2).masked_fill(~keep_k, 0.0).repeat_interleave(rep, 1)
    w = lam.to(dev).double()[None, :, None, None]
    maps, lse = [], []
    for m in range(2):
        s = (qm[m] @ km[m].transpose(-1, -2) * scale).masked_fill(~see, float("-inf"))
        lse.append(torch.logsumexp(s, -1))
        maps.append(torch.exp(s - lse[m].masked_fill(lse[m] == float("-inf"), 0.0)[..., None]))
    C, absC = maps[0] - w * maps[1], maps[0] + w.abs() * maps[1]
    o = C @ V
    back = lambda t, n: t.transpose(1, 2).reshape(B, -1, n, D)
    out = dict(o=(back(o, H), back(u * o.abs() + (u + T32) * (absC @ V.abs()) + tiny, H)),
               lse=(torch.stack(lse, 2).reshape(B, H, Lq), None))
    if do is None:
        return out
    g = wide(do, P).masked_fill(~keep_q, 0.0)
    dA = g @ V.transpose(-1, -2)
    magA = g.abs() @ V.abs().transpose(-1, -2)
    share = lambda t: t.reshape(B, Hkv // 2, rep, Lk, -1).sum(2)
    dq, eq, dk, ek = [], [], [], []
    for m in range(2):
        f = 1.0 if m == 0 else -w
        delta = (maps[m] * dA).sum(-1, keepdim=True)
        ed = (u + T32) * (maps[m] * magA).sum(-1, keepdim=True)
        dS = f * maps[m] * (dA - delta)
        mag = magA + delta.abs()
        fa = 1.0 if m == 0 else w.abs()
        # (the shared power of two also covers max(1, |lam|))
        eS = ((u + 2 * T32) * dS.abs() + fa * maps[m] * (ed + T32 * mag)
              + 2.0 ** -36 * see * mag.amax((-1, -2), keepdim=True) * w.abs().clamp_min(1.0))
        if m == 1:
            dlam = -delta.sum((0, 2, 3))
            el = (ed + T32 * delta.abs()).sum((0, 2, 3))
        dq.append(scale * dS @ km[m])
        eq.append(u * dq[m].abs() + scale * eS @ km[m].abs() + tiny)
        dk.append(share(scale * dS.transpose(-1, -2) @ qm[m]))
        ek.append(u * dk[m].abs() + share(scale * eS.transpose(-1, -2) @ qm[m].abs()) + tiny)
    dv = share(C.transpose(-1, -2) @ g)
    ev = u * dv.abs() + share(((u + T32) * absC + 2.0 ** -36 * see * (1 + w.abs())).transpose(-1, -2)
                              @ g.abs()) + tiny
    two = lambda t, n: torch.stack(t, 2).reshape(B, n, -1, D).transpose(1, 2)
    ul = torch.finfo(lam.dtype).eps / 2
    out.update(dq=(two(dq, H), two(eq, H)), dk=(two(dk, Hkv), two(ek, Hkv)),
               dv=(back(dv, Hkv), back(ev, Hkv)),
               dlam=(dlam, el + ul * dlam.abs() + 1e-30))
    return out

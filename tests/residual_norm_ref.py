"""The residual step with a norm on both sides and its gradients in float64, with
per-element bounds of what fp32 arithmetic and one rounding of each result may be off.

With t a bound for fp32 arithmetic (sums of up to 8,192 squares or products, a lane's part
of at most 64 of them in sequence and the rest in a tree: below 100 roundings of 2^-24, the
square root's reciprocal and a handful of products) and u half a unit in the last place of a's
type (0 for fp32):
  |dy| <= t (|x| + |k ah|),  |dn| <= u |n| + t |n| + r |w_pre| (t-errors of y, its norm's too)
  gradients: t times the sums of the absolute values of their terms, and u of a 16-bit one.
"""
import torch

T32 = 2e-5


def step(x, a, scale, post, pre=None, gate=None, eps=1e-6, dy=None, dns=()):
    """(B, L, D) operands -> dict of name -> (value, bound), float64."""
    u = torch.finfo(a.dtype).eps / 2 if a.dtype != torch.float32 else 0.0
    tiny = torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps if u else 1e-38
    f = lambda t: None if t is None else t.double()
    x, a, scale, post, pre, gate, dy = map(f, (x, a, scale, post, pre, gate, dy))
    g = torch.ones(x.shape[0], 1, x.shape[2], dtype=torch.float64, device=x.device)
    g = g if gate is None else gate[:, None]
    rms = lambda t: torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)
    ra = rms(a)
    ah = a * ra
    k = scale * post * g
    y = x + k * ah
    ey = T32 * (x.abs() + (k * ah).abs())
    out = dict(y=(y, ey))
    if pre is not None:
        ry = rms(y)
        yh = y * ry
        n = yh * pre
        # y's own errors reach n through the value and through the norm
        eyh = ry * ey + T32 * yh.abs() + yh.abs() * ry * (ey * yh.abs()).mean(-1, keepdim=True)
        out["n"] = (n, u * n.abs() + pre.abs() * eyh + tiny)
    if dy is None and not dns:
        return out
    dy = torch.zeros_like(x) if dy is None else dy
    ed = T32 * dy.abs()
    if dns:
        dn = sum(d.double() for d in dns)
        v = dn * pre
        m = (v * yh).mean(-1, keepdim=True)
        mm = (v * yh).abs().mean(-1, keepdim=True)
        dy = dy + ry * (v - yh * m)
        # second-order: the backward's y is the forward's, off by ey
        rel = (ey * yh.abs()).mean(-1, keepdim=True) * ry
        ed = ed + T32 * ry * (v.abs() + yh.abs() * mm) + ry * (
            rel * (v.abs() + 3 * yh.abs() * mm) + eyh * m.abs()
            + yh.abs() * (v.abs() * eyh).mean(-1, keepdim=True))
        rows = (0, 1)
        out["dpre"] = ((dn * yh).sum(rows), (dn.abs() * (eyh + T32 * yh.abs())).sum(rows))
    w = dy * k
    ew = ed * k.abs() + T32 * w.abs()
    m = (w * ah).mean(-1, keepdim=True)
    mm = ((T32 * w.abs() + ew) * ah.abs()).mean(-1, keepdim=True)
    da = ra * (w - ah * m)
    T, eT = (dy * ah).sum(1), ((ed + T32 * dy.abs()) * ah.abs()).sum(1)
    G = g[:, 0]
    out.update(dx=(dy, ed + 1e-38), da=(da, u * da.abs() + ra * (ew + ah.abs() * (mm + T32 * m.abs())) + tiny),
               dscale=((G * T).sum(0) * post, (G.abs() * eT).sum(0) * post.abs() + 1e-38),
               dpost=((G * T).sum(0) * scale, (G.abs() * eT).sum(0) * scale.abs() + 1e-38))
    if gate is not None:
        out["dgate"] = (T * scale * post, eT * (scale * post).abs() + 1e-38)
    return out


def check(got, want, what):
    """Every element of got within the bound of want = (value, bound)."""
    val, tol = want
    assert got.shape == val.shape, (what, got.shape, val.shape)
    err = (got.double() - val).abs()
    ratio = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, "error over bound", ratio, "largest", err.max().item())
    return ratio

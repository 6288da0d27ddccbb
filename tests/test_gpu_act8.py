"""Activations kept in 8 bits: codes and scales against the law bit for bit, the gate
product and the weight gradient that read them against float64, and the MLP that uses them
together.

Tolerances: a 16-bit output is rounded once from fp32, u = eps / 2 of its type, and the
fp32 chain (three exps and reciprocals of one ulp, a dozen products) adds at most 2^-18
relative; the slope of the gate is a sum of two terms that may cancel, so its bound takes
their magnitudes.  The weight gradient's products are exact, its fp32 sums of R terms in
blocks of 64 round at most 64 + ceil(R / 64) + 64 times on a term's way, each 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
CHAIN = 2.0 ** -18


def law(x):
    """(codes (Rb, Cb, 64, 64), scales (Rb, Cb), values fp32 (R, C)) on the CPU."""
    R, C = x.shape
    t = torch.nn.functional.pad(x.float().cpu(), (0, -C % 64, 0, -R % 64))
    t = t.reshape(-(-R // 64), 64, -(-C // 64), 64).transpose(1, 2)
    top = t.abs().amax((2, 3))
    s = top / torch.full_like(top, 127.0) + 1e-12
    s = torch.where(torch.isfinite(top), s, torch.full_like(s, float("nan")))
    y = t / s[..., None, None]
    # halves away from zero on the fp32 quotient, in float64 where + 0.5 is exact
    n = torch.copysign(torch.floor(y.double().abs() + 0.5), y.double())
    codes = torch.where(torch.isnan(n), torch.zeros_like(n), n).to(torch.int8)
    val = codes.float() * s[..., None, None]
    val = val.transpose(1, 2).reshape(t.shape[0] * 64, -1)[:R, :C]
    return codes, s, val


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(
        torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (63, 65), (64, 64), (130, 512), (300, 1365),
                                   (77, 2048), (1000, 7)])
def test_pack_and_unpack(shape, dt):
    from imfvideo_amd import ops
    print("[case]", shape, dt, flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(shape[1], generator=g))).to(dt)
    a = ops.act8_pack(x.cuda())
    codes, s, val = law(x)
    assert torch.equal(a.scales.cpu(), s)
    assert torch.equal(a.codes.cpu(), codes)
    assert torch.equal(ops.act8_unpack(a, dt).cpu(), val.to(dt))
    other = torch.float16 if dt == torch.bfloat16 else torch.bfloat16
    assert torch.equal(ops.act8_unpack(a, other).cpu(), val.to(other))


def test_pack_every_border_between_codes():
    """x at, one step above and one below (k + 1/2) s for every k, over scales of all
    mantissas and magnitudes (fp16's subnormals to bf16's largest)."""
    from imfvideo_amd import ops
    rows = []
    for dt, tops in ((torch.bfloat16, [1.0, 1.9921875, 1.3671875, 127.0, 2.0 ** 127, 2.0 ** -100,
                                       0.0, 254.0]),
                     (torch.float16, [1.0, 65504.0, 127.0, 2.0 ** -24, 127 * 2.0 ** -24, 0.7])):
        for top in tops:
            top = torch.tensor(top).to(dt)
            k = torch.arange(127, dtype=torch.float64) + 0.5
            x = (k * (top.double() / 127)).to(dt)
            i = x.view(torch.int16)
            step = lambda n: torch.clamp(i + n, 0, int(top.view(torch.int16))).to(torch.int16).view(dt)
            x = torch.cat([x, -x, step(1), -step(1), step(-1), -step(-1), top[None]])
            x = torch.clamp(x.float(), -float(top), float(top)).to(dt)
            x = torch.nn.functional.pad(x, (0, 64 * 64 - x.numel())).reshape(64, 64)
            a = ops.act8_pack(x.cuda())
            codes, s, val = law(x)
            assert torch.equal(a.scales.cpu(), s), (dt, top)
            assert torch.equal(a.codes.cpu(), codes), (dt, top)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dt", DTYPES)
def test_a_tile_that_is_not_finite_comes_back_as_nan(dt, bad):
    from imfvideo_amd import ops
    x = torch.randn(130, 200).to(dt)
    x[70, 3] = bad
    y = ops.act8_unpack(ops.act8_pack(x.cuda()), dt).cpu()
    assert torch.isnan(y[64:128, :64]).all()
    y[64:128, :64] = 0
    assert torch.isfinite(y).all()
    dw = ops.linear_wgrad8(torch.ones(130, 8, device="cuda", dtype=dt), ops.act8_pack(x.cuda()))
    assert torch.isnan(dw[:, :64]).all() and torch.isfinite(dw[:, 64:]).all()


def gate64(g, u, beta, lb):
    """(situ, sat, the two terms of situ', sat') in float64."""
    t, s = torch.tanh(g / beta), torch.sigmoid(g)
    slope = (s / torch.cosh(g / beta).square(), beta * t * s * torch.sigmoid(-g))
    if lb is None:
        return beta * t * s, u, slope, torch.ones_like(u)
    return beta * t * s, lb * torch.tanh(u / lb), slope, 1 / torch.cosh(u / lb).square()


# Past g of about -87 the sigmoid is below fp32's smallest normal 2^-126, which the hardware's
# exp2 and reciprocal flush to zero: what it multiplies, at most beta lb = 100 times the
# gradients of the tests (below 8), bounds what is lost.
FLUSHED = 100 * 8 * 2.0 ** -126


def within(got, want, dt, mag=None):
    got, u = got.double().cpu(), torch.finfo(dt).eps / 2
    mag = want.abs() if mag is None else mag
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps + FLUSHED
    err, tol = (got - want).abs(), u * want.abs() + CHAIN * mag + tiny
    assert (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lb", [25.0, None])
@pytest.mark.parametrize("shape", [(1, 1), (65, 63), (274, 1365), (128, 512), (200, 2047)])
def test_gate_forward_backward(shape, lb, dt):
    from imfvideo_amd import ops
    print("[case]", shape, lb, dt, flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    scale = 10.0 ** (2 * torch.rand(shape[1], generator=g) - 1)  # 0.1 to 10, both saturations
    gate = (torch.randn(*shape, generator=g) * scale).to(dt)
    up = (torch.randn(*shape, generator=g) * scale.flip(0)).to(dt)
    dh = torch.randn(*shape, generator=g).to(dt)
    h, g8, u8 = ops.situ8_fwd(gate.cuda(), up.cuda(), 4.0, lb)
    situ, sat, _, _ = gate64(gate.double(), up.double(), 4.0, lb)
    within(h, situ * sat, dt)
    for a, x in ((g8, gate), (u8, up)):
        codes, s, _ = law(x)
        assert torch.equal(a.codes.cpu(), codes) and torch.equal(a.scales.cpu(), s)
    dg, du, h2 = ops.situ8_bwd(dh.cuda(), g8, u8, 4.0, lb, with_h=True)
    only = ops.situ8_bwd(dh.cuda(), g8, u8, 4.0, lb)
    assert torch.equal(only[0], dg) and torch.equal(only[1], du) and len(only) == 2
    gv, uv = law(gate)[2].double(), law(up)[2].double()
    situ, sat, (t1, t2), dsat = gate64(gv, uv, 4.0, lb)
    d = dh.double()
    within(h2, situ * sat, dt)
    within(du, d * situ * dsat, dt)
    within(dg, d * sat * (t1 + t2), dt, (d * sat).abs() * (t1.abs() + t2.abs()))


def test_gate_small_and_far_values():
    """Values whose tanh is linear (the series), saturated ones, zeros and signed ones."""
    from imfvideo_amd import ops
    for dt in DTYPES:
        mags = torch.tensor([0.0, 1e-7, 1e-5, 1e-4, 1e-3, 0.01, 0.05, 0.0624, 0.0626, 0.5, 3.0,
                             12.0, 40.0, 88.0, 200.0, 6e4])
        for m in mags:  # one magnitude per tile, so the 8-bit values are near it
            g = (m * (0.5 + 0.5 * torch.rand(64, 64)) * torch.randn(64, 64).sign()).to(dt)
            u = (m * (0.5 + 0.5 * torch.rand(64, 64)) * torch.randn(64, 64).sign()).to(dt)
            h, g8, u8 = ops.situ8_fwd(g.cuda(), u.cuda(), 4.0, 25.0)
            situ, sat, _, _ = gate64(g.double(), u.double(), 4.0, 25.0)
            within(h, situ * sat, dt)
            dh = torch.randn(64, 64).to(dt)
            dg, du = ops.situ8_bwd(dh.cuda(), g8, u8, 4.0, 25.0)
            situ, sat, (t1, t2), dsat = gate64(law(g)[2].double(), law(u)[2].double(), 4.0, 25.0)
            d = dh.double()
            # fp32's exp arguments of up to 2^8 carry 2^-16, its smallest normal 2^-126
            far = 2.0 ** -15 if m > 40 else 0.0
            within(dg, d * sat * (t1 + t2), dt, (1 + far / CHAIN) * (d * sat).abs() * (t1.abs() + t2.abs()))
            within(du, d * situ * dsat, dt, (1 + far / CHAIN) * (d * situ * dsat).abs())


def test_gate_views_and_odd_strides():
    from imfvideo_amd import ops
    x = torch.randn(100, 2 * 77 + 3, device="cuda").half()
    gate, up = x[:, 1:78], x[:, 79:156]
    h, g8, u8 = ops.situ8_fwd(gate, up, 4.0, 25.0)
    h2, *a = ops.situ8_fwd(gate.contiguous(), up.contiguous(), 4.0, 25.0)
    assert torch.equal(h, h2)
    assert all(torch.equal(p, q) for m, n in zip((g8, u8), a) for p, q in zip(m[:2], n[:2]))
    dh = torch.randn(77, 100, device="cuda").half().t()
    one = torch.randn(1, 77, device="cuda").half().expand(100, 77)
    for d in (dh, one):
        for p, q in zip(ops.situ8_bwd(d, g8, u8, 4.0, 25.0),
                        ops.situ8_bwd(d.contiguous(), g8, u8, 4.0, 25.0)):
            assert torch.equal(p, q)


# rows, M, N: one of each; edges of the 64-row stages and the 128-wide tiles; odd widths
# (rows off 16 bytes); several ranges of rows; more than one column tile of codes past the edge
WG = [(1, 1, 1), (64, 128, 64), (65, 8, 130), (274, 160, 512), (1042, 160, 512), (700, 1365, 512),
      (5000, 130, 65), (333, 77, 1365), (4159, 512, 2048), (20000, 24, 40)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", WG)
def test_weight_gradient(shape, dt):
    from imfvideo_amd import ops
    rows, M, N = shape
    print("[case]", shape, dt, flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(rows, N, generator=g).to(dt)
    dy = (0.1 * torch.randn(rows, M, generator=g)).to(dt)
    a = ops.act8_pack(x.cuda())
    dw = ops.linear_wgrad8(dy.cuda(), a)
    val = law(x)[2].cuda().double()
    d = dy.cuda().double()
    want = d.t().contiguous() @ val
    mag = d.t().abs().contiguous() @ val.abs()
    tol = (128 + -(-rows // 64)) * 2.0 ** -24 * mag + 1e-30
    assert dw.dtype == torch.float32 and dw.shape == (M, N)
    assert ((dw.double() - want).abs() <= tol).all(), ((dw.double() - want).abs() / tol).max().item()
    assert torch.equal(dw, ops.linear_wgrad8(dy.cuda(), a))
    # a band of a wider tensor, aligned and not
    for lo in (8, 3):
        wide = torch.full((rows, M + 40), float("nan"), device="cuda", dtype=dt)
        wide[:, lo:lo + M] = dy.cuda()
        assert torch.equal(ops.linear_wgrad8(wide[:, lo:lo + M], a), dw), lo
    # NaN right behind the last row
    more = torch.full((rows * M + 64,), float("nan"), device="cuda", dtype=dt)
    more[:rows * M] = dy.cuda().reshape(-1)
    assert torch.equal(ops.linear_wgrad8(more[:rows * M].view(rows, M), a), dw)


def test_module_keeps_8_bits_and_its_gradients():
    from imfvideo_amd import ops
    from imfvideo_amd.imf_dit_video import SituAndMul
    x = torch.randn(2, 50, 2 * 96, device="cuda").bfloat16().requires_grad_(True)
    dh = torch.randn(2, 50, 96, device="cuda").bfloat16()
    m = SituAndMul(4.0, 25.0, act8=True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        h = m(x)
    assert sum(t.nbytes for t in kept) == 2 * (2 * 2 * 4096 + 2 * 2 * 4)  # two tiles by two, twice
    g, = torch.autograd.grad(h, x, dh)
    h2, g8, u8 = ops.situ8_fwd(x[..., :96].detach(), x[..., 96:].detach(), 4.0, 25.0)
    assert torch.equal(h, h2)
    assert torch.equal(g, torch.cat(ops.situ8_bwd(dh, g8, u8, 4.0, 25.0), -1))
    with torch.no_grad():
        assert m(x).shape == h.shape
    h = m(x)
    d, = torch.autograd.grad(h.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.float().sum(), x)
    h = m(x)
    with pytest.raises(RuntimeError, match="one gradient at a time"):
        torch.autograd.grad(h, x, torch.ones(3, *h.shape, device="cuda").bfloat16(),
                            is_grads_batched=True)


def mlp_pair(D, Fh, act8=True):
    from imfvideo_amd.imf_dit_video import SwiGLUMlp
    torch.manual_seed(D + Fh)
    m = SwiGLUMlp(D, Fh, situ_beta=4.0, situ_linear_beta=25.0, act8=act8).cuda()
    return m


@pytest.mark.parametrize("D, Fh, L", [(64, 96, 130), (128, 341, 274), (512, 1365, 100)])
def test_mlp_gradients(D, Fh, L):
    """The MLP under bf16 autocast: outputs and gradients against the same chain of 16-bit
    steps in float64 at the kept values (each step's input rounded as the path rounds it)."""
    print("[case]", D, Fh, L, flush=True)
    m = mlp_pair(D, Fh)
    dt = torch.bfloat16
    x = torch.randn(2, L, D, device="cuda").requires_grad_(True)
    dy = torch.randn(2, L, D, device="cuda").to(dt)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        with torch.autocast("cuda", dtype=dt):
            y = m(x)
    assert not any(t.dtype == dt and t.shape[-2:] in ((L, Fh), (2 * L, Fh)) for t in kept)
    grads = torch.autograd.grad(y, [x, m.w1.weight, m.w3.weight, m.w2.weight], dy)
    # the chain again, from the values the path holds
    from imfvideo_amd import ops
    xh = x.detach().to(dt).reshape(-1, D)
    W1, W3, W2 = (w.weight.detach().to(dt) for w in (m.w1, m.w3, m.w2))
    gate, up = xh @ W1.t(), xh @ W3.t()
    h, g8, u8 = ops.situ8_fwd(gate, up, 4.0, 25.0)
    assert torch.equal(y, torch.nn.functional.linear(h, W2).reshape(y.shape))
    d = dy.reshape(-1, D)
    dg, du, hk = ops.situ8_bwd(d @ W2, g8, u8, 4.0, 25.0, with_h=True)
    val = law(xh)[2].cuda().double()
    f = lambda t: t.double()
    R = 2 * L
    for got, A, X in ((grads[1], dg, val), (grads[2], du, val), (grads[3], d, f(hk))):
        want, mag = f(A).t() @ X, f(A).t().abs() @ X.abs()
        tol = (128 + R) * 2.0 ** -24 * mag + 2.0 ** -8 * want.abs() * (got is grads[3]) + 1e-30
        assert ((f(got) - want).abs() <= tol).all()
    dx = f(dg) @ f(W1) + f(du) @ f(W3)
    mag = f(dg).abs() @ f(W1).abs() + f(du).abs() @ f(W3).abs()
    # two products rounded to bf16 and their sum once more
    tol = 2.0 ** -8 * ((f(dg) @ f(W1)).abs() + (f(du) @ f(W3)).abs() + dx.abs()) * 1.01
    tol = tol + Fh * 2.0 ** -23 * mag
    assert ((f(grads[0]).reshape(-1, D) - dx).abs() <= tol).all()


def test_block_with_dense_attention_and_8_bit_activations():
    """The two together in a TransformerBlock: it runs, every parameter gets a finite
    gradient, and the output equals the block's without 8-bit activations to a rounding (only
    the backward reads them; the gate's h may round differently)."""
    from imfvideo_amd.imf_dit_video import (TransformerBlock, dense_attention,
                                            precompute_axial_rope_3d)
    torch.manual_seed(2)
    mk = lambda a: TransformerBlock(128, 2, 64, 32, 32, 32, 64, attn_impl=dense_attention,
                                    act8=a).cuda()
    a, b = mk(True), mk(False)
    with torch.no_grad():
        a.attn_scale.fill_(0.5), a.mlp_scale.fill_(0.5)
    b.load_state_dict(a.state_dict())
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(32, (2, 8, 8), 18))
    x = torch.randn(2, 146, 128, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ya, yb = a(x, cos, sin), b(x, cos, sin)
    assert (ya - yb).abs().max() <= 2.0 ** -6 * yb.abs().max()
    ya.square().mean().backward()
    for n, p in a.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), n
    assert torch.isfinite(x.grad).all()


def test_mlp_falls_back_with_hooks_and_without_gradients():
    m = mlp_pair(64, 96)
    x = torch.randn(3, 64, device="cuda").bfloat16().requires_grad_(True)
    seen = []
    m.w1.register_forward_hook(lambda *a: seen.append(1))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    assert seen and torch.isfinite(torch.autograd.grad(y.float().sum(), x)[0]).all()
    m = mlp_pair(64, 96)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.isfinite(m(x)).all()


def test_graph_replays_match_eager():
    from imfvideo_amd import ops
    gate, up, dh = (torch.randn(700, 200, device="cuda").half() for _ in range(3))

    def step():
        h, g8, u8 = ops.situ8_fwd(gate, up, 4.0, 25.0)
        dg, du = ops.situ8_bwd(dh, g8, u8, 4.0, 25.0)
        a = ops.act8_pack(h)
        return [h, dg, du, ops.linear_wgrad8(dg, a), ops.act8_unpack(a, torch.float16)]

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
    for _ in range(4):
        for t in (gate, up, dh):
            t.copy_(torch.randn(t.shape, device="cuda") * 2)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)

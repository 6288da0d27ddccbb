"""Orthogonalised updates (ops.orthogonalize, Muon) on the GPU against float64.

The kernels' pairs of fp16 numbers carry 22 bits and a sign where fp32 has 24 (a factor of two at
most in what a value is off), and their products leave lo lo out (2^-24 again, as much as an
fp32 product's rounding): a result may be off by four times as much as the same steps in fp32
are (on the CPU), and by the rounding of its own type.  fp32's own error may happen to be
nothing, most easily where a matrix is a single value: it counts as a rounding of each of the
last step's three terms at least, which at a singular value of 1 are |a| + |b| + |c| = 10 times
2^-24 of a result of about 1 (0.7 to 1.2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFS = (3.4445, -4.7750, 2.0315)


def exact(g, steps=5, coeffs=COEFFS, dtype=torch.float64):
    """The steps in float64 (or fp32) on the host."""
    rows = [coeffs] * steps if isinstance(coeffs[0], float) else coeffs
    x = g.cpu().to(dtype)
    turn = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if turn else x
    n = x.double().square().sum((-1, -2), keepdim=True).sqrt()
    x = (x.double() / torch.where(n > 0, n, torch.ones_like(n))).to(dtype)
    for a, b, c in rows:
        A = x @ x.transpose(-1, -2)
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.transpose(-1, -2) if turn else x


def check(got, g, what, steps=5, coeffs=COEFFS):
    """2-norm of the error of each matrix."""
    want = exact(g, steps, coeffs)
    fp32 = (exact(g, steps, coeffs, torch.float32).double() - want)
    assert got.dtype == g.dtype and got.shape == g.shape and torch.isfinite(got).all(), what
    u = 0.0 if g.dtype == torch.float32 else torch.finfo(g.dtype).eps / 2
    norm = lambda t: t.reshape(-1, t.shape[-2] * t.shape[-1]).norm(dim=1)
    err = norm(got.cpu().double() - want)
    last = sum(map(abs, coeffs if isinstance(coeffs[0], float) else coeffs[-1]))
    tol = 4 * (norm(fp32) + last * 2.0 ** -24 * norm(want)) + u * norm(want)
    print("[ratio]", what, (err / tol.clamp_min(1e-300)).max().item(), flush=True)
    assert (err <= tol).all(), (what, (err / tol).max().item())


def matrices(seed, n, R, C, dt=torch.float32, rank=None):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = rn(n, R, C) if rank is None else rn(n, R, rank) @ rn(n, rank, C) + 1e-3 * rn(n, R, C)
    return (1e-3 * x).to(dt).cuda()


@pytest.mark.parametrize("R,C", [(1, 1), (1, 7), (9, 1), (16, 16), (31, 33), (63, 65), (64, 64),
                                 (65, 64), (128, 64), (129, 200), (160, 512), (512, 160),
                                 (512, 512), (300, 1365), (1365, 512), (64, 4096), (700, 701)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_shapes(R, C, dt):
    from imfvideo_amd import ops
    for n in (1, 3):
        g = matrices(R + C, n, R, C, dt)
        check(ops.orthogonalize(g), g, (R, C, dt, n))


@pytest.mark.parametrize("n,R,C", [(20, 512, 512), (64, 100, 140), (6, 512, 2048)])
def test_many_matrices_are_each_its_own(n, R, C):
    """Tiles of 128 and of 64 rows, and a matrix's place among the others, give the same bits."""
    from imfvideo_amd import ops
    g = matrices(n, n, R, C)
    x = ops.orthogonalize(g)
    check(x, g, (n, R, C))
    for i in (0, n // 2, n - 1):
        assert torch.equal(ops.orthogonalize(g[i]), x[i])


def test_the_other_side_up_is_the_transpose():
    from imfvideo_amd import ops
    g = matrices(1, 2, 150, 333)
    assert torch.equal(ops.orthogonalize(g.transpose(1, 2)), ops.orthogonalize(g).transpose(1, 2))
    assert torch.equal(ops.orthogonalize(g.unflatten(0, (1, 2)))[0], ops.orthogonalize(g))


@pytest.mark.parametrize("rank", [1, 5, 40])
def test_nearly_low_rank(rank):
    from imfvideo_amd import ops
    g = matrices(rank, 2, 256, 384, rank=rank)
    check(ops.orthogonalize(g), g, rank)


def test_steps_with_coefficients_of_their_own():
    from imfvideo_amd import ops
    g = matrices(3, 2, 96, 128)
    rows = [(2.0, -1.5, 0.5)] * 3 + [(1.875, -1.25, 0.375)] * 4
    check(ops.orthogonalize(g, 7, rows), g, "rows", 7, rows)
    check(ops.orthogonalize(g, 1), g, "one", 1)
    # 20 steps of the map whose fixed point is 1: orthogonal to fp32's accuracy
    x = ops.orthogonalize(g, 20, (1.875, -1.25, 0.375)).double()
    eye = torch.eye(96, device="cuda", dtype=torch.float64)
    assert (x @ x.transpose(1, 2).contiguous() - eye).abs().max() < 1e-5


def test_scales_and_zeros():
    """The result does not depend on the scale, down and up to fp32's ends; zeros stay."""
    from imfvideo_amd import ops
    g = matrices(4, 1, 80, 112)
    want = ops.orthogonalize(g)
    for e in (-100, -60, 60, 120):
        assert torch.equal(ops.orthogonalize(g * 2.0 ** e), want), e
    z = torch.cat([g, torch.zeros_like(g), g])
    got = ops.orthogonalize(z)
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[0])


def test_a_matrix_that_is_not_finite_is_nan_and_alone():
    from imfvideo_amd import ops
    g = matrices(5, 3, 80, 112)
    want = ops.orthogonalize(g)
    for bad in (float("nan"), float("inf")):
        h = g.clone()
        h[1, 3, 5] = bad
        got = ops.orthogonalize(h)
        assert got[1].isnan().all()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_streams_graphs_and_views():
    from imfvideo_amd import ops
    g = matrices(6, 4, 200, 300)
    want = ops.orthogonalize(g)
    wide = torch.zeros(4, 203, 601, device="cuda")
    wide[:, 3:, 1::2] = g
    assert torch.equal(ops.orthogonalize(wide[:, 3:, 1::2]), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.orthogonalize(g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            kept = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for _ in range(3):
        kept.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want)
        assert torch.equal(ops.orthogonalize(g), want)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_steps_as_its_formula(dt, nesterov):
    """Three steps of matrices of several shapes, some without a gradient, against float64."""
    from imfvideo_amd.muon import Muon
    torch.manual_seed(7)
    shapes = [(64, 96), (64, 96), (160, 64), (33, 7)]
    ps = [torch.nn.Parameter((0.05 * torch.randn(s)).to(dt).cuda()) for s in shapes]
    opt = Muon([dict(params=ps[:2], lr=0.01), dict(params=ps[2:])], lr=0.02, weight_decay=0.1,
               nesterov=nesterov)
    w = [p.detach().double().cpu() for p in ps]
    buf = [torch.zeros_like(x) for x in w]
    # each step rounds a weight once; the update is off by its fp32 error (below 1e-4 of it)
    tol = [torch.zeros_like(x) for x in w]
    u = torch.finfo(dt).eps / 2
    for it in range(3):
        for i, p in enumerate(ps):
            p.grad = None if i == 1 and it == 1 else (1e-3 * torch.randn(shapes[i])).to(dt).cuda()
        opt.step()
        for i, p in enumerate(ps):
            if p.grad is None:
                continue
            g = p.grad.double().cpu()
            buf[i] = 0.95 * buf[i] + g
            lr = 0.01 if i < 2 else 0.02
            x = exact((g + 0.95 * buf[i] if nesterov else buf[i]))
            d = lr * 0.2 * max(shapes[i]) ** 0.5 * x
            w[i] = (1 - lr * 0.1) * w[i] - d
            tol[i] += 2 * u * (w[i].abs() + d.abs()) + 1e-4 * d.abs().max() + 2.0 ** -23 * w[i].abs()
    for i, p in enumerate(ps):
        assert ((p.detach().double().cpu() - w[i]).abs() <= tol[i]).all(), i


def test_offsets_past_32_bits():
    """66 matrices of 2^24 elements, 4.4 GB: each is as it is alone."""
    from imfvideo_amd import ops
    g = torch.empty(66, 4096, 4096, device="cuda")
    for i in (0, 63, 64, 65):
        g[i] = torch.randn(4096, 4096, device="cuda")
    g[1:63] = g[0]
    x = ops.orthogonalize(g, steps=1)
    for i in (0, 62, 63, 65):
        assert torch.equal(ops.orthogonalize(g[i], steps=1), x[i]), i


def test_float64_weights_take_the_eager_products():
    from imfvideo_amd.muon import Muon
    p = torch.nn.Parameter(torch.randn(20, 30, device="cuda", dtype=torch.float64))
    w, g = p.detach().clone(), torch.randn_like(p)
    p.grad = g
    Muon([p], lr=0.1, nesterov=False).step()
    want = w.cpu() - 0.1 * 0.2 * 30 ** 0.5 * exact(g.cpu())
    assert (p.detach().cpu() - want).abs().max() < 1e-9


@pytest.mark.parametrize("n,R,C", [(3, 130, 2100), (40, 512, 512), (2, 2050, 2049), (1, 192, 5000),
                                   (9, 320, 1000)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_forms_on_both_sides_of_the_tile_rule(n, R, C, dt):
    from imfvideo_amd import ops
    g = matrices(n, n, R, C).to(dt)
    check(ops.orthogonalize(g, steps=2), g, (n, R, C, dt), steps=2)
    if R != C:  # (of a square matrix the rows are contracted whichever way it stands)
        t = g.transpose(-1, -2).contiguous()
        assert torch.equal(ops.orthogonalize(t, steps=2),
                           ops.orthogonalize(g, steps=2).transpose(-1, -2))

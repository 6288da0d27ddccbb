"""SwiGLUMlp(act8=True) in the ways that a program trains it: both 16-bit types, weights in 32 or
16 bits, frozen weights and inputs, views, whole blocks' gradients, graphs.

Tolerances: the chain of 16-bit steps is repeated from the values that the path holds, so each
product is compared on the same operands: fp32 sums of R products are off by (128 + R) 2^-24 of
their magnitudes, and a result rounded to 16 bits by u = eps / 2 of it."""
import pytest
import torch

from tests.test_gpu_act8 import law

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def mlp(D, Fh, act8=True, lb=25.0, dtype=torch.float32):
    from imfvideo_amd.imf_dit_video import SwiGLUMlp
    torch.manual_seed(D + Fh)
    return SwiGLUMlp(D, Fh, situ_beta=4.0, situ_linear_beta=lb, act8=act8).cuda().to(dtype)


def call(m, x, dt, auto):
    with torch.autocast("cuda", dtype=dt, enabled=auto):
        return m(x)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("auto", [True, False])
@pytest.mark.parametrize("D, Fh, L, lb", [(64, 96, 130, 25.0), (96, 341, 77, None)])
def test_gradients_by_type(D, Fh, L, lb, auto, dt):
    """Under autocast with fp32 weights, and with 16-bit weights and input."""
    from imfvideo_amd import ops
    print("[case]", D, Fh, L, lb, auto, dt, flush=True)
    wt = torch.float32 if auto else dt
    m = mlp(D, Fh, lb=lb, dtype=wt)
    x = torch.randn(2, L, D, device="cuda").to(wt).requires_grad_(True)
    dy = torch.randn(2, L, D, device="cuda").to(dt)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = call(m, x, dt, auto)
    assert any(t.dtype == torch.int8 for t in kept)  # the 8-bit form ran
    assert not any(t.dtype == dt and t.numel() in (2 * L * Fh, 2 * L * D) for t in kept)
    leaves = [x, m.w1.weight, m.w3.weight, m.w2.weight]
    grads = torch.autograd.grad(y, leaves, dy)
    assert [g.dtype for g in grads] == [t.dtype for t in leaves]
    xh = x.detach().to(dt).reshape(-1, D)
    W1, W3, W2 = (w.weight.detach().to(dt) for w in (m.w1, m.w3, m.w2))
    lin = torch.nn.functional.linear
    h, g8, u8 = ops.situ8_fwd(lin(xh, W1), lin(xh, W3), 4.0, lb)
    assert torch.equal(y.reshape(-1, D), lin(h, W2))
    d = dy.reshape(-1, D)
    dg, du, hk = ops.situ8_bwd(d @ W2, g8, u8, 4.0, lb, with_h=True)
    val = law(xh)[2].cuda().double()
    f, u = lambda t: t.double(), torch.finfo(dt).eps / 2
    R, tiny = 2 * L, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    turn = lambda t: f(t).t().contiguous()
    for got, A, X in ((grads[1], dg, val), (grads[2], du, val), (grads[3], d, f(hk))):
        want, mag = turn(A) @ X, turn(A).abs() @ X.abs()
        # in 16 bits where the weight is (w2's product may round to them on its way, too)
        rounded = 0.0 if got.dtype == torch.float32 and got is not grads[3] else u
        tol = (128 + R) * 2.0 ** -24 * mag + rounded * want.abs() + tiny
        assert ((f(got) - want).abs() <= tol).all()
    a, b = f(dg) @ f(W1), f(du) @ f(W3)
    mag = f(dg).abs() @ f(W1).abs() + f(du).abs() @ f(W3).abs()
    tol = u * (a.abs() + b.abs() + (a + b).abs()) * 1.01 + Fh * 2.0 ** -23 * mag + 3 * tiny
    assert ((f(grads[0]).reshape(-1, D) - a - b).abs() <= tol).all()


@pytest.mark.parametrize("on", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0),
                                (0, 1, 1, 1)])
def test_frozen_weights_and_inputs(on):
    """What is asked for has the bits that it has when everything is; the rest gets nothing."""
    m = mlp(64, 96)
    x = torch.randn(3, 70, 64, device="cuda")
    dy = torch.randn(3, 70, 64, device="cuda").bfloat16()
    leaves = lambda: [xi, m.w1.weight, m.w3.weight, m.w2.weight]
    res = []
    for want in ((1, 1, 1, 1), on):
        xi = x.clone()
        for t, r in zip(leaves(), want):
            t.grad = None
            t.requires_grad_(bool(r))
        call(m, xi, torch.bfloat16, True).backward(dy)
        res.append([t.grad for t in leaves()])
    for full, got, r in zip(*res, on):
        assert (torch.equal(got, full) if r else got is None)


def test_an_expanded_gradient_and_a_strided_input():
    """A sum's gradient has no storage of its own; the input is a band of a wider tensor."""
    m = mlp(64, 96)
    wide = torch.randn(5, 40, 200, device="cuda").bfloat16()
    a = wide[..., 30:94].requires_grad_(True)
    b = a.detach().contiguous().requires_grad_(True)
    ga, = torch.autograd.grad(call(m, a, torch.bfloat16, True).sum(), a)
    y = call(m, b, torch.bfloat16, True)
    gb, = torch.autograd.grad(y, b, torch.ones_like(y))
    assert torch.equal(ga, gb)


def test_forward_mode_takes_the_layers_one_by_one():
    """The 8-bit form is one of reverse mode: a tangent is refused or carried, never dropped."""
    import torch.autograd.forward_ad as fw
    m = mlp(64, 96)
    with fw.dual_level():
        x = fw.make_dual(torch.randn(4, 64, device="cuda").bfloat16(),
                         torch.randn(4, 64, device="cuda").bfloat16())
        try:
            y = call(m, x, torch.bfloat16, True)
        except NotImplementedError:
            return
        assert fw.unpack_dual(y).tangent is not None


@pytest.mark.parametrize("dt", DTYPES)
def test_a_blocks_gradients(dt):
    """A TransformerBlock over dense_attention with 8-bit activations against the same block
    without: the gradients of a loss differ by what the 8 bits hold less.  A code is off by
    half a step of a tile whose largest value is 127 steps: for the projections of normalised
    rows (tiles within about six standard deviations) at most 6 / 254 = 2.4 % of a standard
    deviation and 1 / sqrt(12) of a step = 1.4 % of it in the mean square, in the gate, the
    up branch and the input each; the slopes of the gate are below 1.1 and their own below 1: at most
    10 % of the 2-norm of the MLP's gradients with the 16-bit roundings of both blocks, and of the
    ones behind it, which take it as a part."""
    from imfvideo_amd.imf_dit_video import (TransformerBlock, dense_attention,
                                            precompute_axial_rope_3d)
    torch.manual_seed(3)
    make = lambda a: TransformerBlock(128, 2, 64, 32, 32, 32, 64, attn_impl=dense_attention,
                                      act8=a).cuda()
    a, b = make(True), make(False)
    with torch.no_grad():
        a.attn_scale.fill_(0.5), a.mlp_scale.fill_(0.5)
    b.load_state_dict(a.state_dict())
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(32, (2, 8, 8), 18))
    x = torch.randn(2, 146, 128, device="cuda")
    dy = torch.randn(2, 146, 128, device="cuda")
    res = []
    for m in (a, b):
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=dt):
            y = m(xi, cos, sin)
        y.backward(dy)
        res.append([("x", xi.grad)] + [(n, p.grad) for n, p in m.named_parameters()])
    for (n, s), (_, t) in zip(*res):
        off = ((s - t).norm() / t.norm()).item()
        print("[off]", n, round(off, 5), flush=True)
        assert torch.isfinite(s).all() and t.any() and off <= 0.1, n


@pytest.mark.parametrize("dt", DTYPES)
def test_training_steps_in_a_graph(dt):
    """Forward and backward of the 8-bit MLP captured, replayed on refilled inputs."""
    m = mlp(64, 341)
    x, dy = (torch.randn(2, 130, 64, device="cuda").to(dt) for _ in range(2))

    def step():
        xi = x.detach().requires_grad_(True)
        # (no cache of cast weights: a graph keeps what it captured)
        with torch.autocast("cuda", dtype=dt, cache_enabled=False):
            y = m(xi)
        return [y.detach(), *torch.autograd.grad(y, [xi, m.w1.weight, m.w3.weight, m.w2.weight], dy)]

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
    for _ in range(3):
        for t in (x, dy):
            t.copy_(torch.randn(t.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for s, t in zip(out, step()):
            assert torch.equal(s, t)
        torch.cuda.synchronize()

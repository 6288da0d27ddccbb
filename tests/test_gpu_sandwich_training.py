"""Differential attention, the norms around the residual stream and orthogonalised updates together: blocks
that train with them, eagerly and as one captured step."""
from functools import partial

import pytest
import torch

pytestmark = pytest.mark.gpu


def model(seed):
    from imfvideo_amd.imf_dit_video import DiffAttentionImpl, TransformerBlock
    torch.manual_seed(seed)
    m = torch.nn.ModuleList(
        TransformerBlock(128, 4, 64, 64, 32, 32, 64, sandwich_norm=True,
                         attn_impl=partial(DiffAttentionImpl, num_heads=4)) for _ in range(2)).cuda()
    for b in m:
        torch.nn.init.normal_(b.attn_scale), torch.nn.init.normal_(b.mlp_scale)
    return m


def optimizers(m):
    from imfvideo_amd.muon import Muon, matrix_parameters
    mats, rest = matrix_parameters(m)
    return Muon(mats, lr=0.02, weight_decay=0.1), torch.optim.SGD(rest, lr=1e-3)


def step(m, opts, x, cos, sin, gates, dy):
    for o in opts:
        o.zero_grad(set_to_none=True)
    with torch.autocast("cuda", torch.bfloat16):
        y = x
        for b in m:
            y = b(y, cos, sin, gates)
    y.backward(dy)
    for o in opts:
        o.step()
    return y.detach()


def inputs():
    from imfvideo_amd.imf_dit_video import precompute_axial_rope_3d
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(32, (4, 4, 4), 2))
    x, dy = torch.randn(2, 66, 128, device="cuda"), torch.randn(2, 66, 128, device="cuda")
    gates = tuple(1 + 0.1 * torch.randn(2, 128, device="cuda") for _ in range(2))
    return x, cos, sin, gates, dy


def test_a_captured_step_is_the_eager_one():
    """Three steps from the same weights, eagerly and as replays of one graph: the same bits in
    every weight and momentum."""
    torch.manual_seed(1)
    data = inputs()
    eager, graphed = model(2), model(2)
    oe, og = optimizers(eager), optimizers(graphed)
    start = [p.detach().clone() for p in graphed.parameters()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once eagerly: the momenta exist, nothing of the graph lives on
        step(graphed, og, *data)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for o in og:
        o.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed, og, *data)
    with torch.no_grad():
        for p, s in zip(graphed.parameters(), start):
            p.copy_(s)
        for state in og[0].state.values():
            state["momentum_buffer"].zero_()
    for it in range(3):
        for t in (data[0], data[4]):
            t.copy_(torch.randn(t.shape, device="cuda"))
        want = step(eager, oe, *data)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), it
        for (n, a), b in zip(eager.named_parameters(), graphed.parameters()):
            assert torch.equal(a, b), (it, n)
    for a, b in zip(oe[0].state.values(), og[0].state.values()):
        assert torch.equal(a["momentum_buffer"], b["momentum_buffer"])
    for p, s in zip(graphed.parameters(), start):
        assert torch.isfinite(p).all() and not torch.equal(p, s)


def test_a_block_is_its_operators_one_after_the_other():
    """The block's output from its layers and the two entry points, called by hand."""
    from imfvideo_amd.imf_dit_video import residual_norm
    torch.manual_seed(3)
    x, cos, sin, gates, _ = inputs()
    b = model(4)[0]
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        got = b(x, cos, sin, gates)
        a = b.attn(b.norm1(x).to(torch.bfloat16), cos, sin)
        y, n = residual_norm(x, a, b.attn_scale, b.attn_post_norm.weight, gate=gates[0],
                             pre_weight=b.norm2.weight, eps=b.norm2.eps)
        want, = residual_norm(y, b.mlp(n), b.mlp_scale, b.mlp_post_norm.weight, gate=gates[1],
                              eps=b.mlp_post_norm.eps)
    assert torch.equal(got, want)


def test_gradients_of_the_block_are_the_differences():
    """A directional derivative of a block in fp32, its attention's operands in fp16, against central
    differences of the same block: the output is rounded to 2^-11 of its size, so that differences of
    size h carry an error of about 2^-11 |y| sqrt(n) / h, and the curvature's of h^2."""
    torch.manual_seed(5)
    x, cos, sin, gates, dy = inputs()
    b = model(6)[0]

    def f(t):
        with torch.autocast("cuda", torch.float16):
            return b(t, cos, sin, gates)
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(f(leaf), leaf, dy)
    d = g / g.square().mean().sqrt()  # along the gradient, of size 1
    h = 0.02
    with torch.no_grad():
        up, down = f(x + h * d).double(), f(x - h * d).double()
        size = f(x).double().abs().max()
    diff = ((up - down) / (2 * h) * dy.double()).sum().item()
    got = (g.double() * d.double()).sum().item()
    # roundings: independent, each 2^-11 of the largest at most, a dozen layers; curvature: of h^2
    # times a third derivative that the norms bound by the value over the rows' size of 1
    scale = (g.double().norm() * d.double().norm()).item()
    tol = 12 * 2.0 ** -11 * size.item() * dy.double().norm().item() / (2 * h) + 10 * h * h * scale
    assert abs(diff - got) <= tol, (diff, got, tol)
    assert tol <= 0.2 * abs(got), "a bound that says something"

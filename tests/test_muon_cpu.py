"""Muon and the orthogonalised update on the host: formula, refusals, parameters, state."""
import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import TransformerBlock
from imfvideo_amd.muon import Muon, matrix_parameters, newton_schulz


def test_newton_schulz_keeps_singular_vectors():
    """p(p(..(s))) of each singular value, whichever side is shorter."""
    torch.manual_seed(1)
    for shape in ((2, 5, 9), (9, 5), (4, 4), (1, 6)):
        g = torch.randn(*shape, dtype=torch.float64)
        U, s, V = torch.linalg.svd(g, full_matrices=False)
        s = s / s.square().sum(-1, keepdim=True).sqrt()
        for _ in range(5):
            s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
        want = U @ torch.diag_embed(s) @ V
        assert torch.allclose(newton_schulz(g), want, atol=1e-9)
        rows = [(3.4445, -4.7750, 2.0315)] * 5
        assert torch.equal(newton_schulz(g, 5, rows), newton_schulz(g))
    assert torch.equal(newton_schulz(torch.zeros(3, 4)), torch.zeros(3, 4))


def test_muon_on_the_host():
    torch.manual_seed(2)
    w = torch.nn.Parameter(torch.randn(6, 4))
    v = w.detach().clone()
    opt = Muon([w], lr=0.1, weight_decay=0.5, momentum=0.9)
    buf = torch.zeros_like(v)
    for _ in range(3):
        w.grad = torch.randn(6, 4)
        assert opt.step(lambda: 3) == 3
        buf = 0.9 * buf + w.grad
        v = v * 0.95 - 0.1 * 0.2 * 6 ** 0.5 * newton_schulz(w.grad + 0.9 * buf)
        assert torch.allclose(w, v, rtol=1e-5, atol=1e-6)
    # its state goes through a state dict
    w2 = torch.nn.Parameter(w.detach().clone())
    opt2 = Muon([w2], lr=0.1)
    opt2.load_state_dict(opt.state_dict())
    w2.grad = w.grad.clone()
    opt.step(), opt2.step()
    assert torch.equal(w, w2)


def test_a_loaded_momentum_stays_fp32():
    """Of 16-bit weights too, and apart from the one that it was loaded from."""
    torch.manual_seed(3)
    ws = [torch.nn.Parameter(torch.randn(6, 4).bfloat16()) for _ in range(2)]
    opts = [Muon([w], lr=0.1) for w in ws]
    ws[1].data.copy_(ws[0].data)
    ws[0].grad = torch.randn(6, 4).bfloat16()
    opts[0].step()
    opts[1].load_state_dict(opts[0].state_dict())
    a, b = (o.state[w]["momentum_buffer"] for o, w in zip(opts, ws))
    assert a.dtype == b.dtype == torch.float32 and torch.equal(a, b)
    assert a.data_ptr() != b.data_ptr()


def test_matrices_of_a_block():
    m = TransformerBlock(64, 1, 32, 32, 32, 32, 64, sandwich_norm=True)
    m.register_parameter("alpha_logit", torch.nn.Parameter(torch.zeros(1, 2)))
    m.norm1.weight.requires_grad_(False)
    mats, rest = matrix_parameters(m)
    names = {id(p): n for n, p in m.named_parameters()}
    assert {names[id(p)] for p in mats} == {n for n in names.values() if n.endswith("_proj.weight")
                                            or n.startswith("mlp.w")}
    assert "alpha_logit" in {names[id(p)] for p in rest}
    assert len(mats) + len(rest) == len(names) - 1


def test_refusals():
    p = torch.nn.Parameter(torch.randn(3, 4))
    for bad in (torch.nn.Parameter(torch.randn(3)), torch.nn.Parameter(torch.randn(2, 3, 4))):
        with pytest.raises(ValueError, match="matrices only"):
            Muon([p, bad])
    for kw in (dict(lr=-1), dict(weight_decay=-1), dict(momentum=1.0), dict(rms=0.0)):
        with pytest.raises(ValueError, match="Muon"):
            Muon([p], **kw)
    for steps, c in ((0, ops.NS_COEFFS), (65, ops.NS_COEFFS), (2, [(1.0, 2.0, 3.0)]),
                     (1, (1.0, 2.0)), (1, (1.0, float("nan"), 0.0))):
        with pytest.raises(ValueError, match="orthogonalize"):
            Muon([p], ns_steps=steps, ns_coeffs=c)
        with pytest.raises(ValueError, match="orthogonalize"):
            newton_schulz(torch.randn(3, 3), steps, c)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.orthogonalize(torch.randn(3, 3))


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def test_operands_that_the_kernels_do_not_take():
    gpu = lambda t: t.as_subclass(_Gpu)
    with pytest.raises(TypeError, match="orthogonalize"):
        ops.orthogonalize(gpu(torch.randn(3, 3, dtype=torch.float64)))
    with pytest.raises(ValueError, match="orthogonalize"):
        ops.orthogonalize(gpu(torch.randn(3)))
    with pytest.raises(ValueError, match="too large"):
        ops.orthogonalize(gpu(torch.empty(1, 32769)))
    lib = _lib.load()
    size = lib.sla2h_orthogonalize_workspace_bytes
    assert size(1, 1, 1) > 0 and size(3, 32768, 32768) > 0
    for n, R, C in ((0, 4, 4), (1, 0, 4), (1, 4, 0), (1, 32769, 4), (2 ** 28, 4, 4)):
        assert size(n, R, C) == 0
        assert lib.sla2h_orthogonalize(16, 2, n, R, C, 1, ops._ns_coeffs(1, ops.NS_COEFFS), 16, 16,
                                       None) == 1
    for dtype, steps, ws in ((3, 1, 16), (2, 0, 16), (2, 65, 16), (2, 1, 8), (2, 1, None)):
        assert lib.sla2h_orthogonalize(16, dtype, 1, 4, 4, steps, ops._ns_coeffs(1, ops.NS_COEFFS),
                                       ws, 16, None) == 1


def test_sides_past_the_kernels():
    with pytest.raises(ValueError, match="32,768"):
        Muon([torch.nn.Parameter(torch.zeros(32769, 1))])
    Muon([torch.nn.Parameter(torch.zeros(32768, 1))])
    lib = ops._lib.load()
    size = lib.sla2h_orthogonalize_workspace_bytes
    assert size(1, 32768, 32768) > 0 and size(1, 32769, 1) == 0 and size(0, 1, 1) == 0
    # matrices that one workgroup holds need none
    assert size(1 << 20, 64, 512) == size(1, 1, 1) < 1024 < size(1, 65, 512)


@pytest.mark.parametrize("steps,coeffs,ok", [
    (5, ops.NS_COEFFS, True), (30, ops.NS_COEFFS, True), (6, (1.5, -0.5, 0.0), True),
    (5, (2.0, -1.5, 0.5), True), (1, (10.0, 0.0, 0.0), True), (2, (10.0, 0.0, 0.0), False),
    (1, (1.0, 100.0, 50.0), False), (2, [(3.9, 0.0, 0.0), (1.0, -1.0, 0.0)], True),
    (2, [(4.1, 0.0, 0.0), (1.0, -1.0, 0.0)], False), (64, (1.0, 0.0, 0.0), True),
    (3, (3.0, -3.0, 1.0), True), (2, (0.0, 0.0, -5.0), False)])
def test_coefficients_that_leave_the_kernels_range(steps, coeffs, ok):
    """The bound is the largest value that the polynomials reach from [0, 1], step by step."""
    rows = [coeffs] * steps if not isinstance(coeffs[0], tuple) else coeffs
    top, fits = 1.0, True
    for a, b, c in rows:
        t = torch.linspace(0, top, 100001, dtype=torch.float64)
        fits &= top <= 4.0 and (b * t ** 2 + c * t ** 4).abs().max().item() < 127.0
        top = (a * t + b * t ** 3 + c * t ** 5).abs().max().item()
    assert fits == ok
    call = lambda: ops._ns_coeffs(steps, ops.ns_rows(steps, coeffs))
    if ok:
        call()
    else:
        with pytest.raises(ValueError, match="singular values"):
            call()

"""newton_schulz of a GPU tensor that carries a derivative: it is kept, as on the host."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(5, 9), (2, 40, 30)])
def test_a_gradient_is_kept(shape):
    """Three steps against float64 on the host.  Values and gradients are sums of at most 40 products per
    matrix product, seven products deep in a step and twice that in its backward: below 2,000 roundings of
    2^-24 of the largest, 1.2e-4, were they all of one sign."""
    from imfvideo_amd.muon import newton_schulz
    torch.manual_seed(1)
    g, d = torch.randn(shape), torch.randn(shape)
    x = g.cuda().requires_grad_(True)
    y = newton_schulz(x, 3)
    dx, = torch.autograd.grad(y, x, d.cuda())
    x64 = g.double().requires_grad_(True)
    y64 = newton_schulz(x64, 3)
    want, = torch.autograd.grad(y64, x64, d.double())
    for a, b in ((y, y64), (dx, want)):
        assert (a.double().cpu() - b).abs().max() <= 1.2e-4 * b.abs().max()
    with torch.no_grad():  # the kernels' values are the same to fp32's accuracy
        assert (newton_schulz(x, 3).double().cpu() - y64).abs().max() <= 1.2e-4 * y64.abs().max()


def test_a_tangent_is_kept():
    import torch.autograd.forward_ad as fw
    from imfvideo_amd.muon import newton_schulz
    torch.manual_seed(2)
    g, t = torch.randn(6, 8), torch.randn(6, 8)
    with fw.dual_level():
        got = fw.unpack_dual(newton_schulz(fw.make_dual(g.cuda(), t.cuda()), 3)).tangent
        want = fw.unpack_dual(newton_schulz(fw.make_dual(g.double(), t.double()), 3)).tangent
    assert (got.double().cpu() - want).abs().max() <= 1.2e-4 * want.abs().max()

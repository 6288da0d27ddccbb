"""Muon's step of 16-bit weights on the GPU: decay and update share one rounding."""
import pytest
import torch

from tests.test_gpu_muon import exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lr,decay", [(0.02, 0.5), (0.1, 3.0)])
def test_a_step_rounds_once(dt, lr, decay):
    """Of two matrices in one launch, against float64: half a step of the type, 1e-5 of the largest
    update for the update's own fp32 error (that of the same steps in fp32 is below 2e-6), and 3 * 2^-24
    of the terms for the sum."""
    from imfvideo_amd.muon import Muon
    torch.manual_seed(1)
    ps = [torch.nn.Parameter((0.2 * torch.randn(96, 160)).to(dt).cuda()) for _ in range(2)]
    w = [p.detach().double().cpu() for p in ps]
    g = [torch.randn(96, 160).to(dt) for _ in ps]
    for p, x in zip(ps, g):
        p.grad = x.cuda()
    Muon(ps, lr=lr, weight_decay=decay, nesterov=False).step()
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    for p, w0, x in zip(ps, w, g):
        d = lr * 0.2 * 160 ** 0.5 * exact(x.double())
        want = (1 - lr * decay) * w0 - d
        tol = (torch.finfo(dt).eps / 2 * want.abs() + 1e-5 * d.abs().max()
               + 3 * 2.0 ** -24 * (w0.abs() + d.abs()) + tiny)
        assert ((p.detach().double().cpu() - want).abs() <= tol).all()

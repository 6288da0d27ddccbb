"""newton_schulz's eager products under autocast: in float32 all the same."""
import pytest
import torch

from imfvideo_amd.muon import newton_schulz


def values(g, d, kind, on):
    """The result and its gradient, the call under autocast or not."""
    x = g.to(kind).requires_grad_(True)
    with torch.autocast(kind, torch.bfloat16, enabled=on):
        y = newton_schulz(x, 3)
    return y.detach(), torch.autograd.grad(y, x, d.to(kind))[0]


@pytest.mark.parametrize("kind", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("shape", [(12, 20), (2, 20, 12)])
def test_autocast_changes_nothing(shape, kind):
    torch.manual_seed(1)
    g, d = torch.randn(shape), torch.randn(shape)
    for a, b in zip(values(g, d, kind, True), values(g, d, kind, False)):
        assert a.dtype == b.dtype == torch.float32 and torch.equal(a, b)

"""orthogonalize at the largest singular values that it takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,C", [(1, 1), (1, 700), (40, 30), (130, 200), (300, 2100)])
@pytest.mark.parametrize("a", [3.98, -3.98])
def test_one_singular_value_at_the_bound(R, C, a):
    """A matrix of one element, and one of rank one: |a| in the second step, whose A holds |a|^2.  fp32's
    accuracy: a hundred times 2^-24 of the largest element, as pairs carry 22 bits."""
    from imfvideo_amd import ops
    g = torch.zeros(2, R, C, device="cuda")
    g[0, R // 2, C // 3] = -3.0
    g[1] = torch.ones(R, 1, device="cuda") * torch.linspace(1, 2, C, device="cuda")
    coeffs = [(a, 0.0, 0.0), (0.5, 0.01, -0.001)]
    x = g.double()
    x = x / x.square().sum((1, 2), keepdim=True).sqrt()
    s = a * (0.5 + 0.01 * a ** 2 - 0.001 * a ** 4)
    got = ops.orthogonalize(g, 2, coeffs).double()
    assert torch.isfinite(got).all()
    assert ((got - s * x).abs().amax((1, 2)) <= 100 * 2.0 ** -24 * abs(s) * x.abs().amax((1, 2))).all()

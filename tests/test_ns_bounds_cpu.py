"""The largest singular values that orthogonalize takes: A = X X^T is held in fp16, times 4,096."""
import pytest
import torch

from imfvideo_amd import ops
from imfvideo_amd.muon import Muon, newton_schulz

# a singular value of 1 becomes `a` in the first step, its square times 4,096 an element of A in the second
REFUSED = [4.0, 3.9999, 3.9995, 3.998, 3.992]
TAKEN = [3.98, 3.9, 1.0, -3.98]


def rows(a):
    return [(a, 0.0, 0.0), (1.0, 0.0, 0.0)]


@pytest.mark.parametrize("a", REFUSED)
def test_steps_that_could_reach_infinities_are_refused(a):
    """fp16 holds up to 65,504, and rounds to infinity from 65,520; what is refused leaves a 250th of
    that for the rounding of X and A (2^-11 of a value at most, each)."""
    for call in (lambda: newton_schulz(torch.ones(1, 3), 2, rows(a)),
                 lambda: Muon([torch.nn.Parameter(torch.ones(1, 3))], ns_steps=2, ns_coeffs=rows(a)),
                 lambda: ops._ns_coeffs(2, ops.ns_rows(2, rows(a)))):
        with pytest.raises(ValueError, match="singular values"):
            call()


@pytest.mark.parametrize("a", TAKEN)
def test_steps_within_them(a):
    assert a * a * 4096 * (1 + 2.0 ** -8) < 65520
    x = newton_schulz(torch.ones(1, 4), 2, rows(a))
    assert torch.equal(x, torch.full((1, 4), 0.5) * torch.tensor(a))
    # the last step's values are not squared any more
    ops._ns_coeffs(1, (100.0, 0.0, 0.0))

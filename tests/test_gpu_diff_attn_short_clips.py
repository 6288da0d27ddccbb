"""Differential attention's backward of short clips: as exact in a padded batch as alone."""
import pytest
import torch

from tests.diff_attn_padding import errors

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hkv,n,L,B", [(8, 8, 130, 3000, 3), (8, 8, 300, 3000, 3), (8, 8, 600, 3000, 3),
                                         (8, 4, 300, 4159, 2), (4, 4, 1000, 4159, 3), (8, 2, 500, 2200, 4),
                                         (8, 8, 2000, 4159, 3), (2, 2, 2048, 2300, 3)])
def test_a_clip_keeps_its_gradients_accuracy(H, Hkv, n, L, B, causal, dt):
    """Up to 2,048 rows per key pair.  An error of e roundings beside the result's own makes sqrt(1 + e^2) of
    it: 1.15 allows e = 0.57, where the roundings of dS and of the combined map, as large as the result's
    own, would be e = 1 (1.41)."""
    e = errors(n, H, Hkv, n, n, L, L, B, dt, causal)
    for name in ("dq", "dk", "dv"):
        for v in e[name]:
            assert v <= 1.15, (name, e)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("causal", [False, True])
def test_longer_clips_do_not_depend_on_the_batch_either(causal, dt):
    """2,500 rows, one launch alone and not in the batch: without the second products in dk and dv, e = 1 at
    most; dq with them."""
    e = errors(7, 8, 8, 2500, 2500, 5000, 5000, 3, dt, causal)
    assert max(e["dk"] + e["dv"]) <= 1.45 and max(e["dq"]) <= 1.15, e
    for name in ("dk", "dv"):  # the same roundings of the same numbers, added in other ranges
        assert abs(e[name][0] - e[name][1]) <= 0.02, e

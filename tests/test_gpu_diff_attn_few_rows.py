"""Differential attention's forward of a few rows: as exact in a padded batch as alone."""
import pytest
import torch

from tests.diff_attn_padding import errors

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk,Lq,Lk,B", [(1, 200, 1, 2000, 3), (1, 200, 300, 2000, 3),
                                           (2, 146, 700, 700, 2), (5, 300, 40, 6000, 4),
                                           (16, 180, 16, 1100, 2), (1, 129, 2000, 2000, 2),
                                           (3, 40, 500, 3000, 2)])
def test_a_clip_of_few_rows_keeps_its_accuracy(lq, lk, Lq, Lk, B, causal, dt):
    """With what the rounding of P lost only the result's own rounding is left: an error that is independent
    of it, of e roundings, makes sqrt(1 + e^2) of it, and 1.02 allows e = 0.2, where P's halves leave 2^-8
    of what they carry and fp32's sums 2^-15."""
    for v in errors(lk, 8, 8, lq, lk, Lq, Lk, B, dt, causal)["o"]:
        assert v <= 1.02


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("lq,lk,fine", [(16, 1024, True), (17, 1024, False), (16, 1025, False),
                                        (16, 129, True), (17, 129, False), (17, 128, True)])
def test_rows_on_both_sides_of_the_rule(lq, lk, fine, dt):
    """Row by row, alone and padded.  Without the second products a row's roundings of P are as large as the
    result's at most, where values do not add up (sqrt(2)), and a row of 512 results has 3 % of that by
    chance, 10 % the worst of 17."""
    for v in errors(lq + lk, 8, 8, lq, lk, 300, 1500, 2, dt, False, rows=True)["o"]:
        assert v <= (1.03 if fine else 1.1 * 2 ** 0.5)

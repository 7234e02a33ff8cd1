"""How many bf16 values hold the factor b + centre * s of a group's sum (qmm_rows8_tiles.hip), of every pair of significands at every distance of exponents that a float's 24 bits reach."""
import pytest

torch = pytest.importorskip("torch")


def left(bits, pieces):
    """The largest part of a factor that is left when `pieces` bf16 values have been taken out, of s and b of `bits` bits."""
    big = torch.arange(2 ** (bits - 1), 2 ** bits, dtype=torch.float64)
    worst = 0.0
    for distance in range(0, 26):
        for sign in (1, -1):
            factor = (big[:, None] + sign * big[None, :] * 2.0 ** -distance).float()
            rest = factor
            for _ in range(pieces):
                rest = rest - rest.bfloat16().float()
            part = torch.where(factor == 0, torch.zeros_like(factor), rest / factor)
            worst = max(worst, float(part.abs().max()))
    return worst


def test_two_hold_the_factors_of_bfloat16_scales_and_three_those_of_float16():
    assert left(8, 2) == 0.0
    assert 2.0 ** -18 < left(11, 2) <= 2.0 ** -17  # (what the third is for)
    assert left(11, 3) == 0.0

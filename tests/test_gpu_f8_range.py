"""Experts whose results or weights are near the ends of float32."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 300])
@pytest.mark.parametrize("weight", [2.0 ** 16, 2.0 ** -30])
def test_a_large_column_leaves_those_beside_it(T, weight):
    """Every value of h is silu(16) * 16 = 256 (1 - 2^-23), its codes 448.  Down's product is 448 * 2^119 in one column, -2^110 and zero in those beside it: a weight of 2^16 makes the
    first infinite, the second -2^126, the third zero.  Off by the roundings of h's scale and silu's (2^-20 for all), and of a row held in 11 bits."""
    from mlx_rs_amd import ops
    flat = torch.ones((1, 128, 128), device="cuda").to(o.F8), torch.full((1, 1, 1), 0.125, device="cuda")
    codes = torch.zeros((1, 128, 128), device="cuda")
    codes[:, 5], codes[:, 6:40] = 448.0, -2.0 ** -9
    down = codes.to(o.F8), torch.full((1, 1, 1), 2.0 ** 104, device="cuda")
    x = torch.ones((T, 128), device="cuda", dtype=torch.bfloat16)
    inds = torch.zeros((T, 1), device="cuda", dtype=torch.int32)
    y = ops.switch_glu_f8(x, inds, torch.full((T, 1), weight, device="cuda"), flat, flat, down)
    want = torch.zeros((T, 128), dtype=torch.float64, device="cuda")
    want[:, 5], want[:, 6:40] = 448.0 * 2.0 ** 119 * weight, -2.0 ** 110 * weight
    if weight > 1.0:
        assert (y[:, 5] == float("inf")).all()
        y, want = torch.cat((y[:, :5], y[:, 6:]), 1), torch.cat((want[:, :5], want[:, 6:]), 1)
    o.within(y, want, want.abs() * (2.0 ** -20 + 2.0 ** -11))

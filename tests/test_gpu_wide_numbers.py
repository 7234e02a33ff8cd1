"""Whole numbers beyond 32 bits are refused, not cut to what the library takes; a number of chosen experts beyond any memory before anything is allocated for it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FAR = 2 ** 32  # cut to 32 bits it adds nothing


def test_numbers_of_the_selection():
    import mlx_rs_amd as m
    x = torch.randn(4096, 16, device="cuda")
    select = m.ops.select_experts
    for call in (lambda: select(x, FAR + 2), lambda: select(x, 2, n_groups=FAR + 4, top_groups=2), lambda: select(x, 2, n_groups=4, top_groups=FAR + 2),
                 lambda: select(x, 2 - FAR), lambda: select(x, 2 ** 31 - 1), lambda: select(x, -1)):
        with pytest.raises(m.MoeError):
            call()


def test_numbers_of_quantized_matrices():
    import mlx_rs_amd as m
    w, s, b = m.ops.quantize(torch.randn(32, 256, device="cuda"), 64, 4, torch.bfloat16)
    x8, sx, x = torch.ones(3, 256, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"), torch.ones(3, 256, dtype=torch.bfloat16, device="cuda")
    o = m.ops
    for group, bits in ((FAR + 64, 4), (64, FAR + 4), (64 - FAR, 4)):
        for call in (lambda: o.quantized_linear_rows8(x8, sx, w, s, b, None, group, bits), lambda: o.quantized_linear(x, w, s, b, None, True, group, bits),
                     lambda: o.quantized_matmul(x, w, s, b, True, group, bits)):
            with pytest.raises(m.MoeError, match="out of range"):
                call()

"""The check that the calls make of whole numbers (ops._int32), without a GPU."""
import pytest


def test_what_fits_32_bits():
    pytest.importorskip("torch")
    import mlx_rs_amd as m
    for v in (0, 1, -1, 2 ** 31 - 1, -2 ** 31, True):
        m.ops._int32("f", ("n", 4), ("v", v))
    for v in (2 ** 31, -2 ** 31 - 1, 2 ** 32 + 64, 2 ** 64):
        with pytest.raises(m.MoeError, match="f: v is out of range"):
            m.ops._int32("f", ("n", 4), ("v", v))
    with pytest.raises(TypeError):
        m.ops._int32("f", ("v", 4.0))

"""Which kernel a linear layer on 8-bit rows takes: csrc/rows8_rule.hpp, which needs no GPU, compiled and asked."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KINDS = ["few 16x16", "few 16x32", "few 32x16", "few 32x32", "few 64x32", "tiles 64x64", "tiles 64x128", "tiles 128x128"]


@pytest.fixture(scope="module")
def kind(tmp_path_factory):
    d = tmp_path_factory.mktemp("rule")
    (d / "rule.cpp").write_text('#include "rows8_rule.hpp"\nextern "C" int kind(long M, int N, int K, int tiles) { return (int)mi_moe::rows8_kind(M, N, K, tiles != 0); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "mlx-rs_amd", "csrc"), str(d / "rule.cpp"), "-o", str(d / "rule.so")], check=True)
    lib = C.CDLL(str(d / "rule.so"))
    lib.kind.argtypes = [C.c_long, C.c_int, C.c_int, C.c_int]
    return lambda m, n, k, tiles=True: KINDS[lib.kind(m, n, k, tiles)]


@pytest.mark.parametrize("shape,want", [((16, 4096, 4096), KINDS[0]), ((16, 14336, 4096), KINDS[1]), ((64, 4096, 4096), KINDS[3]), ((128, 4096, 4096), KINDS[4]), ((64, 2048, 2048), KINDS[2]),
                                        ((256, 4096, 4096), KINDS[5]), ((64, 14336, 4096), KINDS[5]), ((1024, 4096, 4096), KINDS[6]), ((2048, 4096, 4096), KINDS[7]),
                                        ((2048, 14336, 4096), KINDS[7])])
def test_kinds_that_were_measured_fastest(kind, shape, want):
    assert kind(*shape) == want


def test_tiles_only_with_a_workspace_and_enough_rows(kind):
    for m in (1, 17, 300, 5000, 1 << 20):
        for n in (1, 500, 4096, 200000):
            for k in (128, 4096, 1 << 20):
                assert "few" in kind(m, n, k, False)
                assert m > 16 or "few" in kind(m, n, k)


def test_the_gpu_tests_reach_every_kind(kind):
    import test_gpu_rows8 as t
    assert {kind(*s) for s in t.SHAPES + t.TILED if s[0] > 2} == set(KINDS)  # (one and two rows take no kind at all)

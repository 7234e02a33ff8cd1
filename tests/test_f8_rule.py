"""Which kernel a product with e4m3 weights takes, in which pieces: csrc/f8_rule.hpp, which needs no GPU, compiled and asked."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """#include "f8_rule.hpp"
using namespace mi_moe;
static F8Sizes sizes(long rows, int N, int K, int mats, int transpose, int exact, int pair_sum) {
  return {rows, N, K, mats ? mats : 1, mats != 0, mats != 0, transpose != 0, false, pair_sum != 0, exact != 0, true, 0};
}
extern "C" int tile_rows(long rows, int N, int K, int mats, int transpose, int exact, int pair_sum) { return f8_tile_rows(sizes(rows, N, K, mats, transpose, exact, pair_sum)); }
extern "C" int plan(long rows, int N, int K, int mats, int transpose, int exact, int pair_sum) {
  const F8Plan p = f8_plan(sizes(rows, N, K, mats, transpose, exact, pair_sum));
  return p.tile * 100 + p.parts;
}
extern "C" long parts_bytes(long M, int N, int K, int pair_sum) { return M <= f8_parts_rows(N, f8_stages(K, pair_sum != 0)) ? (long)f8_parts_bytes(M, N, f8_stages(K, pair_sum != 0)) : 0; }
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    return load(tmp_path_factory.mktemp("rule"))


def load(d):
    (d / "rule.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "mlx-rs_amd", "csrc"), str(d / "rule.cpp"), "-o", str(d / "rule.so")], check=True)
    lib = C.CDLL(str(d / "rule.so"))
    lib.parts_bytes.restype = C.c_long
    for fn in (lib.tile_rows, lib.plan):
        fn.argtypes = [C.c_long] + [C.c_int] * 6
    lib.parts_bytes.argtypes = [C.c_long] + [C.c_int] * 3
    return lib


def kernel(lib, rows, N, K, mats=0, transpose=True, exact=False, pair_sum=False):
    """(rows of a piece or tile, blocks that share a tile); pieces below 64 rows are those of the kernel for a few rows."""
    args = (rows, N, K, mats, transpose, exact, pair_sum)
    few = lib.tile_rows(*args)
    return (few, 1) if few < 64 else divmod(lib.plan(*args), 100)


# bfloat16, then float16 and float32
@pytest.mark.parametrize("shape,want,exact", [
    (dict(rows=1, N=4096, K=2048), (16, 1), (16, 1)), (dict(rows=48, N=4096, K=4096), (32, 1), (32, 1)), (dict(rows=1000, N=4096, K=4096), (64, 1), (64, 1)),
    (dict(rows=4096, N=4096, K=4096), (256, 1), (128, 1)), (dict(rows=1000, N=4096, K=4096, transpose=False), (64, 1), (64, 1)), (dict(rows=1, N=4096, K=4096, transpose=False), (64, 16), (64, 16)),
    (dict(rows=300, N=768, K=2048, mats=128), (16, 1), (16, 1)), (dict(rows=32768, N=2048, K=768, mats=128), (256, 1), (128, 1)),
    (dict(rows=16384, N=1408, K=2048, mats=64, transpose=False), (256, 1), (128, 1)), (dict(rows=8, N=2048, K=768, mats=128, transpose=False, pair_sum=True), (64, 4), (64, 4))])
def test_kernels_by_size(rule, shape, want, exact):
    assert kernel(rule, **shape) == want
    assert kernel(rule, **shape, exact=True) == exact


def test_the_gpu_tests_reach_every_tile(rule):
    torch = pytest.importorskip("torch")  # noqa: F841
    import test_gpu_f8_large as t
    for transpose in (True, False):
        assert [kernel(rule, *shape, transpose=transpose) for shape in t.DENSE] == [(256, 1), (128, 1), (256, 1), (256, 1), (128, 2), (256, 8), (64, 4)]
        assert [kernel(rule, *shape, transpose=transpose, exact=True) for shape in t.DENSE] == [(128, 1), (128, 1), (128, 1), (128, 1), (128, 2), (128, 4), (64, 4)]
    assert kernel(rule, *t.SHARED, mats=1) == (256, 4) and kernel(rule, *t.SHARED, mats=1, exact=True) == (128, 1)


def test_parts_have_room(rule):
    for rows in (1, 16, 49, 64, 100, 256, 300, 1000, 2048, 4096, 10000, 32768, 1 << 20):
        for N in (1, 16, 256, 1000, 4096, 16384, 1 << 20):
            for K in (16, 128, 640, 2048, 4096, 16384, 1 << 20):
                for mats in (0, 1, 16, 128, 512):
                    for transpose, exact in ((True, False), (True, True), (False, False), (False, True)):
                        tile, parts = kernel(rule, rows, N, K, mats, transpose, exact)
                        assert tile in ((16, 32, 64, 128) if exact else (16, 32, 64, 128, 256)) and (tile >= 64 or transpose)
                        assert parts == 1 or parts * rows * N * 4 <= rule.parts_bytes(rows, N, K, False)
                        assert parts == 1 or 2 * parts <= (K + 127) // 128


def test_workspaces_hold_no_parts_where_there_are_none():
    from mlx_rs_amd import load_library
    lib = load_library()

    def linear(M, N, K):
        n = C.c_size_t()
        assert lib.mi_moe_linear_f8_workspace_size(M, N, K, C.byref(n)) == 0
        return n.value

    def rows(M, K):  # codes and scales, and the list of 512 matrices' pieces
        return M * -(-K // 128) * 132 + 16 * (M // 16 + min(M, 513)) + 2048

    assert linear(4096, 4096, 4096) <= rows(1024, 4096) + (33 << 20)  # (as much as for 1024 rows, which may come in parts)
    assert linear(32768, 4096, 4096) <= rows(32768, 4096) and linear(4096, 4096, 256) <= rows(4096, 256)
    for N, K in ((4096, 4096), (1, 16), (16384, 512), (256, 65536), (1000, 1040)):
        sizes = [linear(M, N, K) for M in list(range(0, 5000, 7)) + [10000, 100000, 300000]]
        assert sizes == sorted(sizes)

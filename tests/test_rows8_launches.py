"""How many rows one launch of a linear layer on 8-bit rows takes (csrc/rows8_rule.hpp, compiled and asked on the host): with them every kind's launch, and that of the rows' preparation, has
less than 2^32 threads, whatever the sizes, with a workspace and without."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS = [16, 16, 32, 32, 64, 64, 64, 128]  # of a block, by kind


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("rule")
    (d / "rule.cpp").write_text("""#include "rows8_rule.hpp"
using namespace mi_moe;
extern "C" int kind(long M, int N, int K, int tiles) { return (int)rows8_kind(M, N, K, tiles != 0); }
extern "C" long step(int k, int N, int K, int group) { return rows8_step((Rows8Kind)k, N, K, group); }
extern "C" long blocks(int k, long M, int N) { return rows8_blocks((Rows8Kind)k, M, N); }
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "mlx-rs_amd", "csrc"), str(d / "rule.cpp"), "-o", str(d / "rule.so")], check=True)
    lib = C.CDLL(str(d / "rule.so"))
    lib.kind.argtypes, lib.step.argtypes, lib.blocks.argtypes = [C.c_long, C.c_int, C.c_int, C.c_int], [C.c_int] * 4, [C.c_int, C.c_long, C.c_int]
    lib.step.restype = lib.blocks.restype = C.c_long
    return lib


def sizes():
    for n in list(range(1, 80)) + [100, 127, 128, 129, 500, 1000, 4096, 14336, 10 ** 5, 2 ** 20, 2 ** 23 + 5, 2 ** 26 - 4]:
        for k in (128, 256, 384, 1024, 4096, 2 ** 17, 2 ** 20):
            yield n, k


@pytest.mark.parametrize("tiles", [False, True])
def test_every_launch_has_less_than_2_32_threads(rule, tiles):
    split = set()
    for n, k in sizes():
        for m in (3, 17, 1000, 2 ** 16 + 1, 2 ** 23 - 1, 2 ** 26, 64 * 10 ** 6, 2 ** 27, 2 ** 28 + 5, 2 ** 30):
            kind = rule.kind(m, n, k, tiles)
            for group in (32, 64, 128):
                step = rule.step(kind, n, k, group)
                assert step > 0 and step % ROWS[kind] == 0, (m, n, k, group)
                rows = min(m, step)
                assert rule.blocks(kind, rows, n) * 512 < 2 ** 32, (m, n, k, group)
                if kind >= 5:
                    waves = (rows + 15) // 16 * ((k // group + 7) // 8 * 2)
                    assert (waves + 3) // 4 * 256 < 2 ** 32, (m, n, k, group)
                if m > step:
                    split.add(kind)
    assert split >= ({5, 7} if tiles else {2, 4})  # (kinds that more rows than a launch's are for)


def test_columns_beyond_a_launch(rule):
    for kind in range(8):
        assert rule.step(kind, 2 ** 31 - 1, 128, 64) >= 0
    assert rule.step(0, 2 ** 31 - 1, 128, 64) == 0


@pytest.mark.parametrize("tiles", [False, True])
def test_the_rule_at_the_most_columns(rule, tiles):
    """A count of columns that ends just below 2^31 takes what one a block below takes."""
    for m in (3, 17, 40, 300, 5000):
        for k in (128, 4096):
            assert rule.kind(m, 2 ** 31 - 1, k, tiles) == rule.kind(m, 2 ** 31 - 2 ** 12, k, tiles), (m, k)

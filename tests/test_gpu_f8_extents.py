"""Extents near the ends of what the e4m3 products take: more tiles than a launch has blocks, and more than 2^31 values."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def needs(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
        pytest.skip(f"needs {gigabytes} GB of memory")


def test_more_float32_rows_than_a_launch_has_tiles_for():
    """2^29 + 200 rows in tiles of 128: one launch holds 2^22 of them."""
    from mlx_rs_amd import ops
    needs(130)
    gen = torch.Generator(device="cuda").manual_seed(1)
    M, K = 2 ** 29 + 200, 16
    w, s = o.bank(gen, 1, K)
    x = torch.empty((M, K), device="cuda").uniform_(-1.0, 1.0, generator=gen)
    y = ops.linear_f8(x, w, s)
    at = torch.cat((torch.arange(300), torch.arange(2 ** 28 - 150, 2 ** 28 + 150), torch.arange(M - 500, M))).cuda()
    want, off = o.product(*o.quantize_rows(x[at]), w.double(), s, None, torch.float32)
    o.within(y[at], want, off)


def test_pieces_of_many_matrices_by_many_columns():
    """512 matrices that may have a piece each, by 8192 tiles of columns; 2^30 values of the result, 2^34 of the bank."""
    from mlx_rs_amd import ops
    needs(30)
    gen = torch.Generator(device="cuda").manual_seed(2)
    E, K, N, R = 512, 16, 2 ** 21, 600
    w = torch.empty((E, K, N), device="cuda", dtype=torch.uint8).random_(0, 0x70, generator=gen).view(o.F8)
    s = 0.5 + torch.rand((E, 1, N // 128), generator=gen, device="cuda")
    counts = torch.zeros(E, dtype=torch.int64)
    for e, n in ((0, 3), (1, 100), (7, 1), (255, 200), (256, 65), (400, 64), (510, 1), (511, 140)):
        counts[e] = n
    ends = [0] + counts.cumsum(0).tolist()
    x = torch.randn((R, K), generator=gen, device="cuda").bfloat16()
    y = ops.grouped_linear_f8(x, w, s, torch.tensor(ends, device="cuda", dtype=torch.int32), False)
    codes, scales = o.quantize_rows(x)
    at = torch.cat((torch.arange(300), torch.arange(12345, N, 2097), torch.arange(N - 300, N))).cuda()
    for e in counts.nonzero()[:, 0].tolist():
        rows = slice(ends[e], ends[e + 1])
        each = s[e, 0, at // 128].double()
        want, off = o.product(codes[rows], scales[rows], w[e].view(torch.uint8)[:, at].view(o.F8).double().t(), torch.ones((o.blocks(len(at)), 1), device="cuda"), None, torch.bfloat16)
        o.within(y[rows][:, at], want * each, off * each, f"matrix {e}")
    assert not y[ends[-1]:].any()

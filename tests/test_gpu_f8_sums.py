"""Sums of runs in which some products are far larger than the rest, on the kernels of the e4m3 products."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def rows_and_weights(gen, M, N, K, kind):
    """Codes of both sides in float64, every run's largest row value 448, so that a row's scale is one.
    "pairs": one product of 448 * 448 in a run and minus that in the next, all others 2.75 * 2.75 (below 2^-14 of it) and of one sign.
    "eights": in every eight products one of 448 * 448, of either sign, and small ones of one sign of many sizes."""
    x, w = torch.full((M, K), 2.75, device="cuda"), torch.full((N, K), 2.75, device="cuda")
    if kind == "eights":
        x = torch.exp2(torch.randint(-3, 3, (M, K), generator=gen, device="cuda").float()) * 1.375
        w = torch.exp2(torch.randint(-3, 3, (N, K), generator=gen, device="cuda").float()) * 1.875
    step = 8 if kind == "eights" else 128
    for i, k in enumerate(range(0, K, step)):
        at = k + (5 * i) % min(step, K - k)
        x[:, at] = 448.0
        w[:, at] = 448.0 if i % 2 == 0 else -448.0
    return x.double(), w.double()


def sums(x, w):
    """The sums and what they may be off by in float32: (K + 2) roundings of the magnitudes' sum."""
    return x @ w.t(), (x.shape[1] + 2) * 2.0 ** -24 * (x.abs() @ w.abs().t())


SCALE = 2.0 ** -10  # of the weights' blocks: results in float16's range


def calls(M, dtype, transpose, kind):
    """A linear layer, the same as the only matrix of a grouped product, and what they should give."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    x, w = rows_and_weights(gen, M, 80, 512, kind)
    codes = (w if transpose else w.t()).float().contiguous().to(o.F8)
    scales = torch.full((o.blocks(codes.shape[0]), o.blocks(codes.shape[1])), SCALE, device="cuda")
    rows, offsets = x.to(dtype), torch.tensor([0, M], device="cuda", dtype=torch.int32)
    from mlx_rs_amd import ops
    want, off = sums(x, w)
    return lambda: ops.linear_f8(rows, codes, scales, transpose=transpose), lambda: ops.grouped_linear_f8(rows, codes[None], scales[None], offsets, transpose), want * SCALE, off * SCALE


@pytest.mark.parametrize("kind", ["pairs", "eights"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 3, 40])
def test_a_few_rows(M, dtype, kind):
    linear, grouped, want, off = calls(M, dtype, True, kind)
    o.within(linear(), want, off, f"linear {M} {dtype} {kind}")
    if M <= 4:
        o.within(grouped(), want, off, f"grouped {M} {dtype} {kind}")

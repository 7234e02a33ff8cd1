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


@pytest.mark.parametrize("kind", ["pairs", "eights"])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("M", [1, 40, 100, 300])
def test_float16_and_float32_in_tiles(M, dtype, transpose, kind):
    linear, grouped, want, off = calls(M, dtype, transpose, kind)
    o.within(linear(), want, off, f"linear {M} {dtype} {transpose} {kind}")
    o.within(grouped(), want, off, f"grouped {M} {dtype} {transpose} {kind}")


def down_of_large_products(T, dtype):
    """gate = up = 1 makes every value of h silu(4) * 4, of which all codes are 448; down's products are 448 * 448 and -448 * 448 in every eight, and small ones of one sign.
    What the experts give, what they should, and by what that may be off but for down's sums: the roundings of silu and of h's scale (2^-20 for all of them), float32's of the sum."""
    from mlx_rs_amd import ops
    K = 256
    ones = torch.ones((2, K, 128), device="cuda").to(o.F8), torch.full((2, 2, 1), 4.0 / 128, device="cuda")
    w = torch.full((128, K), 0.0625, device="cuda", dtype=torch.float64)
    w[:, 1::8], w[:, 6::8] = 448.0, -448.0
    w[::2] = w[::2] * torch.where(w[::2].abs() < 1, 7.0, 1.0)
    down = w.float().to(o.F8).expand(2, 128, K).contiguous(), torch.full((2, 1, 2), 2.0 ** -9, device="cuda")
    x = torch.ones((T, 128), device="cuda", dtype=dtype)
    inds = torch.tensor([0, 1], device="cuda", dtype=torch.int32).expand(T, 2).contiguous()
    y = ops.switch_glu_f8(x, inds, torch.full((T, 2), 0.5, device="cuda"), ones, ones, down)
    h = 16.0 / (1.0 + torch.exp(torch.tensor(-4.0, dtype=torch.float64))).item() * 2.0 ** -9
    want = (w.sum(1) * h).expand(T, 128)
    return y, want, want.abs() * 2.0 ** -20 + (w.abs().sum(1) * h * (K + 2) * 2.0 ** -24).expand(T, 128)


@pytest.mark.parametrize("T,dtype", [(1, torch.bfloat16), (1, torch.float16), (3, torch.bfloat16), (3, torch.float16), (40, torch.float16), (300, torch.float16)])
def test_experts_whose_down_has_large_products(T, dtype):
    y, want, off = down_of_large_products(T, dtype)
    o.within(y, want, off, f"experts {T} {dtype}")


def eights(x, w):
    """What sums on the f8 instructions may be off by, as the header has it: of every eight products seven times 2^-13 of the largest, codes below 2^-6 counted as 2^-6, and the
    adding up of the eights in float32."""
    least = lambda c: torch.where(c == 0, 0.0, c.abs().clamp(min=2.0 ** -6))  # noqa: E731
    off = 2.0 ** -22 * (x.abs() @ w.abs().t())
    for k in range(0, x.shape[1], 8):
        off += 7 * 2.0 ** -13 * (least(x[:, None, k:k + 8]) * least(w[None, :, k:k + 8])).amax(-1)
    return off


@pytest.mark.parametrize("kind", ["pairs", "eights", "one", "small"])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("M", [40, 100, 300])
def test_bfloat16_in_tiles_is_off_by_what_the_header_says(M, transpose, kind):
    from mlx_rs_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(M)
    N, K = 80, 512
    x, w = rows_and_weights(gen, M, N, K, kind)
    if kind == "one":  # a large product a run, of the others' sign
        x, w = (torch.where(c.abs() == 448.0, 448.0, c) for c in (x, w))
    if kind == "small":  # eights of codes from 2^-9 on beside the runs' largest
        x, w = (torch.exp2(torch.randint(-9, 3, c.shape, generator=gen, device="cuda").double()) * (2.0 * torch.randint(0, 2, c.shape, generator=gen, device="cuda") - 1.0) for c in (x, w))
        x[:, ::128] = 448.0
    codes = (w if transpose else w.t()).float().contiguous().to(o.F8)
    scales = torch.full((o.blocks(codes.shape[0]), o.blocks(codes.shape[1])), SCALE, device="cuda")
    rows, offsets = x.bfloat16(), torch.tensor([0, M], device="cuda", dtype=torch.int32)
    want, off = sums(x, w)
    off = (off + eights(x, w)) * SCALE
    o.within(ops.linear_f8(rows, codes, scales, transpose=transpose), want * SCALE, off, f"linear {M} {transpose} {kind}")
    o.within(ops.grouped_linear_f8(rows, codes[None], scales[None], offsets, transpose), want * SCALE, off, f"grouped {M} {transpose} {kind}")


@pytest.mark.parametrize("T", [40, 300])
def test_experts_in_bfloat16_are_off_by_what_the_header_says(T):
    y, want, off = down_of_large_products(T, torch.bfloat16)
    h = 16.0 / (1.0 + torch.exp(torch.tensor(-4.0, dtype=torch.float64))).item() * 2.0 ** -9
    o.within(y, want, off + 256 / 8 * 7 * 2.0 ** -13 * 448.0 * h + 2.0 ** -11 * want.abs(), f"experts {T}")


def opposite(T, H, inter, gate1, down1, x_columns):
    """Two experts that a token names with weights 1 and -1: gate, up and down are all 1 but for the second one's gate1 and down1 (or 1); x and dout are ones, x in its first
    x_columns alone.  The arguments of the experts' calls, and float64 values: g = u, h, dh, and a block's scale of gate and of down."""
    ones = torch.ones
    gate, up, down = ones((2, inter, H), device="cuda"), ones((2, inter, H), device="cuda"), ones((2, H, inter), device="cuda")
    gate[:, :, x_columns:], up[:, :, x_columns:] = 1.0, 0.0
    if gate1 is not None:
        gate[1] = gate1
    if down1 is not None:
        down[1] = down1
    sg, sd = 4.0 / x_columns, 2.0 ** -9
    banks = [(w.to(o.F8), torch.full((2, o.blocks(w.shape[1]), o.blocks(w.shape[2])), s, device="cuda")) for w, s in ((gate, sg), (up, sg), (down, sd))]
    x, dout = torch.zeros((T, H), device="cuda", dtype=torch.float16), torch.ones((T, H), device="cuda", dtype=torch.float16)
    x[:, :x_columns] = 1.0
    inds = torch.tensor([0, 1], device="cuda", dtype=torch.int32).expand(T, 2).contiguous()
    weights = torch.tensor([1.0, -1.0], device="cuda").expand(T, 2).contiguous()
    sigma = 1.0 / (1.0 + torch.exp(torch.tensor(-4.0, dtype=torch.float64))).item()
    return (x, inds, weights, *banks), dout, sigma, sg, sd


# (a few rows, tiles of 64 and 128 rows; one tile of columns and several)
@pytest.mark.parametrize("T,H", [(1, 128), (3, 608), (40, 128), (40, 608), (40, 1296), (300, 608), (300, 2048)])
def test_float16_rows_on_their_way_to_the_sum(T, H):
    """Rows of two experts that differ in their last bits: 256 and 256.125 times a number, which 11 bits do not tell apart.  All products are 448 and 504, their sums of a run exact: each
    of two rows has two runs, with a rounding of the scale, of the product with it and of the sum, and the sum over slots another."""
    from mlx_rs_amd import ops
    inter = 256
    down1 = torch.ones((H, inter), device="cuda")
    down1[:, 5] = 1.125
    args, _, sigma, sg, sd = opposite(T, H, inter, None, down1, 16)
    h = 16.0 * sigma
    want = torch.full((T, H), -0.125 * h * sd, dtype=torch.float64, device="cuda")
    o.within(ops.switch_glu_f8(*args), want, want.abs() * 2.0 ** -20 + 2 * 256.125 * h * sd * (3 * 2 + 1) * 2.0 ** -24, f"{T} {H}")


@pytest.mark.parametrize("T,H", [(1, 144), (3, 608), (40, 144), (40, 608), (40, 1296), (300, 608), (300, 2048)])
def test_float16_gradients_on_their_way_to_the_sum(T, H):
    """The same of the tokens' gradient: in the columns where x is zero the second gate may differ and the experts' own gradients are the same."""
    from mlx_rs_amd import ops
    inter = 256
    gate1 = torch.ones((inter, H), device="cuda")
    gate1[5, 16:] = 1.125
    args, dout, sigma, sg, sd = opposite(T, H, inter, gate1, None, 16)
    dg = H * sd * 4.0 * sigma * (1.0 + 4.0 * (1.0 - sigma))
    du = H * sd * 4.0 * sigma
    want = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    want[:, 16:] = -0.125 * dg * sg
    dx, dw = ops.switch_glu_f8_grad(dout, *args)
    o.within(dx, want, want.abs() * 2.0 ** -20 + 2 * 256.125 * (dg + du) * sg * (3 * 4 + 2) * 2.0 ** -24, f"{T} {H}")
    wanted = torch.full((T, 2), H * sd * 16.0 * sigma * inter, dtype=torch.float64, device="cuda")
    o.within(dw, wanted, wanted * (H + inter + 30) * 2.0 ** -24, "weights")

"""The quantized linear layer on rows in eight bits against float64."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step, relative
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def layer(M, N, K, bits, group, dtype, seed=0, bias=False):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + M * 31 + N * 17 + K)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    words = torch.randint(-2 ** 31, 2 ** 31, (N, K * bits // 32), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    scales = (0.01 * (1 + 0.2 * normal(N, K // group))).to(dtype)
    biases = (-scales.float() * (2 ** bits - 1) / 2 + 0.005 * normal(N, K // group)).to(dtype)
    x = (normal(M, K) * 40).round().clamp(-127, 127).to(torch.int8)
    sx = 0.02 * (1 + 0.3 * normal(M).clamp(-2, 2))
    return x, sx, words, scales, biases, (normal(N).to(dtype) if bias else None)


def truth(x, sx, w, s, b, lb, group, bits):
    """(result, size of the terms) in float64."""
    N = w.shape[0]
    shifts = torch.arange(32 // bits, device="cuda", dtype=torch.int32) * bits
    c = ((w[..., None] >> shifts) & (2 ** bits - 1)).double().reshape(N, -1, group)
    dense = (s.double()[..., None] * c + b.double()[..., None]).reshape(N, -1)
    y = torch.matmul(x.double(), dense.t().contiguous()) * sx.double()[:, None]
    centre = 2 ** (bits - 1)
    beta = b.double() + centre * s.double()
    # every term of a kernel's float sums is s times an integer or beta times one, of a word of codes or more: at most the sum of sizes over words
    per = 32 // bits
    size = torch.zeros_like(y)
    xw = x.double().reshape(x.shape[0], -1, per)
    cw = (c.reshape(N, -1) - centre).reshape(N, -1, per)
    sw, bw = s.double().repeat_interleave(group // per, 1), beta.repeat_interleave(group // per, 1)
    for i in range(0, xw.shape[1], 16):
        d = torch.matmul(xw[:, i:i + 16].permute(1, 0, 2).contiguous(), cw[:, i:i + 16].permute(1, 2, 0).contiguous()).abs()
        size += (d * sw[:, i:i + 16].t()[:, None, :].abs()).sum(0)
    size += torch.matmul(xw.sum(-1).abs(), bw.abs().t().contiguous())
    return (y if lb is None else y + lb.double()), size * sx.double()[:, None]


# products whose tiles fill the chip, with last tiles of every kind
TILED = [(257, 3000, 512), (520, 5000, 256), (1300, 4111, 128), (900, 2500, 896), (2100, 4000, 384), (1000, 4096, 512), (256, 4096, 1024)]


def check(y, args, group, bits):
    x, sx, w, s, b, lb = args
    ref, size = truth(x, sx, w, s, b, lb, group, bits)
    # A term goes through at most two additions a group or, in lanes over words, two a word of every 64th and six more; its own product and factor cost two half
    # steps, the row's scale and the bias one each (of the result's size), and the type's rounding half a step of the result.
    K = x.shape[1]
    chain = 2 * max(K // group, K * bits // 32 // 64 + 1) + 8
    bound = torch.finfo(y.dtype).eps / 2 * ref.abs() + (chain + 4) * U * size + 2 * U * ref.abs() + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    if x.shape[0] > 16 and y.dtype != torch.float32:
        # biases of 16-bit layers, many rows: the factor of a group's sum is two bfloat16 values, the second the rounded rest of the first: 2^-9 of 2^-9 of the factor
        bound = bound + 2.0 ** -18 * size
    err = (y.double() - ref).abs()
    assert y.shape == ref.shape and bool((err <= bound).all()), float((err / bound).max())


def run(args, group, bits):
    import mlx_rs_amd as m
    x, sx, w, s, b, lb = args
    y = m.ops.quantized_linear_rows8(x, sx, w, s, b, lb, group, bits)
    assert y.dtype == s.dtype
    return y


# rows x columns x K: one row, one column, K of one group, of no whole 128, rows and columns on both sides of 16, 32, 64 and 128, more of them than a tile, K of an odd number of groups
SHAPES = [(1, 1, 128), (1, 17, 256), (1, 1000, 2048), (2, 64, 384), (7, 33, 640), (15, 16, 128), (16, 48, 1152), (17, 100, 512), (31, 129, 896), (33, 64, 1024), (48, 200, 4096),
          (64, 128, 256), (65, 127, 384), (100, 300, 2176), (128, 256, 640), (129, 513, 128), (200, 96, 1280), (257, 384, 768), (300, 1000, 1024), (520, 272, 512), (13, 9001, 384), (6, 9000, 1152), (30, 4500, 2176)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(dtype, bits, group, M, N, K):
    args = layer(M, N, K, bits, group, dtype, bias=(M + N) % 2 == 1)
    check(run(args, group, bits), args, group, bits)


@pytest.mark.parametrize("M,N,K", TILED)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_in_tiles(dtype, bits, group, M, N, K):
    args = layer(M, N, K, bits, group, dtype, bias=(M + N) % 2 == 1)
    check(run(args, group, bits), args, group, bits)


@pytest.mark.parametrize("group,K", [(32, 32), (32, 96), (64, 64), (64, 192), (32, 160), (64, 4160)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 9, 70])
def test_rows_of_no_whole_128(M, bits, group, K):
    args = layer(M, 37, K, bits, group, torch.bfloat16)
    check(run(args, group, bits), args, group, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_operands_that_start_anywhere(M, bits):
    """Rows off 16 bytes, scales off a word: the same results as where they start even."""
    args = layer(M, 50, 384, bits, 64, torch.float16, bias=True)

    def shifted(t, by):
        flat = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
        flat[by:] = t.reshape(-1)
        return flat[by:].view(t.shape)

    moved = [shifted(t, by) for t, by in zip(args, (3, 1, 1, 1, 3, 1))]
    check(run(moved, 64, bits), args, 64, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 20, 150])
def test_extreme_rows_and_codes(M, bits):
    """All codes at either end and rows of -127 and 127: the integer sums at their largest; rows of zeros; a row whose scale is none."""
    import mlx_rs_amd as m
    N, K, group = 40, 4096, 128
    args = list(layer(M, N, K, bits, group, torch.float32))
    args[2][:10] = 0
    args[2][10:20] = -1
    args[0][:] = 127
    args[0][M // 2:] = -127
    check(run(args, group, bits), args, group, bits)
    args[0][0] = 0
    assert not run(args, group, bits)[0].any()
    args[1][0] = float("nan")
    y = run(args, group, bits)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_a_row_of_minus_128(bits):
    """Not what add_rms_norm_rows8 makes, but a signed byte."""
    for M in (1, 64):
        args = list(layer(M, 32, 1024, bits, 128, torch.float32))
        args[0][:] = -128
        check(run(args, 128, bits), args, 128, bits)


def test_shapes_of_rows_and_no_rows():
    import mlx_rs_amd as m
    x, sx, w, s, b, lb = layer(24, 32, 256, 4, 64, torch.bfloat16)
    y = m.ops.quantized_linear_rows8(x.reshape(2, 3, 4, 256), sx.reshape(2, 3, 4), w, s, b)
    assert y.shape == (2, 3, 4, 32) and torch.equal(y.reshape(24, 32), m.ops.quantized_linear_rows8(x, sx, w, s, b))
    one = m.ops.quantized_linear_rows8(x[0], sx[0], w, s, b)
    assert one.shape == (32,)
    assert m.ops.quantized_linear_rows8(x[:0], sx[:0], w, s, b).shape == (0, 32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits,group", [(4, 32), (4, 64), (4, 128), (8, 32), (8, 64), (8, 128)])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
def test_one_to_five_rows(M, bits, group, dtype):
    """K of less than a wave's step and more, whole steps and not; one column, an odd number, more than a block's."""
    for N, K in ((1, 128), (7, 256), (8, 2048), (33, 1920), (1001, 4096), (300, 8320)):
        args = layer(M, N, K, bits, group, dtype, bias=N % 2 == 1)
        check(run(args, group, bits), args, group, bits)


@pytest.mark.parametrize("M,N,K,step", [(8192 + 70, 2 ** 20, 128, 8192), (2 ** 16 * 8 + 70, 512, 32, 2 ** 16 * 8)])
def test_more_rows_than_a_launch_takes(M, N, K, step):
    """Rows on both sides of where a launch ends, results past 2^32 elements: the bits of a call of their own rows."""
    import mlx_rs_amd as m
    w, s, b = m.ops.quantize(torch.randn(N, K, device="cuda"), 32, 4, torch.bfloat16)
    x = torch.randint(-127, 128, (M, K), device="cuda", dtype=torch.int32).to(torch.int8)
    sx = torch.rand(M, device="cuda")
    y = m.ops.quantized_linear_rows8(x, sx, w, s, b, None, 32, 4)
    for at in (0, step - 64, step, M - 64):
        some = slice(at, at + 64)
        part = m.ops.quantized_linear_rows8(x[some].contiguous(), sx[some].contiguous(), w, s, b, None, 32, 4)
        err, size = (y[some].float() - part.float()).abs(), part.float().abs()
        # two orders of the same float sums: each rounded once to bfloat16, whose steps are 2^-8 of a value and next to which the sums' own differences are little
        assert bool((err <= 2.0 ** -7 * size + 1e-3).all())
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [17, 100, 600])
def test_without_room_for_prepared_rows(M):
    """No workspace, and one that is a byte short: the kernels that need none, never a write outside."""
    import mlx_rs_amd as m
    args = layer(M, 640, 512, 4, 64, torch.bfloat16)
    x, sx, w, s, b, _ = args
    lib = m.load_library()
    need = m.ops._rows8_workspace_bytes(M, 512)
    assert need > 0
    for room, size in ((None, 0), (torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda"), need - 1)):
        y = torch.empty(M, 640, dtype=torch.bfloat16, device="cuda")
        m.capi.check(lib.mi_moe_quantized_linear_rows8(x.data_ptr(), sx.data_ptr(), w.data_ptr(), s.data_ptr(), b.data_ptr(), None, M, 640, 512, 64, 4, 0, y.data_ptr(),
                                                       None if room is None else room.data_ptr(), size, m.ops._stream()))
        check(y, args, 64, 4)
        assert room is None or bool((room == 77).all())


def test_the_workspace_ends_where_it_says():
    import mlx_rs_amd as m
    lib = m.load_library()
    for M, N, K, bits, group in ((600, 640, 512, 4, 64), (130, 2048, 384, 8, 32), (257, 4096, 128, 4, 128)):
        args = layer(M, N, K, bits, group, torch.bfloat16)
        x, sx, w, s, b, _ = args
        need = m.ops._rows8_workspace_bytes(M, K)
        room = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
        y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        m.capi.check(lib.mi_moe_quantized_linear_rows8(x.data_ptr(), sx.data_ptr(), w.data_ptr(), s.data_ptr(), b.data_ptr(), None, M, N, K, group, bits, 0, y.data_ptr(),
                                                       room.data_ptr(), need, m.ops._stream()))
        check(y, args, group, bits)
        assert bool((room[need:] == 77).all())


def test_refusals():
    import mlx_rs_amd as m
    x, sx, w, s, b, lb = layer(4, 32, 256, 4, 64, torch.bfloat16, bias=True)
    f = m.ops.quantized_linear_rows8
    for call in (lambda: f(x.float(), sx, w, s, b), lambda: f(x, sx.half(), w, s, b), lambda: f(x, sx[:3], w, s, b), lambda: f(x[:, :128].contiguous(), sx, w, s, b),
                 lambda: f(x, sx, w, s, b.float()), lambda: f(x, sx, w, s[:, :2].contiguous(), b), lambda: f(x, sx, w, s, b, lb[:5]), lambda: f(x, sx, w, s, b, None, 16),
                 lambda: f(x, sx, w, s, b, None, 64, 2), lambda: f(x, sx, w.t(), s, b), lambda: f(x, sx, w, s, b, None, 64, 3)):
        with pytest.raises(m.MoeError):
            call()

"""Linear layers, grouped products and experts on e4m3 weights, and their gradients, against their definitions in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(gen, M, K, dtype):
    """Rows whose runs have very different sizes, some of zeros."""
    x = torch.randn((M, K), generator=gen, device="cuda") * torch.exp2(torch.randint(-6, 7, (M, 1), generator=gen, device="cuda").float())
    x[torch.rand((M, K), generator=gen, device="cuda") < 0.05] = 0
    if M > 1:
        x[M // 2, :128] = 0
    return x.to(dtype)


# ---------------------------------------------------------------- codes
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (5, 128), (129, 129), (130, 1000), (2, 3, 200), (300, 2048)])
def test_codes_and_scales_are_the_definition_s(shape, dtype):
    from mlx_rs_amd import ops
    gen = gen_of(sum(shape))
    shape = shape if len(shape) > 1 else (1,) + shape
    x = rows_of(gen, shape[0] if len(shape) == 2 else shape[0] * shape[1], shape[-1], dtype).reshape(shape)
    codes, scales = ops.quantize_f8(x, 1)
    want, ws = o.quantize_rows(x.reshape(-1, shape[-1]))
    assert torch.equal(codes.double().reshape(want.shape), want) and torch.equal(scales.double().reshape(ws.shape), ws)
    back = (want * ws.repeat_interleave(128, 1)[:, :shape[-1]]).reshape(shape)
    assert torch.equal(ops.dequantize_f8(codes, scales, torch.float32), back.float()) and torch.equal(ops.dequantize_f8(codes, scales), back.float().bfloat16())
    codes, scales = ops.quantize_f8(x)
    for part, c, s in zip(*(t.reshape((-1,) + tuple(t.shape[-2:])) for t in (x, codes, scales))):
        for i in range(0, part.shape[0], 128):
            for j in range(0, part.shape[1], 128):
                block = part[i:i + 128, j:j + 128].double().reshape(1, -1)
                scale = (block.abs().max() / 448).float().double()
                assert s[i // 128, j // 128].double() == scale
                want = o.to_e4m3((block / scale).float().double()) if scale > 0 else torch.zeros_like(block)
                assert torch.equal(c[i:i + 128, j:j + 128].double().reshape(1, -1), want)
    assert torch.equal(ops.dequantize_f8(codes, scales, torch.float32), (codes.double() * o.spread(scales, *shape[-2:])).float())


def test_codes_at_the_edges():
    from mlx_rs_amd import ops
    x = torch.randn(12, 256, device="cuda")
    x[0, 3], x[1, 200], x[2, 7] = float("inf"), float("nan"), -float("inf")
    x[3] = 0
    x[4] *= 1e-38  # (scales among the least floats)
    x[5] = torch.linspace(-1, 1, 256, device="cuda") * 5e-43
    x[6] *= 1e37
    x[7] = 1e-45
    x[8] = torch.arange(256, device="cuda") - 128.0
    x[9] *= 2.0 ** -79
    x[10, :128], x[10, 0] = 2.0 ** -10, 448.0  # half of the least code: to the even one, zero
    x[11, :128], x[11, 0] = 3 * 2.0 ** -10, 448.0
    codes, scales = ops.quantize_f8(x, 1)
    want, ws = o.quantize_rows(x)
    assert torch.equal(codes.double(), want) and torch.equal(scales.isnan(), ws.isnan()) and torch.equal(scales.double().nan_to_num(), ws.nan_to_num())
    assert scales[0].isnan().tolist() == [True, False] and scales[1].isnan().tolist() == [False, True] and not codes[0, :128].double().any()
    assert not codes[10, 1:128].double().any() and (codes[11, 1:128].double() == 2.0 ** -8).all()


# ---------------------------------------------------------------- linear layers
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(1, 16), (17, 112), (200, 128), (257, 144), (384, 1040), (640, 2048)])
@pytest.mark.parametrize("M", [1, 2, 15, 17, 33, 64, 65, 130, 300])
def test_linear(M, N, K, dtype):
    from mlx_rs_amd import ops
    gen = gen_of(M * N + K)
    w, s = o.bank(gen, N, K)
    x = rows_of(gen, M, K, dtype)
    bias = torch.randn(N, generator=gen, device="cuda").to(dtype)
    codes, scales = o.quantize_rows(x)
    for b in (None, bias):
        want, off = o.product(codes, scales, w.double(), s, b, dtype)
        o.within(ops.linear_f8(x, w, s, b), want, off, f"linear {M} {N} {K} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(1, 16), (17, 112), (200, 128), (257, 400), (1040, 384)])
@pytest.mark.parametrize("M", [1, 17, 65, 200, 300])
def test_input_gradient(M, N, K, dtype):
    from mlx_rs_amd import ops
    gen = gen_of(M * N + K)
    w, s = o.bank(gen, N, K)
    dy = rows_of(gen, M, N, dtype)
    codes, scales = o.quantize_rows(dy)
    want, off = o.product(codes, scales, w.double().t(), s.t(), None, dtype)
    o.within(ops.linear_f8(dy, w, s, transpose=False), want, off, f"gradient {M} {N} {K} {dtype}")


def test_leading_axes_and_views():
    from mlx_rs_amd import ops
    gen = gen_of(5)
    w, s = o.bank(gen, 48, 64)
    x = torch.randn(2, 3, 65, generator=gen, device="cuda")[..., 1:].contiguous().bfloat16()
    y = ops.linear_f8(x, w, s)
    assert y.shape == (2, 3, 48) and torch.equal(y.reshape(6, 48), ops.linear_f8(x.reshape(6, 64), w, s))
    assert torch.equal(ops.linear_f8(x[1, 2], w, s), ops.linear_f8(x[1, 2][None], w, s)[0])
    shifted = torch.empty(6 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:]
    shifted.copy_(x.reshape(-1))
    assert torch.equal(ops.linear_f8(shifted.reshape(6, 64), w, s), y.reshape(6, 48))
    assert ops.linear_f8(x[:0], w, s).shape == (0, 3, 48)


@pytest.mark.parametrize("M", [3, 300])
def test_a_row_that_is_not_finite_stays_its_own(M):
    from mlx_rs_amd import ops
    gen = gen_of(M)
    w, s = o.bank(gen, 80, 256)
    x = rows_of(gen, M, 256, torch.bfloat16)
    y = ops.linear_f8(x, w, s)
    x[1, 5], x[2, 200] = float("nan"), float("inf")
    z = ops.linear_f8(x, w, s)
    assert z[1:3].isnan().all() and torch.equal(z[3:], y[3:]) and torch.equal(z[0], y[0])


# ---------------------------------------------------------------- grouped
def grouped_oracle(x, w, s, ends, transpose, dtype):
    codes, scales = o.quantize_rows(x)
    outer = w.shape[1] if transpose else w.shape[2]
    y = torch.zeros(x.shape[0], outer, dtype=torch.float64, device="cuda")
    off = torch.zeros_like(y)
    for e in range(w.shape[0]):
        at = slice(ends[e], ends[e + 1])
        if ends[e] < ends[e + 1]:
            y[at], off[at] = o.product(codes[at], scales[at], w[e].double() if transpose else w[e].double().t(), s[e] if transpose else s[e].t(), None, dtype)
    return y, off


COUNTS = {"one row": [0, 1, 0], "few": [2, 0, 3, 1, 0, 17, 4], "ragged": [70, 0, 1, 300, 64, 65, 0, 128], "one expert": [140], "long": [700, 3, 257, 0, 256],
          "nobody": [0, 0]}


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("behind", [0, 5, 90])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped(counts, behind, transpose, dtype):
    from mlx_rs_amd import ops
    counts = COUNTS[counts]
    N, K = 272, 400
    gen = gen_of(sum(counts) + behind)
    w, s = o.bank(gen, N, K, len(counts))
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    R = ends[-1] + behind
    x = rows_of(gen, R, K if transpose else N, dtype)
    y = ops.grouped_linear_f8(x, w, s, torch.tensor(ends, device="cuda", dtype=torch.int32), transpose)
    want, off = grouped_oracle(x, w, s, ends, transpose, dtype)
    assert y.shape == want.shape and not y[ends[-1]:].any()
    if R:
        o.within(y, want, off, f"grouped {counts} {behind} {transpose} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", ["few", "ragged"])
def test_grouped_along_a_long_axis(counts, dtype):
    """Few tiles of many stages: blocks that share a tile's summed axis, rows of no expert among theirs."""
    from mlx_rs_amd import ops
    counts = COUNTS[counts]
    N, K = 2576, 144
    gen = gen_of(sum(counts))
    w, s = o.bank(gen, N, K, len(counts))
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    x = rows_of(gen, ends[-1] + 7, N, dtype)
    y = ops.grouped_linear_f8(x, w, s, torch.tensor(ends, device="cuda", dtype=torch.int32), False)
    want, off = grouped_oracle(x, w, s, ends, False, dtype)
    assert not y[ends[-1]:].any()
    o.within(y, want, off, f"along {counts} {dtype}")


def test_many_experts():
    from mlx_rs_amd import ops
    gen = gen_of(1)
    E, N, K = 512, 32, 128
    w, s = o.bank(gen, N, K, E)
    pick = torch.sort(torch.randint(0, E, (1500,), generator=gen, device="cuda"))[0]
    ends = [0] + torch.bincount(pick, minlength=E).cumsum(0).tolist()
    x = rows_of(gen, 1500, K, torch.bfloat16)
    offsets = torch.tensor(ends, device="cuda", dtype=torch.int32)
    want, off = grouped_oracle(x, w, s, ends, True, torch.bfloat16)
    o.within(ops.grouped_linear_f8(x, w, s, offsets), want, off)
    dy = rows_of(gen, 1500, N, torch.bfloat16)
    want, off = grouped_oracle(dy, w, s, ends, False, torch.bfloat16)
    o.within(ops.grouped_linear_f8(dy, w, s, offsets, False), want, off)


@pytest.mark.parametrize("offsets", [[0, 9, 3], [-5, 2, 8], [2 ** 31 - 1, 0, 4], [0, 100, 200]])
@pytest.mark.parametrize("R", [8, 400])
def test_offsets_out_of_order_or_range_reach_no_other_memory(R, offsets):
    """What comes out is nobody's business; the call ends and its neighbours stay what they were."""
    from mlx_rs_amd import ops
    gen = gen_of(R)
    w, s = o.bank(gen, 64, 128, 2)
    x = rows_of(gen, R, 128, torch.bfloat16)
    offsets = torch.tensor(offsets, device="cuda", dtype=torch.int32)
    for transpose, rows in ((True, x), (False, x[:, :64].contiguous())):
        assert ops.grouped_linear_f8(rows, w, s, offsets, transpose).shape == (R, 64 if transpose else 128)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- experts
def experts_oracle(x, inds, weights, gate, up, down, dout=None):
    """The forward result, or dx and dweights, in 64 bits, with what each may be off by: a code of a computed value may be the next one where its quotient is nearer to the
    border of two codes than what the value may be off by."""
    T, H = x.shape
    k, E, inter = inds.shape[1], gate[0].shape[0], gate[0].shape[1]
    half = o.HALF_STEP[x.dtype]
    codes, scales = o.quantize_rows(x)
    out, off = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dw, dw_off = torch.zeros(T, k, dtype=torch.float64, device="cuda"), torch.zeros(T, k, dtype=torch.float64, device="cuda")
    if dout is not None:
        dcodes, dscales = o.quantize_rows(dout)
    sums = torch.float32 if dout is not None or x.dtype == torch.float16 else torch.bfloat16  # the gradients' first products come in float32, and gate and up of float16 tokens

    def next_codes(v, v_off):
        """Codes of v, and by what the values that they stand for may be off from another right result's."""
        q, s = o.quantize_rows(v)
        wide = s.repeat_interleave(128, 1)[:, :v.shape[1]]
        quotient = v / wide
        most = torch.stack([v[:, c].abs().amax(-1) for c in o.runs_of(v)], 1).repeat_interleave(128, 1)[:, :v.shape[1]]
        far = torch.stack([v_off[:, c].amax(-1) for c in o.runs_of(v)], 1).repeat_interleave(128, 1)[:, :v.shape[1]] / most  # (of the scale)
        q_off = v_off / wide + quotient.abs() * (far + 2.0 ** -22)
        step = torch.exp2(torch.frexp(quotient)[1].double().sub(1).clamp(min=-6) - 3)
        may = ((quotient - q).abs() + q_off >= step / 2 * (1 - 2.0 ** -20))
        return q, s, torch.where(may, step * 1.01 + q_off, 0.0) * wide + (q * wide).abs() * (far + 2.0 ** -22)

    for e in range(E):
        t, slot = (inds == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        g, g_off = o.product(codes[t], scales[t], gate[0][e].double(), gate[1][e], None, sums)
        u, u_off = o.product(codes[t], scales[t], up[0][e].double(), up[1][e], None, sums)
        sig = torch.sigmoid(g)
        h = g * sig * u
        slope = (sig * (1 + g * (1 - sig))).abs()
        few = 2.0 ** -24 * (8 + 2 * g.abs())  # the exponential's argument is rounded
        h_off = (slope * u.abs() + u_off) * g_off + (g * sig).abs() * u_off + h.abs() * few
        w = weights[t, slot].double()[:, None]
        if dout is None:
            q, s, q_off = next_codes(h, h_off)
            y, y_off = o.product(q, s, down[0][e].double(), down[1][e], None, x.dtype)
            y_off = y_off + q_off @ (down[0][e].double() * o.spread(down[1][e], H, inter)).abs().t()
            y_off = y_off + half * (y.abs() + y_off)  # (rounded ahead of the sum over the slots)
            out.index_add_(0, t, w * y)
            off.index_add_(0, t, w.abs() * (y_off + 2.0 ** -22 * y.abs()))
            continue
        dh, dh_off = o.product(dcodes[t], dscales[t], down[0][e].double().t(), down[1][e].t(), None, torch.float32)
        dw[t, slot] = (dh * h).sum(-1)
        dw_off[t, slot] = (dh_off * h.abs() + dh.abs() * h_off + (inter + 4) * 2.0 ** -24 * (dh * h).abs()).sum(-1)
        dh, dh_off = dh * w, dh_off * w.abs()
        parts = []
        for v, by_dh, by_u, by_g in ((dh * u * sig * (1 + g * (1 - sig)), u * sig * (1 + g * (1 - sig)), dh * sig * (1 + g * (1 - sig)), dh * u),
                                     (dh * g * sig, g * sig, torch.zeros_like(g), dh * slope)):
            parts.append(next_codes(v, (by_dh.abs() * dh_off + by_u.abs() * u_off + by_g.abs() * g_off * 1.1 + v.abs() * few + (dh * u).abs() * few) * 1.01))
        for (q, s, q_off), (c, cs) in zip(parts, (gate, up)):
            wide = c[e].double() * o.spread(cs[e], inter, H)
            y, y_off = o.product(q, s, c[e].double().t(), cs[e].t(), None, x.dtype)
            out.index_add_(0, t, y)
            off.index_add_(0, t, y_off + q_off @ wide.abs() + half * (y.abs() + y_off) * 1.01 + 2.0 ** -22 * y.abs())
    return (out, off) if dout is None else (out, off, dw, dw_off)


EXPERTS = [(1, 1, 1, 16, 16), (1, 8, 128, 256, 192), (5, 2, 4, 144, 272), (40, 2, 4, 256, 128), (300, 2, 4, 272, 400), (700, 1, 2, 128, 256), (130, 4, 64, 128, 112), (3, 2, 8, 256, 2064), (20, 2, 3, 1296, 1040), (40, 1, 64, 256, 144)]


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("shape", EXPERTS)
def test_experts_and_their_gradients(shape, dtype, padded):
    from mlx_rs_amd import ops
    T, k, E, H, inter = shape
    gen = gen_of(T + H)
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").to(dtype) for _ in range(2))
    inds = torch.rand((T, E), generator=gen, device="cuda").topk(k, -1)[1].to(torch.int32)
    if padded:
        inds[::3] = E
        inds[1::3, k - 1] = -1
        x[::3] = float("nan")  # padding's rows have no part in anything
        dout[::3] = float("inf")
    for wtype in (torch.bfloat16, torch.float32):
        w = torch.rand((T, k), generator=gen, device="cuda").to(wtype)
        y = ops.switch_glu_f8(x, inds, w, gate, up, down)
        want, off = experts_oracle(x, inds, w, gate, up, down)
        o.within(y, want, off, f"experts {shape} {dtype}")
        dx, dw = ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down)
        want, off, want_w, off_w = experts_oracle(x, inds, w, gate, up, down, dout)
        o.within(dx, want, off, f"dx {shape} {dtype}")
        o.within(dw, want_w, off_w, f"dweights {shape} {dtype}")
        if padded:
            assert not y[::3].any() and not dx[::3].any() and not dw[::3].any() and not dw[1::3, k - 1].any()


def test_the_same_expert_twice_and_nobody_at_all():
    from mlx_rs_amd import ops
    gen = gen_of(3)
    gate, up, down = o.bank(gen, 64, 128, 3), o.bank(gen, 64, 128, 3), o.bank(gen, 128, 64, 3)
    x = torch.randn((2, 128), generator=gen, device="cuda").bfloat16()
    twice = torch.tensor([[1, 1], [2, 2]], device="cuda", dtype=torch.int32)
    w = torch.tensor([[0.25, 0.5], [1.0, 0.0]], device="cuda")
    want, off = experts_oracle(x, twice, w, gate, up, down)
    o.within(ops.switch_glu_f8(x, twice, w, gate, up, down), want, off)
    nobody = torch.full_like(twice, 3)
    assert not ops.switch_glu_f8(x, nobody, w, gate, up, down).any()
    assert not any(t.any() for t in ops.switch_glu_f8_grad(x, x, nobody, w, gate, up, down))
    assert ops.switch_glu_f8(x[:0], twice[:0], w[:0], gate, up, down).shape == (0, 128)


@pytest.mark.parametrize("T,k,H", [(1, 4, 1024), (1, 8, 256), (2, 4, 4096), (4, 2, 1040), (3, 2, 144), (1, 16, 2048), (2, 32, 2048), (4, 8, 1024), (7, 3, 1040), (16, 16, 128), (40, 8, 256)])
def test_few_tokens_all_at_one_expert(T, k, H):
    """A matrix with more rows than tokens: pieces as long as the kernels for a few rows take."""
    from mlx_rs_amd import ops
    gen = gen_of(T)
    gate, up, down = o.bank(gen, 144, H, 8), o.bank(gen, 144, H, 8), o.bank(gen, H, 144, 8)
    x = torch.randn((T, H), generator=gen, device="cuda").bfloat16()
    inds = torch.full((T, k), 5, device="cuda", dtype=torch.int32)
    inds[0, 0] = 2
    inds[-1, k // 2] = -1  # (and a slot that names none)
    w = torch.rand((T, k), generator=gen, device="cuda")
    want, off = experts_oracle(x, inds, w, gate, up, down)
    o.within(ops.switch_glu_f8(x, inds, w, gate, up, down), want, off)


@pytest.mark.parametrize("T", [3, 300])
def test_a_result_past_float32_leaves_those_beside_it(T):
    """Down's product is infinite in one column and near the end of float32 in the others.  h is 128 equal values, all codes 448, and every product of a power of two: what is
    left are silu(16) * 16 = 256 (1 - 2^-23), the roundings of the scales (2^-24 each), of a result held in 11 bits and of the sum to bfloat16."""
    from mlx_rs_amd import ops
    codes = torch.ones((2, 128, 128), device="cuda")
    flat = (codes.to(o.F8), torch.full((2, 1, 1), 0.125, device="cuda"))
    codes[:, 5] = 448.0
    codes[:, 6] = -448.0
    down = (codes.to(o.F8), torch.full((2, 1, 1), 2.0 ** 105, device="cuda"))
    x = torch.ones((T, 128), device="cuda", dtype=torch.bfloat16)
    inds = torch.tensor([0, 1], device="cuda", dtype=torch.int32).expand(T, 2).contiguous()
    y = ops.switch_glu_f8(x, inds, torch.full((T, 2), 0.25, device="cuda"), flat, flat, down).double()
    assert (y[:, 5] == float("inf")).all() and (y[:, 6] == -float("inf")).all()
    rest = torch.cat((y[:, :5], y[:, 7:]), 1) * 2.0 ** -119
    assert (rest - 1.0).abs().max() <= 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20


@pytest.mark.parametrize("T", [3, 200])
def test_experts_by_differences(T):
    """dweights is the change of sum(out * dout) with a weight, in the forward's own numbers but for their roundings: out is linear in the weights."""
    from mlx_rs_amd import ops
    gen = gen_of(T)
    E, H, inter, k = 4, 256, 384, 2
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").bfloat16() for _ in range(2))
    inds = torch.rand((T, E), generator=gen, device="cuda").topk(k, -1)[1].to(torch.int32)
    w = torch.rand((T, k), generator=gen, device="cuda")
    _, dw = ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down)
    for s in range(k):
        one = torch.zeros_like(w)
        one[:, s] = 1.0
        y = ops.switch_glu_f8(x, inds, one, gate, up, down).double()
        change = (y * dout.double()).sum(-1)
        # h and dout are in e4m3 on one side only: each term off by up to 2^-4 of its size, H of them at random (and bfloat16's roundings)
        bound = 6 * 2.0 ** -4 * (y.square().sum(-1) * dout.double().square().mean(-1)).sqrt() + 1e-9
        assert ((dw[:, s].double() - change).abs() <= bound).all()


def test_a_run_of_them_is_the_experts():
    """Sorted tokens through grouped layers and back, as a program with its own activation would, against the one call."""
    from mlx_rs_amd import ops
    gen = gen_of(9)
    T, k, E, H, inter = 150, 3, 6, 256, 256
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x = torch.randn((T, H), generator=gen, device="cuda").bfloat16()
    logits = torch.randn((T, E), generator=gen, device="cuda")
    inds, w = ops.select_experts(logits, k)
    inds[::7] = E
    rows, order, inverse, offsets = ops.sort_tokens(x, inds, E)
    g, u = ops.grouped_linear_f8(rows.float(), *gate, offsets), ops.grouped_linear_f8(rows.float(), *up, offsets)
    y = ops.grouped_linear_f8(torch.nn.functional.silu(g) * u, *down, offsets)
    out = ops.unsort_tokens(y, w, inverse)
    one = ops.switch_glu_f8(x, inds, w, gate, up, down)
    want, off = experts_oracle(x, inds, w, gate, up, down)
    o.within(out, want, off, "one after the other")
    o.within(one, want, off, "at once")
    # and the way back
    dout = torch.randn((T, H), generator=gen, device="cuda").bfloat16()
    dy, dw = ops.unsort_tokens_grad(dout.float(), y, w, inverse)
    dh = ops.grouped_linear_f8(dy, *down, offsets, False)
    sig = torch.sigmoid(g)
    drows = ops.grouped_linear_f8(dh * u * sig * (1 + g * (1 - sig)), *gate, offsets, False) + ops.grouped_linear_f8(dh * g * sig, *up, offsets, False)
    dx = ops.sort_tokens_grad(drows, inverse)
    once, once_w = ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down)
    # (the weighted gradient is rounded to e4m3 on one way, the plain one on the other: each value is off by up to 2^-4, 256 of a sum at random)
    assert (dx - once.float()).norm() <= 0.06 * dx.norm() and (dw.float() - once_w.float()).norm() <= 0.06 * dw.float().norm()


@pytest.mark.parametrize("T", [2, 200])
def test_captured_and_replayed_on_another_stream(T):
    from mlx_rs_amd import ops
    gen = gen_of(T)
    E, H, inter, k = 8, 256, 272, 2
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").bfloat16() for _ in range(2))
    inds = torch.randint(-1, E + 1, (T, k), generator=gen, device="cuda", dtype=torch.int32)
    w = torch.rand((T, k), generator=gen, device="cuda")
    lw, ls = o.bank(gen, 80, H)
    offsets = torch.tensor([0, 1, 1, T, T, T, T, T, T], device="cuda", dtype=torch.int32)

    def run():
        return (ops.switch_glu_f8(x, inds, w, gate, up, down), *ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down), ops.linear_f8(x, lw, ls),
                ops.grouped_linear_f8(x, *gate, offsets), ops.grouped_linear_f8(x, *down, offsets, False))

    run()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(run())
    side = torch.cuda.Stream()
    for _ in range(4):
        x.copy_(torch.randn((T, H), generator=gen, device="cuda"))
        inds.copy_(torch.randint(-1, E + 1, (T, k), generator=gen, device="cuda", dtype=torch.int32))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        want = run()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    import mlx_rs_amd as m
    from mlx_rs_amd import ops
    gen = gen_of(0)
    w, s = o.bank(gen, 256, 128)
    bw, bs = o.bank(gen, 256, 128, 2)
    x, offsets = torch.zeros(3, 128, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int32)
    g, d = o.bank(gen, 64, 128, 2), o.bank(gen, 128, 64, 2)
    xb, inds, rw = x.bfloat16(), torch.zeros(3, 2, device="cuda", dtype=torch.int32), torch.zeros(3, 2, device="cuda")
    odd = torch.zeros(24, 24, device="cuda").to(o.F8)
    one = torch.ones(1, 1, device="cuda")
    for needle, call in [("block_rows", lambda: ops.quantize_f8(x, 64)), ("w must be", lambda: ops.quantize_f8(x[0])), ("bfloat16", lambda: ops.quantize_f8(x.double())),
                         ("do not go", lambda: ops.dequantize_f8(w, s[:1])), ("expected dtype", lambda: ops.dequantize_f8(x, s)), ("dtype", lambda: ops.dequantize_f8(w, s, torch.int8)),
                         ("scales must be", lambda: ops.linear_f8(x, w, s[:1])), ("x must be", lambda: ops.linear_f8(x[:, :64].contiguous(), w, s)),
                         ("expected dtype", lambda: ops.linear_f8(x, w.float(), s)), ("linear_bias", lambda: ops.linear_f8(x, w, s, x[0])),
                         ("transpose", lambda: ops.linear_f8(torch.zeros(3, 256, device="cuda"), w, s, x[0], transpose=False)),
                         ("multiple of 16", lambda: ops.linear_f8(x[:, :24].contiguous(), odd, one)), ("multiple of 16", lambda: ops.linear_f8(x[:, :24].contiguous(), odd, one, transpose=False)),
                         ("contiguous", lambda: ops.linear_f8(x, w.t(), s)), ("offsets", lambda: ops.grouped_linear_f8(x, bw, bs, offsets[:2])),
                         ("rows must be", lambda: ops.grouped_linear_f8(x, bw, bs, offsets, False)), ("w must be", lambda: ops.grouped_linear_f8(x, w, s, offsets)),
                         ("dtype must be", lambda: ops.switch_glu_f8(x, inds, rw, g, g, d)), ("down must be", lambda: ops.switch_glu_f8(xb, inds, rw, g, g, g)),
                         ("inds and weights", lambda: ops.switch_glu_f8(xb, inds[:2], rw, g, g, d)), ("expected dtype", lambda: ops.switch_glu_f8(xb, inds.long(), rw, g, g, d)),
                         ("dout must be", lambda: ops.switch_glu_f8_grad(xb[:2], xb, inds, rw, g, g, d)), ("expected dtype", lambda: ops.switch_glu_f8_grad(x, xb, inds, rw, g, g, d)),
                         ("experts", lambda: ops.switch_glu_f8(xb, inds, rw, g, tuple(t[:1] for t in g), d)), ("device tensor", lambda: ops.linear_f8(x, w.cpu(), s))]:
        with pytest.raises(m.MoeError, match=needle):
            call()


def test_the_module_is_the_call():
    import mlx_rs_amd as m
    gen = gen_of(4)
    dense = [torch.randn(s, generator=gen, device="cuda").bfloat16() * 0.05 for s in ((3, 200 // 8 * 16, 256), (3, 400, 256), (3, 256, 400))]
    block = m.SwitchGluF8(*(m.F8SwitchLinear.quantize(w) for w in dense))
    x, dout = (torch.randn((2, 5, 256), generator=gen, device="cuda").bfloat16() for _ in range(2))
    inds, w = m.ops.select_experts(torch.randn((2, 5, 3), generator=gen, device="cuda"), 2)
    banks = [m.ops.quantize_f8(d) for d in dense]
    block.training_mode(True)
    assert block.training and torch.equal(block(x, inds, w), m.ops.switch_glu_f8(x, inds, w, *banks))
    flat = m.ops.switch_glu_f8(x.reshape(10, 256), inds.reshape(10, 2), w.reshape(10, 2), *banks)
    assert torch.equal(block.forward(x, inds, w).reshape(10, 256), flat)
    assert all(torch.equal(a, b) for a, b in zip(block.gradient(dout, x, inds, w), m.ops.switch_glu_f8_grad(dout, x, inds, w, *banks)))

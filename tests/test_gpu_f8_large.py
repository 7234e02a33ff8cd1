"""The e4m3 operators at the sizes of prompts and training batches: large tiles, several of them on each side, blocks that share a tile, experts behind the sorting of many pairs; memory
around what a call may write."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402
from test_gpu_f8 import DTYPES, experts_oracle, gen_of, rows_of  # noqa: E402

pytestmark = pytest.mark.gpu

# rows, columns, summed axis: of which tiles and parts are made, test_f8_rule.py says
DENSE = [(4096, 2100, 1040), (3000, 2100, 1040), (16500, 270, 400), (4100, 4112, 272), (4096, 600, 8208), (2100, 300, 16384), (700, 300, 4112)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", DENSE)
def test_linear(M, N, K, dtype):
    from mlx_rs_amd import ops
    gen = gen_of(M + N)
    w, s = o.bank(gen, N, K)
    x = rows_of(gen, M, K, dtype)
    bias = torch.randn(N, generator=gen, device="cuda").to(dtype)
    codes, scales = o.quantize_rows(x)
    want, off = o.product(codes, scales, w.double(), s, bias, dtype)
    o.within(ops.linear_f8(x, w, s, bias), want, off, f"linear {M} {N} {K} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", DENSE)
def test_input_gradient(M, N, K, dtype):
    from mlx_rs_amd import ops
    N = (N + 15) // 16 * 16  # (the result's columns, weights' rows of whole sixteens)
    gen = gen_of(M + K)
    w, s = o.bank(gen, K - 5, N)
    dy = rows_of(gen, M, K - 5, dtype)
    codes, scales = o.quantize_rows(dy)
    want, off = o.product(codes, scales, w.double().t(), s.t(), None, dtype)
    o.within(ops.linear_f8(dy, w, s, transpose=False), want, off, f"gradient {M} {N} {K} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("transpose", [True, False])
def test_grouped_by_many_pieces_and_columns(transpose, dtype):
    """More pieces than are dealt one by one, several tiles of columns, rows of no matrix behind them."""
    from mlx_rs_amd import ops
    gen = gen_of(6)
    E, N, K = 24, 608, 528
    w, s = o.bank(gen, N, K, E)
    counts = [(37 * e * e) % 700 for e in range(E)]
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    x = rows_of(gen, ends[-1] + 300, K if transpose else N, dtype)
    y = ops.grouped_linear_f8(x, w, s, torch.tensor(ends, device="cuda", dtype=torch.int32), transpose)
    codes, scales = o.quantize_rows(x)
    assert not y[ends[-1]:].any()
    for e in range(E):
        at = slice(ends[e], ends[e + 1])
        if counts[e]:
            want, off = o.product(codes[at], scales[at], w[e].double() if transpose else w[e].double().t(), s[e] if transpose else s[e].t(), None, dtype)
            o.within(y[at], want, off, f"grouped {e} {transpose} {dtype}")


SHARED = (507, 250, 1040)  # rows by one matrix: listed pieces of 256 rows, a tile of which four blocks share (of 128 rows and one block in float16 and float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_by_blocks_that_share_large_tiles(dtype):
    from mlx_rs_amd import ops
    M, N, K = SHARED
    gen = gen_of(7)
    w, s = o.bank(gen, N, K, 1)
    x = rows_of(gen, M, K, dtype)
    y = ops.grouped_linear_f8(x, w, s, torch.tensor([0, M - 7], device="cuda", dtype=torch.int32))
    codes, scales = o.quantize_rows(x)
    want, off = o.product(codes[:M - 7], scales[:M - 7], w[0].double(), s[0], None, dtype)
    o.within(y[:M - 7], want, off, f"shared {dtype}")
    assert not y[M - 7:].any()


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("T,k,E,H,inter", [(600, 4, 8, 608, 272), (1500, 2, 40, 272, 400), (2100, 1, 1, 528, 144)])
def test_experts_and_their_gradients(T, k, E, H, inter, dtype):
    """More than 2048 pairs, padding among them."""
    from mlx_rs_amd import ops
    gen = gen_of(T + H)
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").to(dtype) for _ in range(2))
    inds = torch.rand((T, E), generator=gen, device="cuda").topk(k, -1)[1].to(torch.int32)
    inds[::7] = E
    inds[1::5, k - 1] = -1
    x[::7] = float("nan")
    dout[::7] = float("inf")
    w = torch.rand((T, k), generator=gen, device="cuda")
    y = ops.switch_glu_f8(x, inds, w, gate, up, down)
    want, off = experts_oracle(x, inds, w, gate, up, down)
    o.within(y, want, off, f"experts {T} {dtype}")
    dx, dw = ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down)
    want, off, want_w, off_w = experts_oracle(x, inds, w, gate, up, down, dout)
    o.within(dx, want, off, f"dx {T} {dtype}")
    o.within(dw, want_w, off_w, f"dweights {T} {dtype}")
    assert not y[::7].any() and not dx[::7].any() and not dw[::7].any() and not dw[1::5, k - 1].any()


@pytest.mark.parametrize("E", [1, 2, 8, 15, 16])
@pytest.mark.parametrize("T,k", [(1025, 2), (3000, 1), (700, 5)])
def test_many_pairs_of_few_experts(T, k, E):
    from mlx_rs_amd import ops
    gen = gen_of(T)
    inds = torch.randint(-1, E + 1, (T, k), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn((T, 24), generator=gen, device="cuda")
    rows, order, inverse, offsets = ops.sort_tokens(x, inds, E)
    want = o.sort(inds.cpu(), E)
    assert order.tolist() == want[0] and inverse.reshape(-1).tolist() == want[1] and offsets.tolist() == want[2]
    expect = x[order.long() // k].clone()
    expect[want[2][-1]:] = 0
    assert torch.equal(rows, expect)


def test_sorted_rows_of_more_than_two_to_the_31_values():
    from mlx_rs_amd import ops
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of memory")
    gen = gen_of(8)
    T, k, E, H = 70000, 8, 64, 4096
    inds = torch.randint(-1, E, (T, k), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn((T, H), generator=gen, device="cuda").bfloat16()
    rows, order, inverse, offsets = ops.sort_tokens(x, inds, E)
    named = int(offsets[-1])
    key = torch.where(inds.reshape(-1) < 0, E, inds.reshape(-1))
    assert torch.equal(order.long(), torch.sort(key, stable=True)[1]) and named < T * k
    for r in range(0, T * k, 50000):
        part = slice(r, min(r + 50000, T * k))
        token = x[order[part].long() // k]
        token[max(named - r, 0):] = 0
        assert torch.equal(rows[part], token)
    w = torch.rand((T, k), generator=gen, device="cuda")
    y, dx = ops.unsort_tokens(rows, w, inverse), ops.sort_tokens_grad(rows, inverse)
    drows, dw = ops.unsort_tokens_grad(x, rows, w, inverse)
    for t in (0, 1, 35000, T - 1):
        mine = (inverse[t] >= 0)
        terms = x[t].double() * torch.where(mine, w[t], 0.0).double()[:, None]
        o.within(y[t], terms.sum(0), terms.abs().sum(0) * (k + 1) * 2.0 ** -24, "unsort")
        o.within(dx[t], x[t].double() * int(mine.sum()), x[t].double().abs() * k * (k + 1) * 2.0 ** -24, "sort's gradient")
        at = torch.where(mine, inverse[t], -1 - inverse[t]).long()
        o.within(drows[at], terms, terms.abs() * 2.0 ** -24, "the rows' gradient")
        square = x[t].double().square().sum()
        o.within(dw[t], torch.where(mine, square, 0.0), torch.where(mine, square, 0.0) * (H + 1) * 2.0 ** -24, "the weights' gradient")


@pytest.mark.parametrize("offsets", [[0, 9, 3], [-5, 2, 8], [2 ** 31 - 1, 0, 4], [0, 100, 200], [3, 3, 3], [0, 5, 8]])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("R", [8, 400])
def test_offsets_out_of_order_or_range_write_nothing_else(R, transpose, offsets):
    """The result, the workspace and the operands lie in one allocation, with marked memory between them; only the result and the workspace change."""
    import ctypes as C
    import mlx_rs_amd as m
    lib = m.load_library()
    gen = gen_of(R)
    N, K, E = 64, 128, 2
    wide = K if transpose else N
    w, s = o.bank(gen, N, K, E)
    x = rows_of(gen, R, wide, torch.bfloat16)
    out = N if transpose else K
    need = C.c_size_t()
    assert lib.mi_moe_linear_f8_workspace_size(R, out, wide, C.byref(need)) == 0
    held = [x.view(torch.uint8).reshape(-1), w.view(torch.uint8).reshape(-1), s.view(torch.uint8).reshape(-1), torch.tensor(offsets, device="cuda", dtype=torch.int32).view(torch.uint8)]
    sizes = [t.numel() for t in held] + [R * out * 2, need.value]
    guard, places, end = 4096, [], 4096
    for n in sizes:
        places.append(end)
        end += (n + 255) // 256 * 256 + guard
    memory = torch.randint(0, 256, (end,), generator=gen, device="cuda", dtype=torch.uint8)
    for t, at in zip(held, places):
        memory[at:at + t.numel()] = t
    before = memory.clone()
    p = [memory.data_ptr() + at for at in places]
    status = lib.mi_moe_grouped_linear_f8(p[0], p[1], p[2], p[3], R, E, out, wide, int(transpose), 0, p[4], p[5], need.value, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0
    for at, n in zip(places[4:], sizes[4:]):
        before[at:at + n] = memory[at:at + n]
    assert torch.equal(memory, before)

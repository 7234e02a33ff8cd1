"""Tokens sorted by expert and back, weighted, and their gradients, against their definitions."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def routing(gen, T, k, E, padded):
    inds = torch.randint(0, E, (T, k), generator=gen, device="cuda", dtype=torch.int32)
    if padded:
        u = torch.rand((T, k), generator=gen, device="cuda")
        inds[u < 0.1] = E
        inds[u > 0.95] = -1
        inds[u > 0.99] = 2 ** 31 - 1
    return inds


# (T, k, E, H): one token, odd widths, both sides of where the kernels change (2048 pairs), the most experts and slots, rows of several passes
SHAPES = [(1, 1, 1, 1), (1, 8, 128, 2048), (5, 3, 7, 33), (256, 8, 128, 64), (257, 8, 128, 64), (64, 32, 512, 24), (700, 6, 64, 515), (3, 2, 8, 9000), (3000, 2, 512, 40)]


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sort_and_back(shape, dtype, padded):
    from mlx_rs_amd import ops
    T, k, E, H = shape
    gen = torch.Generator(device="cuda").manual_seed(T + k)
    inds = routing(gen, T, k, E, padded)
    x = torch.randn((T, H), generator=gen, device="cuda").to(dtype)
    rows, order, inverse, offsets = ops.sort_tokens(x, inds, E)
    want = o.sort(inds.cpu(), E)
    assert order.tolist() == want[0] and inverse.reshape(-1).tolist() == want[1] and offsets.tolist() == want[2]
    expect = x[order.long() // k].clone()
    expect[want[2][-1]:] = 0
    assert torch.equal(rows, expect)

    named = (inverse >= 0)[..., None]
    at = inverse.long().clamp(min=0)
    rows = torch.randn((T * k, H), generator=gen, device="cuda").to(dtype)
    rows[want[2][-1]:] = float("nan")  # what nobody names has no part in anything
    picked = torch.where(named, rows.double()[at], 0.0)
    off = picked.abs().sum(1) * (k + 1) * 2.0 ** -24
    o.within(ops.sort_tokens_grad(rows, inverse), picked.sum(1), off, "sort's gradient")
    for wtype in DTYPES:
        w = torch.rand((T, k), generator=gen, device="cuda").to(wtype)
        w[inverse < 0] = float("inf")
        terms = torch.where(named, picked * w.double()[..., None], 0.0)
        o.within(ops.unsort_tokens(rows, w, inverse), terms.sum(1), terms.abs().sum(1) * (k + 1) * 2.0 ** -24, "unsort")
        dout = torch.randn((T, H), generator=gen, device="cuda").to(dtype)
        drows, dw = ops.unsort_tokens_grad(dout, rows, w, inverse)
        g = dout.double()[:, None] * torch.where(named, w.double()[..., None], 0.0)
        back = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        back[torch.where(inverse >= 0, inverse, -1 - inverse).reshape(-1).long()] = g.reshape(-1, H)
        o.within(drows, back, back.abs() * 2.0 ** -24, "the rows' gradient")
        dots = dout.double()[:, None] * picked
        o.within(dw, dots.sum(-1), dots.abs().sum(-1) * (H + 1) * 2.0 ** -24, "the weights' gradient")


def test_nobody_and_no_tokens():
    from mlx_rs_amd import ops
    x = torch.randn(4, 24, device="cuda").bfloat16()
    rows, order, inverse, offsets = ops.sort_tokens(x, torch.full((4, 2), 9, device="cuda", dtype=torch.int32), 9)
    assert not rows.any() and inverse.tolist() == [[-1, -2], [-3, -4], [-5, -6], [-7, -8]] and not offsets.any() and order.tolist() == list(range(8))
    assert not ops.unsort_tokens(torch.full_like(rows, float("nan")), torch.ones(4, 2, device="cuda"), inverse).any()
    drows, dw = ops.unsort_tokens_grad(x, rows, torch.ones(4, 2, device="cuda"), inverse)
    assert not drows.any() and not dw.any()
    none = torch.empty((0, 2), device="cuda", dtype=torch.int32)
    rows, order, inverse, offsets = ops.sort_tokens(x[:0], none, 9)
    assert rows.shape == (0, 24) and order.shape == (0,) and inverse.shape == (0, 2) and offsets.tolist() == [0] * 10
    assert ops.unsort_tokens(rows, torch.empty(0, 2, device="cuda"), inverse).shape == (0, 24)
    assert ops.sort_tokens_grad(rows, inverse).shape == (0, 24)
    assert [t.shape[0] for t in ops.unsort_tokens_grad(x[:0], rows, torch.empty(0, 2, device="cuda"), inverse)] == [0, 0]


def test_places_outside_the_rows_count_as_none():
    from mlx_rs_amd import ops
    rows = torch.randn(6, 16, device="cuda")
    inverse = torch.tensor([[0, 6], [2 ** 31 - 1, -2 ** 31], [3, -7]], device="cuda", dtype=torch.int32)
    w = torch.ones(3, 2, device="cuda")
    want = torch.stack([rows[0], torch.zeros(16, device="cuda"), rows[3]])
    assert torch.equal(ops.unsort_tokens(rows, w, inverse), want) and torch.equal(ops.sort_tokens_grad(rows, inverse), want)
    drows, dw = ops.unsort_tokens_grad(torch.ones(3, 16, device="cuda"), rows, w, inverse)
    assert (drows[[0, 3]] == 1).all() and (dw[:, 1] == 0).all() and dw[1, 0] == 0


@pytest.mark.parametrize("T", [40, 600])
def test_captured_and_replayed(T):
    from mlx_rs_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(T)
    k, E, H = 4, 16, 128
    x, inds = torch.randn((T, H), generator=gen, device="cuda").bfloat16(), routing(gen, T, k, E, True)
    w = torch.rand((T, k), generator=gen, device="cuda")

    def run():
        rows, order, inverse, offsets = ops.sort_tokens(x, inds, E)
        return rows, order, inverse, offsets, ops.unsort_tokens(rows, w, inverse), ops.sort_tokens_grad(rows, inverse), *ops.unsort_tokens_grad(x, rows, w, inverse)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):
        x.copy_(torch.randn((T, H), generator=gen, device="cuda"))
        inds.copy_(routing(gen, T, k, E, True))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    import mlx_rs_amd as m
    from mlx_rs_amd import ops
    x, inds = torch.zeros(3, 8, device="cuda"), torch.zeros(3, 2, device="cuda", dtype=torch.int32)
    w, rows, inverse = torch.zeros(3, 2, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(3, 2, device="cuda", dtype=torch.int32)
    for needle, call in [("inds", lambda: ops.sort_tokens(x, inds[:2], 4)), ("expected dtype", lambda: ops.sort_tokens(x, inds.long(), 4)),
                         ("n_experts", lambda: ops.sort_tokens(x, inds, 0)), ("n_experts", lambda: ops.sort_tokens(x, inds, 513)),
                         ("out of range", lambda: ops.sort_tokens(x, inds, 2 ** 40)), ("contiguous", lambda: ops.sort_tokens(x.t(), inds, 4)),
                         ("top_k", lambda: ops.sort_tokens(x, torch.zeros(3, 33, device="cuda", dtype=torch.int32), 4)), ("bfloat16", lambda: ops.sort_tokens(x.double(), inds, 4)),
                         ("6 rows", lambda: ops.sort_tokens_grad(rows[:5], inverse)), ("6 rows", lambda: ops.unsort_tokens(rows[:5], w, inverse)),
                         ("weights", lambda: ops.unsort_tokens(rows, w[:2], inverse)), ("inverse", lambda: ops.unsort_tokens(rows, w, inverse.reshape(-1))),
                         ("dout", lambda: ops.unsort_tokens_grad(x[:2], rows, w, inverse)), ("expected dtype", lambda: ops.unsort_tokens_grad(x.half(), rows, w, inverse)),
                         ("device", lambda: ops.unsort_tokens(rows, w.cpu(), inverse))]:
        with pytest.raises(m.MoeError, match=needle):
            call()

"""Experts from logits (softmax and sigmoid scores, a bias, groups), and the gradient of their weights, against float64 on the host."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NONE, OUT = -math.inf, -math.inf


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def scores_of(row, scoring):
    """float64 scores of a row of logits; what is no number has no part in the others'."""
    if scoring == "sigmoid":
        return [math.nan if x != x else 0.0 if x < -745 else 1.0 / (1.0 + math.exp(-x)) for x in row]
    seen = [x for x in row if x == x]
    most = max(seen, default=-math.inf)
    if most == -math.inf:
        return [math.nan if x != x else 0.0 for x in row]
    e = [math.nan if x != x else math.exp(x - most) for x in row]
    total = math.fsum(x for x in e if x == x)
    return [x / total for x in e]


def choose(row, k, scoring, bias, groups, top_groups, group_score):
    """The definition, in the order of words: ids, best first, and the scores."""
    s = scores_of(row, scoring)
    E, size = len(row), len(row) // groups
    with_bias = [x if bias is None else x + bias[i] for i, x in enumerate(s)]
    with_bias = [-math.inf if row[i] == -math.inf else x for i, x in enumerate(with_bias)]
    key = [x if x == x else None for x in (row if bias is None else with_bias)]  # None: behind everything
    open_ = set(range(groups))
    if groups > 1:
        rank = []
        for g in range(groups):
            its = range(g * size, (g + 1) * size)
            of = [key[i] for i in its] if group_score == "max" else [with_bias[i] for i in its]
            best = sorted((-math.inf if x is None or x != x else x for x in of), reverse=True)
            rank.append(best[0] if group_score == "max" or size == 1 else best[0] + best[1])
        open_ = set(sorted(range(groups), key=lambda g: (-rank[g], g))[:top_groups])
    able = [i for i in range(E) if i // size in open_]
    ids = sorted(able, key=lambda i: (key[i] is None, 0.0 if key[i] is None else -key[i], i))[:k]
    return ids, s


def check(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0, dtype=torch.float32):
    import mlx_rs_amd as m
    inds, w = m.ops.select_experts(logits, k, scoring, bias, groups, top_groups, group_score, renormalize, scale, dtype)
    assert inds.shape == logits.shape[:-1] + (k,) and w.shape == inds.shape and w.dtype == dtype and inds.dtype == torch.int32
    rows = logits.double().cpu().reshape(-1, logits.shape[-1]).tolist()
    b = None if bias is None else bias.double().cpu().tolist()
    for t, row in enumerate(rows):
        ids, s = choose(row, k, scoring, b, groups, top_groups, group_score)
        assert inds.reshape(-1, k)[t].tolist() == ids, (t, ids)
        if renormalize and scoring == "softmax":  # (shares of the chosen, which are there also where a softmax over all rounds to zero, as of logits 1e38 below the largest)
            s = dict(zip(ids, scores_of([row[i] for i in ids], scoring)))
        total = math.fsum(s[i] for i in ids) if renormalize else 1.0
        for j, i in enumerate(ids):
            ref = (0.0 if total == 0 else s[i] / total) * scale
            got = float(w.reshape(-1, k)[t, j])
            # float64 up to one rounding to float32 and one to the type
            assert (got != got) if ref != ref else abs(got - ref) <= (half_step(dtype) + 2.0 ** -24) * abs(ref) + 2.0 ** -126 * 2.0 ** -6, (t, j, got, ref)
    return inds, w


# experts and groups: one expert, fewer than lanes, one short of and one past a lane's run, a group a lane, groups that leave lanes idle (3, 5, 33), all 512
SHAPES = [(1, 1), (8, 1), (63, 1), (64, 1), (65, 1), (128, 1), (200, 1), (512, 1), (16, 4), (64, 8), (256, 8), (160, 8), (64, 64), (33, 33), (495, 33), (9, 3), (300, 5), (512, 2), (102, 17), (126, 9)]


@pytest.mark.parametrize("E,groups", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_selection(dtype, scoring, E, groups):
    """All forms of a shape; bfloat16 logits have many equal ones."""
    gen = torch.Generator().manual_seed(E * 64 + groups)
    logits = (torch.randn(21, E, generator=gen) * 1.5).to(dtype).cuda()
    bias = (torch.randn(E, generator=gen) * 0.05).cuda()
    size = E // groups
    for i, top_groups in enumerate({1, (groups + 1) // 2, groups}):
        k = min(32, 8 if i else 32, size * top_groups)
        for b in (None, bias):
            for group_score in ("max", "top2"):
                check(logits, k, scoring, b, groups, top_groups, group_score, i % 2 == 0, 2.5 if i else 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [0, 1, 2, 3, 4, 5, 1000])
def test_numbers_of_tokens_and_types_of_weights(T, dtype):
    logits = torch.randn(T, 72, generator=torch.Generator().manual_seed(T)).cuda()
    check(logits, 6, "sigmoid", torch.linspace(-0.1, 0.1, 72).cuda(), 8, 3, "top2", True, 1.5, dtype)
    check(logits, 6, "softmax", None, renormalize=False, dtype=dtype)
    check(logits.reshape(1, T, 72), 1, "softmax", dtype=dtype)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_masked_and_missing_logits(scoring, biased):
    """-inf, the lowest value, infinities below zero in whole groups and whole rows, and what is no number."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(8, 32, generator=gen)
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2] = torch.finfo(torch.float32).min
    logits[2, 7] = 1.0
    logits[3, ::2] = -math.inf
    logits[4, 5] = math.nan
    logits[5] = math.nan
    logits[6, :31] = math.nan
    logits[7, :16] = -math.inf
    bias = (torch.randn(32, generator=gen) * 0.5 - 2.0).cuda() if biased else None  # (below zero: an expert that is out does not come in by its bias)
    for groups, top in ((1, 1), (4, 2), (32, 8)):
        for group_score in ("max", "top2"):
            for renormalize in (True, False):
                check(logits.cuda(), 5, scoring, bias, groups, top, group_score, renormalize)


def test_ties_go_to_the_lower_id():
    import mlx_rs_amd as m
    logits = torch.zeros(3, 256, device="cuda")
    logits[1, 100:] = -0.0
    logits[2, 37] = 1.0
    for bias in (None, torch.zeros(256, device="cuda")):
        inds, w = m.ops.select_experts(logits, 8, "sigmoid", bias, 8, 2, "top2")
        assert inds[0].tolist() == list(range(8)) and inds[1].tolist() == list(range(8)) and inds[2].tolist() == [37, 0, 1, 2, 3, 4, 5, 6]
        assert bool((w[0] == 0.125).all())


def test_keys_that_differ_by_less_than_a_float():
    """Scores and bias are compared in float64: 1e-12 apart is apart, in either order."""
    import mlx_rs_amd as m
    logits = torch.zeros(1, 64, device="cuda")
    bias = torch.full((64,), -0.5, device="cuda")  # every key is 0
    logits[0, 40] = 4e-12  # 1e-12 more
    logits[0, 9] = -4e-12
    inds, _ = m.ops.select_experts(logits, 64 // 2, "sigmoid", bias)
    assert inds[0, 0] == 40 and 9 not in inds[0].tolist()[:31]
    # as close as one expert in a thousand draws comes: the rest of the order goes by ids
    assert inds[0, 1:].tolist() == [i for i in range(34) if i not in (9, 40)][:31]


def check_many(rows, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """4099 tokens that repeat `rows`: each repetition in other lanes and beside other tokens, and all with the same result, which the first ones are checked for."""
    import mlx_rs_amd as m
    at = torch.arange(4099, device="cuda") % rows.shape[0]
    args = (k, scoring, bias, groups, top_groups, group_score, renormalize, scale, torch.float32)
    inds, w = m.ops.select_experts(rows[at], *args)
    small_inds, small_w = check(rows, *args)
    assert bool((inds == small_inds[at]).all())
    assert torch.equal(w.view(torch.int32), w[:rows.shape[0]][at].view(torch.int32))
    # both are within one rounding of the same number
    assert torch.allclose(w, small_w[at], rtol=2.0 ** -22, atol=2.0 ** -148, equal_nan=True)


# a row of lanes a token: 4, 8, 16 and 32 experts a lane, uneven ones, groups that leave lanes of the row idle, and what only a wave holds (more groups, more chosen)
MANY = [(1, 1, 1), (8, 1, 8), (17, 1, 16), (64, 1, 15), (65, 1, 14), (100, 1, 16), (128, 1, 8), (200, 1, 8), (256, 1, 16), (257, 1, 5), (500, 1, 16), (512, 1, 10),
        (16, 4, 2), (256, 8, 8), (160, 8, 6), (9, 3, 3), (300, 5, 16), (512, 2, 8), (126, 9, 4), (16, 16, 2), (512, 16, 16), (64, 64, 8), (64, 1, 17), (102, 17, 6)]


@pytest.mark.parametrize("E,groups,k", MANY)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tokens(dtype, scoring, E, groups, k):
    gen = torch.Generator().manual_seed(E * 64 + groups + k)
    rows = (torch.randn(21, E, generator=gen) * 1.5).to(dtype).cuda()
    bias = (torch.randn(E, generator=gen) * 0.05).cuda()
    top = groups if groups == 1 else max(groups // 2, -(-k // (E // groups)))
    for b in (None, bias, torch.zeros_like(bias)):
        for group_score in ("max", "top2") if groups > 1 else ("max",):
            for renormalize in (True, False):
                check_many(rows, k, scoring, b, groups, top, group_score, renormalize, 2.5)


test_every_layout_of_many_tokens = test_many_tokens  # (collected by this name: a test further down has the other)


@pytest.mark.parametrize("E,groups,k", MANY)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_every_layout_of_many_float16_tokens(scoring, E, groups, k):
    test_every_layout_of_many_tokens(torch.float16, scoring, E, groups, k)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [1, 2, 7, 8, 14, 15, 16])
def test_many_tokens_with_keys_close_together(k, scoring):
    """Biases that are minus the score but for steps of 1e-9 to 1e-5: the order, the last that is in and the first that is out are all nearer than floats tell, in some rows."""
    gen = torch.Generator().manual_seed(k)
    one = torch.randn(1, 96, generator=gen)
    s = torch.tensor(scores_of(one[0].tolist(), scoring), dtype=torch.float64)
    for step in (1e-9, 1e-7, 1e-6, 1e-5):
        bias = (-s + step * torch.randperm(96, generator=gen).double()).float()
        rows = (one + step * torch.randn(16, 96, generator=gen)).cuda()
        check_many(rows, k, scoring, bias.cuda())
        check_many(rows, min(k, 12), scoring, bias.cuda(), 8, 4, "top2", False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_many_tokens_masked(scoring, biased):
    gen = torch.Generator().manual_seed(5)
    rows = torch.randn(9, 32, generator=gen)
    rows[0] = -math.inf
    rows[1, 3:] = -math.inf
    rows[2] = torch.finfo(torch.float32).min
    rows[2, 7] = 1.0
    rows[3, ::2] = -math.inf
    rows[4, 5] = math.nan
    rows[5] = math.nan
    rows[6, :31] = math.nan
    rows[7, :16] = -math.inf
    bias = (torch.randn(32, generator=gen) * 0.5 - 2.0).cuda() if biased else None
    for groups, top in ((1, 1), (4, 2), (16, 4)):
        for group_score in ("max", "top2"):
            for renormalize in (True, False):
                check_many(rows.cuda(), 5, scoring, bias, groups, top, group_score, renormalize)


def gradient(logits, inds, dw, scoring, renormalize, scale):
    """torch's derivative of the definition, float64 on the host."""
    x = logits.double().cpu().requires_grad_()
    s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, -1)
    w = s.gather(-1, inds.cpu().long())
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    (w * scale * dw.double().cpu()).sum().backward()
    return x.grad


@pytest.mark.parametrize("E,k,T", [(1, 1, 3), (8, 2, 1), (64, 8, 5), (65, 7, 2), (200, 32, 9), (512, 8, 33), (128, 1, 0)])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(dtype, scoring, renormalize, E, k, T):
    import mlx_rs_amd as m
    gen = torch.Generator().manual_seed(E * k + T)
    logits = (torch.randn(T, E, generator=gen) * 1.5).to(dtype).cuda()
    inds, _ = m.ops.select_experts(logits, k, scoring, renormalize=renormalize)
    for wt in DTYPES:
        dw = torch.randn(T, k, generator=gen).to(wt).cuda()
        got = m.ops.select_experts_grad(dw, logits, inds, scoring, renormalize, 2.5)
        assert got.dtype == dtype and got.shape == logits.shape
        ref = gradient(logits, inds, dw, scoring, renormalize, 2.5)
        # float64, then one rounding to float32 and one to the type; what cancels (the weighted mean of dw) does in float64, and torch's own derivative does too: 1e-14 of the terms
        bound = (half_step(dtype) + 2.0 ** -24) * ref.abs() + 1e-13 * 2.5 * float(dw.abs().max() if T else 0) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
        assert bool(((got.double().cpu() - ref).abs() <= bound).all())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(scoring, renormalize):
    """Along a direction, differences of the forward definition in float64 with the choice held: their error is of the order 1e-8."""
    import mlx_rs_amd as m
    gen = torch.Generator().manual_seed(9)
    logits, d, dw = torch.randn(4, 24, generator=gen), torch.randn(4, 24, generator=gen), torch.randn(4, 5, generator=gen)
    inds, _ = m.ops.select_experts(logits.cuda(), 5, scoring)
    got = m.ops.select_experts_grad(dw.cuda(), logits.cuda(), inds, scoring, renormalize, 1.5).double().cpu()
    at = inds.cpu().long()

    def value(x):
        s = (torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, -1)).gather(1, at)
        return float((1.5 * dw.double() * (s / s.sum(1, keepdim=True) if renormalize else s)).sum())

    x, t = logits.double(), 1e-4
    along = (value(x + t * d.double()) - value(x - t * d.double())) / (2 * t)
    assert abs(float((got * d.double()).sum()) - along) <= 1e-6 * float((got * d.double()).abs().sum())


@pytest.mark.parametrize("E,k", [(1, 1), (3, 2), (17, 16), (40, 17), (65, 9), (512, 16), (511, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_any_ids(dtype, E, k):
    """Ids that no selection would give: repeated any number of times, outside, in every slot; 1 to 9 tokens, nothing written behind the last."""
    import mlx_rs_amd as m
    gen = torch.Generator().manual_seed(E + k)
    for T in (1, 2, 3, 4, 5, 9):
        logits = torch.randn(T, E, generator=gen).to(dtype).cuda()
        inds = torch.randint(-1, min(E, 6) + 1, (T, k), generator=gen).to(torch.int32).cuda()  # (-1 and, of few experts, E: outside)
        dw = torch.randn(T, k, generator=gen).cuda()
        inside = (inds >= 0) & (inds < E)
        for scoring in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                room = torch.full((T * E + 64,), 7.0, dtype=dtype, device="cuda")
                m.capi.check(m.load_library().mi_moe_select_experts_grad(dw.data_ptr(), 2, logits.data_ptr(), m.ops._DTYPES[dtype], inds.data_ptr(), T, E, k, int(scoring == "sigmoid"),
                                                                         int(renormalize), 1.5, room.data_ptr(), m.ops._stream()))
                assert bool((room[T * E:] == 7).all())
                x = logits.double().cpu().requires_grad_()
                s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, -1)
                w = s.gather(1, inds.cpu().long().clamp(0, E - 1)) * inside.cpu()
                if renormalize:
                    total = w.sum(-1, keepdim=True)
                    w = w / torch.where(total == 0, torch.ones_like(total), total)
                (w * 1.5 * dw.double().cpu()).sum().backward()
                # (as in test_gradient, the terms that meet in one id up to 32)
                bound = (half_step(dtype) + 2.0 ** -24) * x.grad.abs() + 1e-12 * float(dw.abs().max()) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
                assert bool(((room[:T * E].reshape(T, E).double().cpu() - x.grad).abs() <= bound).all())


def test_gradient_of_repeated_and_foreign_ids_and_masked_rows():
    import mlx_rs_amd as m
    logits = torch.randn(4, 16, generator=torch.Generator().manual_seed(2)).cuda()
    logits[2] = -math.inf
    logits[3, 4:] = -math.inf
    dw = torch.randn(4, 3, generator=torch.Generator().manual_seed(3)).cuda()
    inds = torch.tensor([[1, 1, 5], [3, -1, 16], [0, 1, 2], [0, 9, 1]], dtype=torch.int32, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        got = m.ops.select_experts_grad(dw, logits, inds, scoring, True).double().cpu()
        assert torch.allclose(got[0], gradient(logits[:1], inds[:1], dw[:1], scoring, True, 1.0)[0], rtol=2.0 ** -23, atol=1e-12)
        alone = m.ops.select_experts_grad(dw[1:2, :1].contiguous(), logits[1:2].contiguous(), inds[1:2, :1].contiguous(), scoring, True).double().cpu()
        assert torch.equal(got[1], alone[0])
        assert not got[2].any()  # nothing chosen has a score
        assert torch.isfinite(got[3]).all() and float(got[3, 9]) == 0.0
        whole = m.ops.select_experts_grad(dw, logits, inds, scoring, False)
        assert torch.isfinite(whole).all() and not whole[2].any()


def test_many_tokens():
    """A prompt's selection in one call is that of its parts."""
    import mlx_rs_amd as m
    logits = torch.randn(70000, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    bias = torch.randn(128, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 0.05
    inds, w = m.ops.select_experts(logits, 8, "sigmoid", bias, 4, 2, "top2", dtype=torch.float32)
    for a in (0, 33333, 69990):
        i2, w2 = m.ops.select_experts(logits[a:a + 10].contiguous(), 8, "sigmoid", bias, 4, 2, "top2", dtype=torch.float32)
        assert torch.equal(inds[a:a + 10], i2) and torch.equal(w[a:a + 10], w2)


def test_refusals():
    import mlx_rs_amd as m
    x = torch.zeros(4, 16, device="cuda")
    i = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for call in (lambda: m.ops.select_experts(x, 2, "other"), lambda: m.ops.select_experts(x, 2, group_score="other"), lambda: m.ops.select_experts(x, 0),
                 lambda: m.ops.select_experts(x, 17), lambda: m.ops.select_experts(x, 2, bias=x[0, :8]), lambda: m.ops.select_experts(x, 2, bias=x[0].half()),
                 lambda: m.ops.select_experts(x.t(), 2), lambda: m.ops.select_experts(x, 2, dtype=torch.float64), lambda: m.ops.select_experts(x, 9, n_groups=4, top_groups=2),
                 lambda: m.ops.select_experts_grad(x, x, i), lambda: m.ops.select_experts_grad(x[:, :2].contiguous(), x, i.long()),
                 lambda: m.ops.select_experts_grad(x[:3, :2].contiguous(), x, i[:3].contiguous())):
        with pytest.raises(m.MoeError):
            call()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [5, 4100])
def test_masked_experts_and_groups_of_a_router(scoring, T):
    """Experts that every token has masked, by a logit or by a bias of -inf, among others that are close together."""
    import mlx_rs_amd as m
    gen = torch.Generator().manual_seed(T)
    rows = torch.randn(5, 48, generator=gen)
    rows[:, 40:] = -math.inf
    bias = torch.randn(48, generator=gen) * 1e-6
    bias[[3, 17]] = -math.inf
    bias[24:30] = -math.inf  # all of a group of six
    at = torch.arange(T) % 5
    for groups, top, group_score in ((1, 1, "max"), (8, 3, "top2"), (8, 5, "max"), (48, 40, "top2")):
        for k in (4, 9):
            for b in (None, bias.cuda()):
                inds, w = m.ops.select_experts(rows[at].cuda(), k, scoring, b, groups, top, group_score, dtype=torch.float32)
                small, small_w = check(rows.cuda(), k, scoring, b, groups, top, group_score)
                assert bool((inds == small[at.cuda()]).all()) and torch.allclose(w, small_w[at.cuda()], rtol=2.0 ** -22, atol=0)


def test_weights_of_scores_that_a_softmax_rounds_to_zero():
    """The expert with all of the softmax is not open: the shares are those of the chosen logits among themselves, whether floats or doubles decide the choice."""
    logits = torch.full((2, 32), -1000.0)
    logits[:, 0] = 1000.0
    logits[:, 9] = -999.0
    bias = torch.zeros(32)
    bias[0] = -5.0
    spread = bias + torch.arange(32) * 1e-3
    for b in (bias, spread):
        check(logits.cuda(), 4, "softmax", b.cuda(), 4, 2, "max")
        check_many(logits.cuda(), 4, "softmax", b.cuda(), 4, 2, "max")


def test_more_tokens_than_a_launch_takes():
    """2^25 and three tokens of 128 experts: results and gradients on both sides of where a launch ends, logits past 2^32 elements."""
    import mlx_rs_amd as m
    T, E, k = 2 ** 25 + 3, 128, 2
    base = torch.randn(4093, E, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    logits = torch.empty((T, E), dtype=torch.bfloat16, device="cuda")
    for i in range(0, T, 4093 * 512):
        part = logits[i:i + 4093 * 512]
        part.copy_(base.repeat(512, 1)[:part.shape[0]])
    inds, w = m.ops.select_experts(logits, k)
    want_i, want_w = m.ops.select_experts(base, k)
    dw = torch.randn(T, k, device="cuda").to(torch.bfloat16)
    d = m.ops.select_experts_grad(dw, logits, inds)
    for at in (0, 2 ** 25 - 4093, 2 ** 25 - 2, T - 4093):
        r = torch.arange(at, min(at + 4093, T), device="cuda") % 4093
        part = slice(at, at + r.numel())
        assert torch.equal(inds[part], want_i[r]) and torch.equal(w[part], want_w[r])
        assert torch.equal(d[part], m.ops.select_experts_grad(dw[part].contiguous(), logits[part].contiguous(), inds[part].contiguous()))

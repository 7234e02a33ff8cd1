"""Groups of experts of which some are masked: what such a group is worth, against the definition in float64 on the host and against torch's own operations."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_select as base  # noqa: E402


def choose(row, k, scoring, bias, groups, top_groups, group_score):
    """base.choose with the rank by two as the header words it: s + bias, where an expert whose logit is -inf or no number has a score of zero and one whose bias is adds nothing; a
    group without a logit and a bias above -inf comes last."""
    s = base.scores_of(row, scoring)
    E, size = len(row), len(row) // groups
    b = [0.0] * E if bias is None else bias
    able = [row[i] > -math.inf and b[i] > -math.inf for i in range(E)]
    biased = [-math.inf if row[i] == -math.inf else s[i] + b[i] for i in range(E)]
    key = [x if x == x else None for x in (row if bias is None else biased)]
    open_ = set(range(groups))
    if groups > 1:
        rank = []
        for g in range(groups):
            its = range(g * size, (g + 1) * size)
            two = group_score == "top2" and size > 1
            of = [s[i] + b[i] if row[i] > -math.inf else b[i] for i in its] if two else [key[i] for i in its]
            best = sorted((x for x in of if x is not None and x > -math.inf), reverse=True)
            rank.append(sum(best[:2 if two else 1]) if any(able[i] for i in its) and best else -math.inf)
        open_ = set(sorted(range(groups), key=lambda g: (-rank[g], g))[:top_groups])
    ids = sorted((i for i in range(E) if i // size in open_), key=lambda i: (key[i] is None, 0.0 if key[i] is None else -key[i], i))[:k]
    return ids, s


@pytest.fixture(autouse=True)
def definition(monkeypatch):
    monkeypatch.setattr(base, "choose", choose)


# groups of two, more, an odd number, and (the last two) more groups than a row of lanes has a token's
SHAPES = [(8, 4), (32, 16), (64, 8), (60, 5), (256, 8), (27, 9), (66, 33), (128, 64)]


def masked_rows(E, groups, gen):
    """Rows whose groups have none, one, two and all of their experts."""
    size = E // groups
    rows = torch.randn(17, E, generator=gen) * 2
    for t in range(17):
        for g in range(groups):
            left = (0, 1, 2, size, 1)[int(torch.randint(5, (1,), generator=gen))]
            gone = torch.randperm(size, generator=gen)[left:]
            rows[t, g * size + gone] = -math.inf
    rows[1] = -math.inf
    rows[1, E - 2] = 3.0  # one expert of all
    rows[2, rows[2] == -math.inf] = math.nan  # what is missing is no number
    rows[3] = torch.where((rows[3] == -math.inf) & (torch.rand(E, generator=gen) < 0.5), torch.tensor(math.nan), rows[3])
    return rows


@pytest.mark.parametrize("E,groups", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biases", ["none", "small", "below zero", "masks too"])
@pytest.mark.parametrize("run", [base.check, base.check_many], ids=["few", "many"])
def test_groups_with_masked_experts(run, biases, scoring, E, groups):
    gen = torch.Generator().manual_seed(E + groups)
    rows = masked_rows(E, groups, gen)
    bias = None if biases == "none" else torch.randn(E, generator=gen) * 0.1 - (2.0 if biases == "below zero" else 0.0)
    if biases == "masks too":
        bias[torch.randperm(E, generator=gen)[:E // 3]] = -math.inf
        bias[torch.randperm(E, generator=gen)[:2]] = math.nan
    for top in sorted({1, max(1, groups // 4), groups // 2}):
        for k in sorted({1, min(8, top * (E // groups))}):
            for renormalize in (True, False):
                run(rows.cuda(), k, scoring, None if bias is None else bias.cuda(), groups, top, "top2", renormalize)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [17, 4099])
def test_without_a_bias_a_masked_expert_is_a_score_of_zero(T, scoring):
    """By sums, sorts and comparisons of whole tensors, with at least one expert left in as many groups as are open."""
    import mlx_rs_amd as m
    for E, groups, top, k in ((8, 4, 1, 1), (8, 4, 2, 2), (64, 8, 3, 5), (32, 16, 4, 4)):
        gen = torch.Generator().manual_seed(E + top)
        logits = torch.randn(T, E, generator=gen).cuda() * 2
        size, at = E // groups, torch.arange(E, device="cuda")
        keep = torch.randint(size, (T, groups), generator=gen).cuda().repeat_interleave(size, 1) == at % size  # one of each group
        whole = (torch.rand(T, groups, generator=gen) < 0.3).cuda().repeat_interleave(size, 1)
        logits = logits.masked_fill(~(keep | whole), -math.inf)
        s = torch.sigmoid(logits.double()) if scoring == "sigmoid" else torch.softmax(logits.double(), -1)
        rank = s.reshape(T, groups, size).sort(-1, descending=True)[0][..., :2].sum(-1)
        order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, :top]
        open_ = torch.zeros_like(rank, dtype=torch.bool).scatter(1, order, True).repeat_interleave(size, 1)
        want = torch.sort(torch.where(open_, logits.double(), -math.inf), dim=-1, descending=True, stable=True)[1][:, :k]
        left = (open_ & (logits > -math.inf)).sum(-1) >= k
        inds, _ = m.ops.select_experts(logits, k, scoring, None, groups, top, "top2")
        assert int(left.sum()) > T // 2 and torch.equal(inds[left].long(), want[left])


def test_the_only_expert_that_is_left():
    import mlx_rs_amd as m
    logits = torch.full((3, 8), -math.inf, device="cuda")
    logits[0, 2] = 3.0
    logits[1] = torch.tensor([-4.0, -4.0, 10.0, -math.inf, -5.0, -5.0, -6.0, -6.0])
    logits[2, 7] = -30.0
    for rows in (logits, logits.repeat(1400, 1)):
        inds, w = m.ops.select_experts(rows, 1, "sigmoid", None, 4, 1, "top2", False, dtype=torch.float32)
        assert inds[:3, 0].tolist() == [2, 2, 7] and bool((inds == inds[:3].repeat(rows.shape[0] // 3, 1)).all())
        inds, _ = m.ops.select_experts(rows, 2, "sigmoid", None, 4, 2, "top2")
        assert inds[1].tolist() == [2, 0]
        # biases of masked experts, however large, do not bring in a group of masked ones alone
        high = torch.tensor([5.0, 5.0, 0, 0, 5.0, 5.0, 5.0, 0], device="cuda")
        assert m.ops.select_experts(rows, 1, "sigmoid", high, 4, 1, "top2")[0][:3, 0].tolist()[::2] == [2, 7]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_masked_and_missing_logits(scoring, biased):
    """The inputs of the tests of these names in test_gpu_select.py, whose own definition ranks a group with one expert left as one with none."""
    base.test_masked_and_missing_logits(scoring, biased)
    base.test_many_tokens_masked(scoring, biased)

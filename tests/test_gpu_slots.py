"""Slots of a caller's routing that name no expert contribute nothing to the block's result, whatever stands in for them holds."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_layer import CONFIGS, block  # noqa: E402

TOKENS = [1, 3, 7, 40, 65, 300, 1500]


def routing(cfg, T, foreign, seed=0, first=0):
    """k different experts a token, of those from `first` on; slots of `foreign` [T, k] name none."""
    gen = torch.Generator().manual_seed(seed + T)
    inds = torch.stack([first + torch.randperm(cfg.n_experts - first, generator=gen)[:cfg.top_k] for _ in range(T)]).int()
    w = (torch.randint(1, 8, (T, cfg.top_k), generator=gen) / 16).bfloat16()
    outside = torch.tensor([-1, cfg.n_experts, 2 ** 31 - 1], dtype=torch.int32)[torch.randint(3, (T, cfg.top_k), generator=gen)]
    return torch.where(foreign, outside, inds).cuda(), w.cuda()


def filled(T, k, every):
    foreign = torch.zeros(T, k, dtype=torch.bool)
    foreign[::every] = True
    return foreign


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3e38])
def test_rows_of_a_padded_batch(value, T, config):
    """Padded tokens hold anything: their results are zeros, and the others' have the bits that they have beside rows of ones."""
    from mlx_rs_amd import synth
    blk, cfg = block(*config)
    foreign = filled(T, cfg.top_k, 3)
    pad = foreign[:, 0].cuda()
    inds, w = routing(cfg, T, foreign)
    x = synth.make_tokens(cfg, T, seed=1, device="cuda")
    x[pad] = 1.0
    want = blk.forward_routed(x, inds, w).clone()
    x[pad] = value
    got = blk.forward_routed(x, inds, w)
    assert not got[pad].any() and torch.isfinite(got).all()
    assert torch.equal(got, want)


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("T", TOKENS)
def test_experts_that_stand_in(T, config):
    """The experts with the lowest numbers, which stand in for slots that name none or one twice, give no numbers: nobody names them, and every result is one."""
    from mlx_rs_amd import synth
    blk, cfg = block(*config)
    first = cfg.n_experts - cfg.top_k
    gen = torch.Generator().manual_seed(T)
    foreign = torch.rand(T, cfg.top_k, generator=gen) < 0.4
    inds, w = routing(cfg, T, foreign, first=first)
    if cfg.top_k > 1:
        inds[::2, 1] = inds[::2, 0]  # twice
    w[0, 0] = -0.0 if T > 1 else w[0, 0]  # (a weight like any other)
    x = synth.make_tokens(cfg, T, seed=1, device="cuda")
    want, dbg = blk.forward_routed(x, inds, w, debug=True)
    want = want.clone()
    named = (dbg["topk_idx"] >= first) & (dbg["topk_w"] != 0)
    assert bool((dbg["topk_w"][~named] == 0).all())
    for bank in (blk.down_proj, blk.up_proj):
        kept = bank.scales.clone()
        bank.scales[:first] = float("nan")
        got = blk.forward_routed(x, inds, w)
        bank.scales.copy_(kept)
        # (a stand-in with a high number is one that some token names: its results are numbers)
        assert torch.isfinite(got).all()
        assert torch.equal(got, want)


def test_a_weight_of_zero_is_no_empty_slot():
    """Zero times a result that is none is none, for either zero."""
    from mlx_rs_amd import synth
    blk, cfg = block(256, 8, 2, 512)
    x = synth.make_tokens(cfg, 4, seed=1, device="cuda")
    x[2:] = float("nan")
    inds = torch.tensor([[0, 1], [2, 3], [0, 1], [4, 5]], dtype=torch.int32, device="cuda")
    for zero in (0.0, -0.0):
        out = blk.forward_routed(x, inds, torch.full((4, 2), zero, dtype=torch.bfloat16, device="cuda"))
        assert not out[:2].any() and torch.isnan(out[2:]).all()


def test_more_tokens_than_a_launch_takes_are_refused():
    """From 2^26 - 3 tokens on the launches of a wave a token would have 2^32 threads; nothing is launched, and nothing is read."""
    import mlx_rs_amd as m
    blk, _ = block(128, 2, 1, 128)
    x = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(4096, dtype=torch.int32, device="cuda")
    lib, p = m.load_library(), x.data_ptr()
    for T in (2 ** 26 - 3, 2 ** 26, 2 ** 30):
        for call in (lambda: lib.mi_moe_forward_routed(blk._handle, p, ids.data_ptr(), p, T, p, p, 4096, None, m.ops._stream()),
                     lambda: lib.mi_moe_forward(blk._handle, p, T, p, p, 4096, None, m.ops._stream())):
            assert call() != 0 and f"{T} tokens" in m.capi.last_error(), m.capi.last_error()
    assert lib.mi_moe_forward(blk._handle, p, 2 ** 26 - 4, p, p, 4096, None, m.ops._stream()) != 0 and "workspace too small" in m.capi.last_error()
    torch.cuda.synchronize()
    assert not x.any()

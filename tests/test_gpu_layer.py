"""The operators around the experts as a decoder layer uses them: the block on a given routing, and a run of norm, selection, experts and projections, eager and captured."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def block(hidden, experts, k, inter, bits=4, group=64, seed=3):
    import mlx_rs_amd as m
    from mlx_rs_amd import synth
    cfg = m.MoeConfig(hidden, experts, k, inter, bits, group, 0)
    return synth.make_block(cfg, seed=seed, device="cuda", gen_device="cuda"), cfg


CONFIGS = [(256, 8, 2, 512, 4, 64), (256, 128, 8, 256, 4, 64), (512, 64, 6, 384, 8, 64), (256, 16, 4, 256, 4, 32), (256, 16, 4, 256, 8, 128), (192, 9, 3, 64, 8, 64), (128, 16, 4, 128, 2, 64)]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("T", [1, 5, 40, 65, 300, 1500])
def test_the_block_s_own_routing_gives_its_own_bits(T, config):
    from mlx_rs_amd import synth
    blk, cfg = block(*config)
    x = synth.make_tokens(cfg, T, seed=1, device="cuda")
    out, dbg = blk.forward(x, debug=True)
    routed, again = blk.forward_routed(x, dbg["topk_idx"], dbg["topk_w"], debug=True)
    assert torch.equal(routed, out)
    for name in dbg:
        assert torch.equal(again[name], dbg[name]), name


@pytest.mark.parametrize("T", [3, 100, 700])
def test_repeated_and_foreign_ids(T):
    """An expert named twice is one with the sum of the weights; an id outside the experts is a slot of no weight."""
    from mlx_rs_amd import synth
    from test_gpu_codes import block_truth
    blk, cfg = block(256, 16, 4, 256)
    x = synth.make_tokens(cfg, T, seed=2, device="cuda")
    gen = torch.Generator().manual_seed(T)
    inds = torch.stack([torch.randperm(16, generator=gen)[:4] for _ in range(T)]).int()
    w = (torch.randint(1, 8, (T, 4), generator=gen) / 16).bfloat16()
    odd, odd_w = inds.clone(), w.clone()
    plain, plain_w = inds.clone(), w.clone()
    odd[0::3, 2] = odd[0::3, 0]  # twice
    plain_w[0::3, 0] += w[0::3, 2]
    plain_w[0::3, 2] = 0
    odd[1::3, 1], odd[1::3, 3] = -1, 16
    plain_w[1::3, 1], plain_w[1::3, 3] = 0, 0
    odd[2::3] = odd[2::3, :1]  # one expert four times
    plain_w[2::3, 0] = w[2::3].float().sum(1).bfloat16()
    plain_w[2::3, 1:] = 0
    got, dbg = blk.forward_routed(x, odd.cuda(), odd_w.cuda(), debug=True)
    ids = dbg["topk_idx"].sort(1)[0]
    assert bool((ids[:, 1:] != ids[:, :-1]).all()) and bool((ids >= 0).all()) and bool((ids < 16).all())
    # three roundings to bfloat16 (h, y and the result), each at most 2^-8 of its values and typically 0.42 of that, over all; a row on its own three at most.  (Not the bits of the
    # call with the plain routing: which kernel a segment takes goes by its length, and the slots of no weight lengthen other segments.)
    ref = block_truth(blk, x, {"topk_idx": plain.cuda(), "topk_w": plain_w.cuda()})
    assert float((got.double() - ref).norm() / ref.norm()) <= 2.0 ** -8
    assert float(((got.double() - ref).norm(dim=1) / ref.norm(dim=1)).max()) <= 3 * 2.0 ** -8
    nothing = blk.forward_routed(x, torch.full_like(odd, 99).cuda(), odd_w.cuda())
    assert not nothing.any()


def test_routed_refusals():
    import mlx_rs_amd as m
    blk, cfg = block(256, 8, 2, 512)
    x = torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
    i, w = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: blk.forward_routed(x, i.long(), w), lambda: blk.forward_routed(x, i, w.float()), lambda: blk.forward_routed(x, i[:2], w[:2]),
                 lambda: blk.forward_routed(x, i[:, :1].contiguous(), w[:, :1].contiguous()), lambda: blk.forward_routed(x[:, :128].contiguous(), i, w)):
        with pytest.raises(m.MoeError):
            call()
    assert blk.forward_routed(x[:0], i[:0], w[:0]).shape == (0, 256)


class Layer:
    """h = x + r; the expert block on norm(h), routed by sigmoid scores with a bias and groups; then the next sublayer's norm in eight bits and its projection."""

    def __init__(self, hidden=256, experts=32, k=4, bits=4, seed=7):
        import mlx_rs_amd as m
        self.ops = m.ops
        self.blk, self.cfg = block(hidden, experts, k, 256, bits, seed=seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.w1, self.w2 = ((1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).bfloat16() for _ in range(2))
        self.bias = 0.05 * torch.randn(experts, generator=gen, device="cuda")
        self.q, self.s, self.b = m.ops.quantize(0.02 * torch.randn(384, hidden, generator=gen, device="cuda"))

    def __call__(self, x, r):
        y, h = self.ops.add_rms_norm(x, r, self.w1, 1e-6)
        inds, weights = self.ops.select_experts(self.ops.router_logits(y, self.blk.gate_weight), self.cfg.top_k, "sigmoid", self.bias, 8, 4, "top2", True, 2.5)
        moe = self.blk.forward_routed(y, inds, weights)
        rows8, scales, h2 = self.ops.add_rms_norm_rows8(moe, h, self.w2, 1e-6)
        return self.ops.quantized_linear_rows8(rows8, scales, self.q, self.s, self.b), h2, inds, weights, moe


def inputs(T, hidden=256, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(T, hidden, generator=gen).bfloat16().cuda() for _ in range(2))


@pytest.mark.parametrize("T", [1, 6, 64, 130, 600])
def test_a_decoder_layer(T):
    """Each step against float64 from the step before's own results."""
    import test_gpu_rows8 as rows8
    from test_gpu_codes import block_truth
    from test_gpu_norm import truth as norm
    from test_gpu_select import choose
    lay = Layer()
    x, r = inputs(T)
    y, h2, inds, weights, moe = lay(x, r)
    h = (x.float() + r.float()).bfloat16()
    n1 = norm(h, lay.w1, 1e-6).bfloat16()
    mine, _ = lay.ops.add_rms_norm(x, r, lay.w1, 1e-6)
    assert float((mine.double() - n1.double()).abs().max()) <= 2.0 ** -7 * float(n1.abs().max())
    logits = lay.ops.router_logits(mine, lay.blk.gate_weight)
    for t in range(0, T, 37):
        ids, _ = choose(logits[t].double().tolist(), 4, "sigmoid", lay.bias.double().tolist(), 8, 4, "top2")
        assert inds[t].tolist() == ids
    ref = block_truth(lay.blk, mine, {"topk_idx": inds, "topk_w": weights})
    assert float((moe.double() - ref).norm() / ref.norm()) <= 2.0 ** -8
    assert torch.equal(h2, (moe.float() + h.float()).bfloat16())
    q, s, _ = lay.ops.add_rms_norm_rows8(moe, h, lay.w2, 1e-6)
    rows8.check(y, (q, s, lay.q, lay.s, lay.b, None), 64, 4)
    whole = torch.matmul(norm(h2, lay.w2, 1e-6), lay.ops.dequantize(lay.q, lay.s, lay.b, dtype=torch.float32).double().t().contiguous())
    # eight bits: every value of a row half a step of a 127th of its largest off at most, a uniform error of a twelfth root of that
    assert float((y.double() - whole).norm() / whole.norm()) <= 0.02


@pytest.mark.parametrize("T", [1, 40, 200])
def test_captured_and_replayed(T):
    """A captured layer on new inputs, with eager work of the same operators between the replays, and another captured layer of other workspaces beside it."""
    lays = [Layer(seed=7), Layer(seed=8)]
    static = [list(inputs(T, seed=s)) for s in (1, 2)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for lay, (x, r) in zip(lays, static):
            lay(x, r)
    torch.cuda.synchronize()
    for lay, (x, r) in zip(lays, static):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lay(x, r))
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            for to, new in zip(static[i], inputs(T, seed=10 + 2 * turn + i)):
                to.copy_(new)
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        for lay, (x, r), out in zip(lays, static, outs):
            for a, b in zip(out, lay(x, r)):
                assert torch.equal(a, b)


def test_gradients_captured_and_replayed():
    import mlx_rs_amd as m
    T, H, E = 300, 264, 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    h, dy, w = (torch.randn(s, generator=gen, device="cuda") for s in ((T, H), (T, H), (H,)))
    logits, dw = torch.randn(T, E, generator=gen, device="cuda"), torch.randn(T, 4, generator=gen, device="cuda")

    def step():
        inds, _ = m.ops.select_experts(logits, 4, "sigmoid")
        return m.ops.add_rms_norm_grad(dy, h, w, 1e-6, h) + (m.ops.select_experts_grad(dw, logits, inds, "sigmoid"),)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for turn in range(4):
        for t in (h, dy, w, logits, dw):
            t.normal_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    import mlx_rs_amd as m
    lay = Layer()
    xs = [list(inputs(90, seed=s)) for s in (4, 5)]
    want = [[t.clone() for t in lay(*x)] for x in xs]
    lays = [lay, Layer()]  # (forwards through one handle do not overlap)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(lays[i](*xs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            for a, b in zip(run, want[i]):
                assert torch.equal(a, b)

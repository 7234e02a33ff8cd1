"""SwitchGluF8 without a GPU: which tensors its calls are made on."""
import pytest

torch = pytest.importorskip("torch")
import mlx_rs_amd as m  # noqa: E402


def bank(seed):
    return m.F8SwitchLinear(torch.full((2, 16, 16), float(seed)), torch.full((2, 1, 1), float(seed)))


@pytest.fixture
def seen(monkeypatch):
    calls = []
    monkeypatch.setattr(m.ops, "switch_glu_f8", lambda x, inds, weights, *banks: calls.append(banks))
    monkeypatch.setattr(m.ops, "switch_glu_f8_grad", lambda dout, x, inds, weights, *banks: calls.append(banks))

    def of(block):
        calls.clear()
        block.forward(0, 1, 2)
        block(0, 1, 2)
        block.gradient(0, 1, 2, 3)
        assert len(calls) == 3 and all(a is b for c in calls[1:] for p, q in zip(c, calls[0]) for a, b in zip(p, q))
        return calls[0]
    return of


def test_the_calls_take_the_weights_that_the_module_has(seen):
    projections = [bank(i) for i in range(3)]
    block = m.SwitchGluF8(*projections)
    assert all(got[0] is p.weight and got[1] is p.scales for got, p in zip(seen(block), projections))
    block.up_proj = bank(7)  # another bank
    assert seen(block)[1][0] is block.up_proj.weight
    block.gate_proj.weight, block.gate_proj.scales = bank(8).weight, bank(8).scales  # a bank's tensors loaded again
    assert seen(block)[0][0] is block.gate_proj.weight and seen(block)[0][1] is block.gate_proj.scales

"""Which function switch_glu_f8_grad differentiates: the experts without the rounding of silu(gate) * up, on rounded tokens, for a rounded gradient at the result."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402
from test_gpu_f8 import experts_oracle, gen_of  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,E,H,inter", [(1, 2, 4, 144, 272), (40, 2, 4, 256, 128), (200, 3, 4, 272, 400)])
def test_the_weights_gradient_is_the_derivative_in_64_bits(T, k, E, H, inter, dtype):
    from mlx_rs_amd import ops
    gen = gen_of(T)
    banks = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").to(dtype) for _ in range(2))
    inds = torch.rand((T, E), generator=gen, device="cuda").topk(k, -1)[1].to(torch.int32)
    weights = torch.rand((T, k), generator=gen, device="cuda")
    rounded = [c * s.repeat_interleave(128, 1)[:, :H] for c, s in (o.quantize_rows(x), o.quantize_rows(dout))]
    gate, up, down = (c.double() * o.spread(s, *c.shape[1:]) for c, s in banks)
    w = weights.double().requires_grad_()
    loss = 0.0
    for t in range(T):
        for s in range(k):
            e = int(inds[t, s])
            g, u = gate[e] @ rounded[0][t], up[e] @ rounded[0][t]
            loss = loss + w[t, s] * ((down[e] @ (g * torch.sigmoid(g) * u)) * rounded[1][t]).sum()
    loss.backward()
    _, dw = ops.switch_glu_f8_grad(dout, x, inds, weights, *banks)
    _, _, want, off = experts_oracle(x, inds, weights, *banks, dout)
    assert ((want - w.grad).abs() <= off * 1e-6).all()  # (the oracle's own dweights are that derivative)
    o.within(dw, w.grad, off, f"{T} {dtype}")

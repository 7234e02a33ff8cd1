"""The biases' terms of the linear layer on 8-bit rows where they cancel: rows with a large mean, groups whose factors are large and of opposite signs, results that are what is left."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_rows8 as base  # noqa: E402

# few rows, and every kind of tiles; two groups a column, four, more
SHAPES = [(16, 2000, 128, 64), (40, 100, 256, 128), (1300, 4111, 128, 64), (2100, 4000, 256, 128), (300, 9000, 128, 64), (1300, 4111, 128, 32), (1000, 4096, 512, 64), (400, 5001, 128, 64)]


@pytest.mark.parametrize("M,N,K,group", SHAPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", base.DTYPES)
def test_factors_that_cancel(dtype, bits, M, N, K, group):
    gen = torch.Generator(device="cuda").manual_seed(M + N + K + bits)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    G, centre = K // group, 2 ** (bits - 1)
    words = torch.randint(-2 ** 31, 2 ** 31, (N, K * bits // 32), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    scales = ((1 + uniform(N, G)) * 2.0 ** -8 / centre).to(dtype)  # centre * scales are below a step of a float16 bias
    pairs = 8 * (1 + uniform(N, G // 2, 1))
    biases = torch.cat([pairs, -pairs], -1).reshape(N, G).to(dtype)
    x = torch.randint(64, 128, (M, 1), generator=gen, device="cuda").to(torch.int8).expand(M, K).contiguous()
    sx = 2.0 ** -6 * (1 + uniform(M))
    args = (x, sx, words, scales, biases, None)
    y = base.run(args, group, bits)
    ref, size = base.truth(x, sx, words, scales, biases, None, group, bits)
    # Every product is exact: integers below 2^14 in two pieces times a factor of 24 bits in three.  A group's terms are six of them and one multiply-add, an addition each that is off by a
    # step of what is summed so far at most (two half steps; not all matrix instructions round to the nearest); the factor itself, the row's scale and the product with it a half step each.
    # Few rows have a product or two a group in place of six, and eight waves' sums to add.
    terms = 7 * G + 8
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + (2 * terms + 4) * base.U * size + 2.0 ** -24
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())

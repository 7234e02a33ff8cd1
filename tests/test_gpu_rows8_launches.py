"""Linear layers on 8-bit rows of a few dozen columns and more rows than one launch takes."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("workspace", [False, True])
@pytest.mark.parametrize("N,M", [(72, 2 ** 26), (33, 2 ** 27 + 77)])
def test_many_rows_of_few_columns(N, M, workspace):
    """Every row has the result that it has among a few: without a workspace (8 blocks of 32 x 16 and less a launch too many, once), and with one."""
    import mlx_rs_amd as m
    K, lib = 128, m.load_library()
    gen = torch.Generator(device="cuda").manual_seed(N)
    w, s, b = m.ops.quantize(torch.randn(N, K, generator=gen, device="cuda"), 64, 4, torch.bfloat16)
    few = 4096
    x = torch.randint(-127, 128, (few, K), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    sx = torch.rand(few, generator=gen, device="cuda")
    some = slice(0, 64)
    want = m.ops.quantized_linear_rows8(x, sx, w, s, b)
    alone = m.ops.quantized_linear_rows8(x[some].contiguous(), sx[some].contiguous(), w, s, b)
    assert bool(((want[some].float() - alone.float()).abs() <= 2.0 ** -7 * alone.float().abs() + 1e-3).all())
    big, scales = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    for at in range(0, M, few * 1024):
        part = big[at:at + few * 1024]
        part.copy_(x.repeat(1024, 1)[:part.shape[0]])
        scales[at:at + few * 1024] = sx.repeat(1024)[:part.shape[0]]
    need = m.ops._rows8_workspace_bytes(M, K) if workspace else 0
    room = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    m.capi.check(lib.mi_moe_quantized_linear_rows8(big.data_ptr(), scales.data_ptr(), w.data_ptr(), s.data_ptr(), b.data_ptr(), None, M, N, K, 64, 4, 0, y.data_ptr(),
                                                   None if room is None else room.data_ptr(), need, m.ops._stream()))
    at = torch.arange(few * 256, device="cuda") % few
    for first in range(0, M, few * 256):
        part = y[first:first + few * 256].float()
        ref = want[at[:part.shape[0]]].float()
        # two orders of the same float sums, each rounded once to bfloat16
        assert bool(((part - ref).abs() <= 2.0 ** -7 * ref.abs() + 1e-3).all()), first
    del big, scales, y, room
    torch.cuda.empty_cache()

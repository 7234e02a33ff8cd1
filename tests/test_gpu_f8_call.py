"""The calls around the e4m3 operators and the sorted tokens in native code against the general path: the same results, and what they do not take goes the general way."""
import pytest

torch = pytest.importorskip("torch")
import f8_cases as o  # noqa: E402
from test_gpu_layer_call import general, native, same  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def calls(T, dtype):
    """Of every operator: its name, the native call's arguments, and the public call."""
    from mlx_rs_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(T)
    E, k, H, inter = 6, 2, 128, 48
    x, dout = (torch.randn((T, H), generator=gen, device="cuda").to(dtype) for _ in range(2))
    inds = torch.randint(-1, E + 1, (T, k), generator=gen, device="cuda", dtype=torch.int32)
    w = torch.rand((T, k), generator=gen, device="cuda")
    rows, _, inverse, offsets = ops.sort_tokens(x, inds, E)
    gate, up, down = o.bank(gen, inter, H, E), o.bank(gen, inter, H, E), o.bank(gen, H, inter, E)
    lw, ls = o.bank(gen, 160, H)
    bias = torch.randn(160, generator=gen, device="cuda").to(dtype)
    dy = torch.randn((T, 160), generator=gen, device="cuda").to(dtype)
    out = [("sort_tokens", (x, inds, E), lambda: ops.sort_tokens(x, inds, E)), ("sort_tokens_grad", (rows, inverse), lambda: ops.sort_tokens_grad(rows, inverse)),
           ("unsort_tokens", (rows, w, inverse), lambda: ops.unsort_tokens(rows, w, inverse)),
           ("unsort_tokens_grad", (dout, rows, w, inverse), lambda: ops.unsort_tokens_grad(dout, rows, w, inverse)),
           ("linear_f8", (x, lw, ls, bias, True), lambda: ops.linear_f8(x, lw, ls, bias)), ("linear_f8", (x, lw, ls, None, True), lambda: ops.linear_f8(x, lw, ls)),
           ("linear_f8", (dy, lw, ls, None, False), lambda: ops.linear_f8(dy, lw, ls, transpose=False)),
           ("grouped_linear_f8", (rows, *gate, offsets, True), lambda: ops.grouped_linear_f8(rows, *gate, offsets)),
           ("grouped_linear_f8", (rows, *down, offsets, False), lambda: ops.grouped_linear_f8(rows, *down, offsets, False))]
    if dtype != torch.float32:
        out += [("switch_glu_f8", (x, inds, w, *gate, *up, *down), lambda: ops.switch_glu_f8(x, inds, w, gate, up, down)),
                ("switch_glu_f8_grad", (dout, x, inds, w, *gate, *up, *down), lambda: ops.switch_glu_f8_grad(dout, x, inds, w, gate, up, down))]
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [0, 1, 40, 1200])
def test_native_calls_equal_the_general_path(T, dtype, general):  # noqa: F811
    for name, args, run in calls(T, dtype):
        want = general(run)
        assert same(run(), want), name
        if T == 0:
            assert native(name, args) is None, name
        else:
            assert same(native(name, args), want), name


def test_what_is_not_plain_goes_the_general_way():
    class Sub(torch.Tensor):
        pass

    for name, args, _ in calls(4, torch.bfloat16):
        assert native(name, args) is not None
        for i, a in enumerate(args):
            if isinstance(a, torch.Tensor):
                for v in (a.as_subclass(Sub), a.cpu(), a.tolist(), torch.stack([a, a], -1)[..., 0] if a.element_size() > 1 else a.transpose(-1, -2), a[None]):
                    if v is a or (isinstance(v, torch.Tensor) and type(v) is torch.Tensor and v.dim() == a.dim() + 1 and name == "linear_f8" and i in (0, 3)):
                        continue  # (a linear layer takes any leading axes)
                    wrong = list(args)
                    wrong[i] = v
                    assert native(name, wrong) is None, (name, i)
            elif a is True or a is False:
                assert native(name, [*args[:i], 1, *args[i + 1:]]) is None

"""The calls around the norm, the selection and the linear layer on 8-bit rows in native code against the general path: the same results, and what
they do not take (subclasses, transforms, strides, refusals) goes the general way."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
H, E, N = 128, 24, 48


def calls(shape, dtype):
    """Of every operator: its name, the native call's arguments, and the public call."""
    import mlx_rs_amd as m
    gen = torch.Generator(device="cuda").manual_seed(len(shape))
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, r, dy, dh = (rand(*shape, H).to(dtype) for _ in range(4))
    w, lb = rand(H).to(dtype), rand(N).to(dtype)
    q, s, b = m.ops.quantize(rand(N, H), 64, 4, dtype)
    x8, rs, _ = m.ops.add_rms_norm_rows8(x, None, w)
    logits, bias = rand(*shape, E).to(dtype), rand(E)
    inds, weights = m.ops.select_experts(logits, 3, dtype=dtype)
    o = m.ops
    return [("add_rms_norm", (x, r, w, 1e-5), lambda: o.add_rms_norm(x, r, w)),
            ("add_rms_norm", (x, None, w, 1e-5), lambda: o.add_rms_norm(x, None, w)),
            ("add_rms_norm_rows8", (x, r, w, 1e-6), lambda: o.add_rms_norm_rows8(x, r, w, 1e-6)),
            ("add_rms_norm_rows8", (x, None, w, 1), lambda: o.add_rms_norm_rows8(x, None, w, 1)),
            ("add_rms_norm_grad", (dy, x, w, 1e-5, dh), lambda: o.add_rms_norm_grad(dy, x, w, 1e-5, dh)),
            ("add_rms_norm_grad", (dy, x, w, 1e-5, None), lambda: o.add_rms_norm_grad(dy, x, w)),
            ("quantized_linear_rows8", (x8, rs, q, s, b, lb, 64, 4), lambda: o.quantized_linear_rows8(x8, rs, q, s, b, lb)),
            ("quantized_linear_rows8", (x8, rs, q, s, b, None, 64, 4), lambda: o.quantized_linear_rows8(x8, rs, q, s, b)),
            ("select_experts", (logits, 3, "softmax", None, 1, 1, "max", True, 1.0, dtype), lambda: o.select_experts(logits, 3, dtype=dtype)),
            ("select_experts", (logits, 4, "sigmoid", bias, 4, 2, "top2", False, 2.5, torch.bfloat16),
             lambda: o.select_experts(logits, 4, "sigmoid", bias, 4, 2, "top2", False, 2.5)),
            ("select_experts_grad", (weights, logits, inds, "softmax", True, 1.0), lambda: o.select_experts_grad(weights, logits, inds)),
            ("select_experts_grad", (weights, logits, inds, "sigmoid", False, 3), lambda: o.select_experts_grad(weights, logits, inds, "sigmoid", False, 3))]


@pytest.fixture
def general(monkeypatch):
    """Runs a call on the general path alone."""
    import mlx_rs_amd as m

    def run(fn):
        with monkeypatch.context() as c:
            c.setattr(m.ops, "_linear_call", lambda: lambda *a: None)
            return fn()
    return run


def many(v):
    return v if isinstance(v, tuple) else (v,)


def same(a, b):
    return len(many(a)) == len(many(b)) and all(u.dtype == v.dtype and u.device == v.device and torch.equal(u, v) for u, v in zip(many(a), many(b)))


def native(name, args):
    import mlx_rs_amd as m
    return getattr(m.ops._linear_call().__self__, name)(*args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (), (3, 5), (40,), (2, 0)])
def test_native_calls_equal_the_general_path(shape, dtype, general):
    for name, args, run in calls(shape, dtype):
        want = general(run)
        assert same(run(), want), name
        if 0 in shape:
            assert native(name, args) is None, name
            continue
        assert same(native(name, args), want), name
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = run()
        side.synchronize()
        assert same(other, want), name


def test_without_a_residual_the_sum_is_the_operand_itself():
    import mlx_rs_amd as m
    x, w = torch.randn((3, H), device="cuda"), torch.ones(H, device="cuda")
    assert m.ops.add_rms_norm(x, None, w)[1] is x and m.ops.add_rms_norm_rows8(x, None, w)[2] is x


def test_what_is_not_plain_goes_the_general_way():
    class Sub(torch.Tensor):
        pass

    for name, args, _ in calls((4,), torch.bfloat16):
        assert native(name, args) is not None
        for i, a in enumerate(args):
            if isinstance(a, torch.Tensor):
                wrong = [a.as_subclass(Sub), a.cpu(), a.double(), a.tolist()]
                if a.shape[-1:] != (E,) or a.dim() == 1:  # (twice as many logits are logits)
                    wrong.append(torch.cat([a, a], -1))
                if a.dim() > 1 or name not in ("add_rms_norm", "add_rms_norm_rows8", "add_rms_norm_grad"):
                    wrong.append(torch.stack([a, a], -1)[..., 0])
                for odd in wrong:
                    assert native(name, args[:i] + (odd,) + args[i + 1:]) is None, (name, i, type(odd))
                if i == 0:
                    seen = []
                    torch.func.vmap(lambda v: (seen.append(native(name, (v,) + args[1:])), v)[1])(a)
                    assert seen == [None]
            elif a is not None and not isinstance(a, torch.dtype):
                odd = [None, 10 ** 400, -10 ** 400, [], "none"] + ([1.5] if isinstance(a, (str, bool)) else [])
                for o in odd:
                    assert native(name, args[:i] + (o,) + args[i + 1:]) is None, (name, i, o)
        with pytest.raises(TypeError, match=name):
            native(name, args[:-1])


def test_refusals_are_worded():
    import mlx_rs_amd as m
    x, w = torch.randn((4, H), device="cuda"), torch.ones(H, device="cuda")
    logits = torch.randn((4, E), device="cuda")
    for fn, text in ((lambda: m.ops.add_rms_norm(x, x, w, -1.0), "eps"), (lambda: m.ops.add_rms_norm(x, x[:2], w), "residual"), (lambda: m.ops.select_experts(logits, 25), "top_k"),
                     (lambda: m.ops.select_experts(logits, 3, "tanh"), "scoring"), (lambda: m.ops.select_experts(logits, 3, n_groups=5), "groups"),
                     (lambda: m.ops.select_experts(logits, 3, dtype=torch.int32), "dtype")):
        with pytest.raises(m.MoeError, match=text):
            fn()


def test_the_interpreter_is_let_go_around_the_launch():
    """The library's functions replaced by CPython's own question whether this thread holds the interpreter: 0, as a status, is a result."""
    import ctypes as C
    import mlx_rs_amd as m
    held = C.cast(C.pythonapi.PyGILState_Check, C.c_void_p).value
    at = lambda n: C.cast(getattr(m.load_library(), "mi_moe_" + n), C.c_void_p).value  # noqa: E731
    all_calls = calls((4,), torch.bfloat16)
    try:
        m.ops._linear_call().__self__.bind_layer(held, held, at("add_rms_norm_grad_workspace_size"), held, at("quantized_linear_rows8_workspace_size"), held, held, held)
        for name, args, _ in all_calls:
            assert not isinstance(native(name, args), (int, type(None))), name
    finally:
        m.ops._linear_call.cache_clear()
        m.ops._linear_call()
    for name, args, run in all_calls:
        assert same(native(name, args), run())


@pytest.mark.parametrize("after", [0, 1])
def test_what_a_mode_raises_from_an_allocation_is_what_the_caller_sees(after, general):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Refuses(TorchDispatchMode):
        left = after

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if "empty" in str(func):
                self.left -= 1
                if self.left < 0:
                    raise LookupError("no allocations here")
            return func(*args, **(kwargs or {}))

    for name, args, run in calls((4,), torch.bfloat16):
        want = run()
        if after and len(many(want)) == 1 or name == "add_rms_norm" and args[1] is None:
            continue  # (one allocation)
        with pytest.raises(LookupError, match="no allocations here"), Refuses():
            run()
        assert same(run(), want)


def test_native_calls_under_capture():
    for name, args, run in calls((33,), torch.bfloat16):
        want = tuple(t.clone() for t in many(run()))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = run()
        for _ in range(3):
            for t in many(y):
                if not any(t is a for a in args):
                    t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert same(tuple(many(y)), want) and same(tuple(many(run())), want), name

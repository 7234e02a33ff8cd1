"""The residual's addition with the norm behind it, its rows in eight bits, and its backward pass, against float64."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step, relative
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# rows x hidden: one value, less than an octet, odd rows on every kernel (a wave a row up to 1024 values, 256 threads up to 8192, 1024 beyond), both sides of each
# line, last octets of every length, more rows than a block has
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 511), (9, 512), (7, 520), (3, 1023), (6, 1024), (1, 1025), (4, 2045), (3, 2048), (2, 4091), (1, 4096), (3, 5120), (2, 8190),
          (1, 8200), (2, 16384), (1, 20001), (1, 32768), (0, 64), (700, 96), (300, 2050)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def operands(T, H, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed * 1000003 + T * 40009 + H)
    x, r, dy, dh = (torch.randn(T, H, generator=gen).to(dtype).cuda() * s for s in (1.0, 1.5, 1.0, 0.7))
    return x, r, (1.0 + 0.2 * torch.randn(H, generator=gen)).to(dtype).cuda(), dy, dh


def truth(h, w, eps):
    h = h.double()
    return w.double() * h / (h.square().mean(-1, keepdim=True) + eps).sqrt()


def check_norm(y, h, x, r, w, eps):
    assert torch.equal(h, x if r is None else (x.float() + r.float()).to(x.dtype))
    ref = truth(h, w, eps)
    # one rounding to the type; in float32 before it: mean, its sum with eps, square root and quotient (each half a step, the first two halved by the root; the
    # root and the quotient may be a whole one off), two products: six half steps at most.  Below the normal numbers a step is that of the smallest.
    bound = (half_step(y.dtype) + 8 * U) * ref.abs() + torch.finfo(y.dtype).smallest_normal * 2 * half_step(y.dtype)
    assert bool(((y.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_add_rms_norm(dtype, T, H):
    import mlx_rs_amd as m
    x, r, w, _, _ = operands(T, H, dtype)
    for residual in (r, None):
        y, h = m.ops.add_rms_norm(x, residual, w, 1e-6)
        assert y.shape == x.shape and y.dtype == dtype
        check_norm(y, h, x, residual, w, 1e-6)
        if dtype == torch.bfloat16 and H % 8 == 0 and T:
            assert torch.equal(y, m.ops.rms_norm(h, w, 1e-6))  # the same bits


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_in_eight_bits(dtype, T, H):
    import mlx_rs_amd as m
    x, r, w, _, _ = operands(T, H, dtype, 1)
    q, s, h = m.ops.add_rms_norm_rows8(x, r, w, 1e-6)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    p = h.double() * w.double()  # exact
    most = p.abs().amax(-1, keepdim=True) if T else p[:, :1]
    assert torch.equal(q.double(), torch.where(most > 0, (127.0 * p / most).round(), torch.zeros_like(p)))
    rstd = 1.0 / (h.double().square().mean(-1) + 1e-6).sqrt()
    ref = most[:, 0] * rstd / 127.0
    assert bool(((s.double() - ref).abs() <= 6 * U * ref).all())


@pytest.mark.parametrize("T,H", SHAPES + [(2500, 640), (3000, 1500), (1100, 4096)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(dtype, T, H):
    """Against torch's derivative of the definition in float64."""
    import mlx_rs_amd as m
    h, _, w, dy, dh = operands(T, H, dtype, 2)
    h64, w64 = h.double().requires_grad_(), w.double().requires_grad_()
    y = w64 * h64 / (h64.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    (y * dy.double()).sum().backward()
    rstd = 1.0 / (h.double().square().mean(-1, keepdim=True) + 1e-5).sqrt()
    hat, wdy = h.double() * rstd, w.double() * dy.double()
    one, two = (rstd * wdy).abs(), (rstd * hat * (wdy * hat).mean(-1, keepdim=True)).abs()  # the terms of a result
    products = (dy.double() * hat).abs().sum(0)
    below = torch.finfo(dtype).smallest_normal * half_step(dtype) * 2  # half a step of what is below the normal numbers is smallest_normal * eps / 2
    for through in (dh, None):
        dx, dw = m.ops.add_rms_norm_grad(dy, h, w, 1e-5, through)
        ref = h64.grad + (0 if through is None else through.double())
        # float32 before the rounding.  rstd: the mean and its sum with eps are half a step off, which the root halves, the root and the quotient one each: three.
        # First term: rstd, the product with it, that of w and dy, the difference: six.  Second: rstd in hat, in the mean and in front, and a product or a rounding with
        # each, the difference: thirteen (the mean's sum is float64's).  The sum with dh: half a step of the result.
        bound = half_step(dtype) * ref.abs() + U * (6 * one + 13 * two + 2 * ref.abs()) + below
        assert bool(((dx.double() - ref).abs() <= bound).all())
        # float32 sums in any order lose at most a half step of the sum of sizes for every addition a term goes through, and hat has five
        additions = min(T, 64 + T // 256 + 600)
        assert bool(((dw.double() - w64.grad).abs() <= half_step(dtype) * w64.grad.abs() + (additions + 6) * U * products + below).all())
    dx2, dw2 = m.ops.add_rms_norm_grad(dy, h, w, 1e-5)
    assert torch.equal(dw, dw2) and torch.equal(dx, dx2)  # (the order does not change)


def test_gradient_against_differences():
    """d/dt of sum(dy y) along a direction, from differences of the definition in float64 (their error is of the order t^2, 1e-8) and from the kernel."""
    import mlx_rs_amd as m
    h, _, w, dy, d = operands(5, 300, torch.float32, 3)
    dx, dw = m.ops.add_rms_norm_grad(dy, h, w, 1e-5)
    t, h64, w64 = 1e-4, h.double(), w.double()

    def value(hh, ww):
        return float((dy.double() * truth(hh, ww, 1e-5)).sum())

    along = (value(h64 + t * d.double(), w64) - value(h64 - t * d.double(), w64)) / (2 * t)
    assert abs(float((dx.double() * d.double()).sum()) - along) <= 1e-5 * float((dx.double() * d.double()).abs().sum())
    v = d[0].double()
    along = (value(h64, w64 + t * v) - value(h64, w64 - t * v)) / (2 * t)
    assert abs(float((dw.double() * v).sum()) - along) <= 1e-5 * float((dw.double() * v).abs().sum())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros_infinities_and_extremes(dtype):
    import mlx_rs_amd as m
    H = 264
    x, r, w, dy, _ = operands(6, H, dtype, 4)
    x[0] = 0
    r[0] = 0
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    big = 3e4 if dtype == torch.float16 else 1e30  # (squares beyond float32, not float64)
    x[3], r[3] = big, 0
    tiny = 6e-8 if dtype == torch.float16 else 1e-37  # (squares below float32)
    x[4], r[4] = tiny, 0
    y, h = m.ops.add_rms_norm(x, r, w, 0.0)
    q, s, h8 = m.ops.add_rms_norm_rows8(x, r, w, 0.0)
    assert torch.equal(h.view(torch.int16 if dtype != torch.float32 else torch.int32), h8.view(torch.int16 if dtype != torch.float32 else torch.int32))
    for t in (3, 4, 5):
        check_norm(y[t:t + 1], h[t:t + 1], x[t:t + 1], r[t:t + 1], w, 0.0)
    assert not q[0].any() and not q[1].any() and not q[2].any()
    assert torch.isnan(s[1]) and torch.isnan(s[2]) and torch.isfinite(s[3:]).all()
    q0, s0, _ = m.ops.add_rms_norm_rows8(x[:1], r[:1], w, 1e-5)
    y0, _ = m.ops.add_rms_norm(x[:1], r[:1], w, 1e-5)
    assert not y0.any() and float(s0) == 0.0 and not q0.any()
    # other rows of the batch are as they are alone
    y5, _ = m.ops.add_rms_norm(x[5:], r[5:], w, 0.0)
    assert torch.equal(y[5:], y5)
    dx, _ = m.ops.add_rms_norm_grad(dy, h, w, 1e-5)
    dx5, _ = m.ops.add_rms_norm_grad(dy[5:].contiguous(), h[5:].contiguous(), w, 1e-5)
    assert torch.equal(dx[5:], dx5)


def test_halfway_codes():
    """Products halfway between two codes go to the even one: 127 p / most = n + 1/2 exactly."""
    import mlx_rs_amd as m
    x = torch.zeros(1, 16, dtype=torch.float32, device="cuda")
    x[0, 0] = 254.0
    x[0, 1:8] = torch.tensor([1.0, 3.0, 5.0, -1.0, -3.0, 251.0, 253.0])
    q, _, _ = m.ops.add_rms_norm_rows8(x, None, torch.ones(16, device="cuda"), 1e-6)
    assert q[0, :8].tolist() == [127, 0, 2, 2, 0, -2, 126, 126]


def test_unaligned_rows_and_updates_in_place():
    """Operands that start anywhere, and the sum written over the residual, through the C entry."""
    import mlx_rs_amd as m
    lib = m.load_library()
    for dtype in DTYPES:
        T, H, dt = 5, 1003, m.ops._DTYPES[dtype]
        x, r, w, dy, dh = operands(T, H, dtype, 5)
        y, h = m.ops.add_rms_norm(x, r, w, 1e-6)
        dx, dw = m.ops.add_rms_norm_grad(dy, h, w, 1e-6, dh)

        def shifted(t):
            flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
            flat[1:] = t.reshape(-1)
            return flat

        xs, rs, ws, dys, hs, dhs = (shifted(t) for t in (x, r, w, dy, h, dh))
        ys = torch.zeros(T * H + 2, dtype=dtype, device="cuda")
        at = lambda t: t.data_ptr() + t.element_size()  # noqa: E731
        m.capi.check(lib.mi_moe_add_rms_norm(at(xs), at(rs), at(ws), 1e-6, T, H, dt, at(rs), at(ys), m.ops._stream()))
        assert torch.equal(ys[1:-1], y.reshape(-1)) and float(ys[0]) == 0 and float(ys[-1]) == 0
        assert torch.equal(rs[1:], h.reshape(-1))
        room = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        out = torch.zeros(H + 2, dtype=dtype, device="cuda")
        m.capi.check(lib.mi_moe_add_rms_norm_grad(at(dys), at(hs), at(dhs), at(ws), 1e-6, T, H, dt, at(dhs), at(out), room.data_ptr(), room.numel(), m.ops._stream()))
        assert torch.equal(dhs[1:], dx.reshape(-1)) and torch.equal(out[1:-1], dw) and float(out[0]) == 0 and float(out[-1]) == 0


def test_more_values_than_32_bits_count():
    import mlx_rs_amd as m
    T, H = 131100, 32768  # 2^32 values and some rows
    h = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    h.fill_(2.0)
    h[-1] = 0.5
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    y, _ = m.ops.add_rms_norm(h, None, w, 0.0)
    assert bool((y[::9000] == 1).all()) and bool((y[-2:] == 1).all())
    del y
    q, s, _ = m.ops.add_rms_norm_rows8(h, None, w, 0.0)
    assert bool((q[-1] == 127).all()) and bool((q[::9000] == 127).all()) and abs(float(s[-1]) * 127 - 1) < 1e-6
    del q, s, h, w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("with_residual", [True, False])
def test_more_rows_than_a_launch_takes(with_residual):
    """2^21 rows a launch: the rows around its end and the last ones, as in a call of their own."""
    import mlx_rs_amd as m
    T, H = 2 ** 21 + 5, 24
    x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    r = torch.randn(T, H, device="cuda").to(torch.bfloat16) if with_residual else None
    w = torch.randn(H, device="cuda").to(torch.bfloat16)
    got = m.ops.add_rms_norm(x, r, w) + m.ops.add_rms_norm_rows8(x, r, w)
    for part in (slice(0, 9), slice(2 ** 21 - 7, 2 ** 21 + 3), slice(T - 4, T)):
        some = (x[part].contiguous(), None if r is None else r[part].contiguous(), w)
        for a, b in zip(got, m.ops.add_rms_norm(*some) + m.ops.add_rms_norm_rows8(*some)):
            assert torch.equal(a[part], b)


def test_refusals():
    import mlx_rs_amd as m
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: m.ops.add_rms_norm(x, x.float(), w), lambda: m.ops.add_rms_norm(x, x[:2], w), lambda: m.ops.add_rms_norm(x, x, w[:32]),
                 lambda: m.ops.add_rms_norm(x.t(), None, w), lambda: m.ops.add_rms_norm(x, None, w.float()), lambda: m.ops.add_rms_norm(x.double(), None, w),
                 lambda: m.ops.add_rms_norm(x, None, w, -1.0), lambda: m.ops.add_rms_norm_grad(x, x, w, 1e-5, x[:1]), lambda: m.ops.add_rms_norm_grad(x[:1], x, w),
                 lambda: m.ops.add_rms_norm_rows8(x, x[:, :32], w)):
        with pytest.raises(m.MoeError):
            call()

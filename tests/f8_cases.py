"""Oracles in 64 bits for the e4m3 operators and the sorted tokens, with bounds of what their results may be off by."""
import torch

RUN = 128
F8 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}  # the least positive value: below the normal ones half of it is the rounding's error


def blocks(n):
    return -(-n // RUN)


def to_e4m3(q):
    """The nearest value of the type's grid (ties to even): four significant bits down to 2^-6, steps of 2^-9 below."""
    step = torch.exp2(torch.frexp(q)[1].double().sub(1).clamp(min=-6) - 3)
    return torch.clamp(torch.round(q / step) * step, -448.0, 448.0)


def runs_of(x, size=RUN):
    for c in range(0, x.shape[-1], size):
        yield slice(c, min(c + size, x.shape[-1]))


def quantize_rows(x):
    """(codes as float64, scales float64 [rows, runs]) by the definition: scale and quotient rounded to float32."""
    x = x.double()
    codes = torch.zeros_like(x)
    scales = torch.zeros(x.shape[0], blocks(x.shape[1]), dtype=torch.float64, device=x.device)
    for j, c in enumerate(runs_of(x)):
        most = x[:, c].abs().amax(-1, keepdim=True)
        s = torch.where(most < float("inf"), (most / 448.0).float().double(), float("nan"))  # (NaN: not below)
        fine = s > 0
        codes[:, c] = torch.where(fine, to_e4m3(torch.nan_to_num((x[:, c] / torch.where(fine, s, 1.0)).float().double())), 0.0)
        scales[:, j] = s[:, 0]
    return codes, scales


def spread(scales, n, k):
    """A bank's block scales over its values."""
    return scales.double().repeat_interleave(RUN, -2)[..., :n, :].repeat_interleave(RUN, -1)[..., :k]


def product(codes, scales, w, ws, bias, dtype):
    """q(x) . W^T for codes [M, K], scales [M, runs], W codes [N, K] as float64 and block scales: the result and what one of `dtype` may be off by.
    A run's sum of 128 exact products on the f8 instructions: each product loses what lies below 2^-13 of the largest one, in either direction, 128 of them at random
    2^-13 sqrt(128) / 2 = 2^-10.5 of it; 2^-9.5 is allowed for.  In float32 (results of that type): (128 + runs) roundings of the sum of the magnitudes."""
    M, K = codes.shape
    N = w.shape[0]
    y = torch.zeros(M, N, dtype=torch.float64, device=codes.device)
    mags, runs_most = torch.zeros_like(y), torch.zeros_like(y)
    for j, c in enumerate(runs_of(codes)):
        s = scales[:, j:j + 1] * ws[:, j].double().repeat_interleave(RUN)[None, :N]
        y += torch.nan_to_num(s) * (codes[:, c] @ w[:, c].t()) + torch.where(s.isnan(), s, 0.0)
        s = torch.nan_to_num(s).abs()
        mags += s * (codes[:, c].abs() @ w[:, c].abs().t())
        for n in range(0, N, 64):
            runs_most[:, n:n + 64] += s[:, n:n + 64] * (codes[:, None, c].abs() * w[None, n:n + 64, c].abs()).amax(-1)
    if bias is not None:
        y = y + bias.double()
    off = mags * (RUN + scales.shape[1] + 2) * 2.0 ** -24
    if dtype != torch.float32:
        off = off + runs_most * 2.0 ** -9.5
    return y, off


def within(got, want, off, what=""):
    """got of a type against want in 64 bits, which may be off by `off` before the rounding to that type."""
    bound = off + HALF_STEP[got.dtype] * (want.abs() + off) + LEAST[got.dtype] / 2
    d = (got.double() - want).abs()
    same_nan = torch.equal(got.isnan(), want.isnan())
    d, bound = d[~want.isnan()], bound[~want.isnan()]
    worst = (d / bound).max().item() if d.numel() else 0.0
    assert same_nan and worst <= 1.0, f"{what}: NaN where they belong: {same_nan}, worst error {worst:.3g} of its bound"
    return worst


def bank(gen, n, k, experts=None):
    """e4m3 weights over the type's range, zeros and denormals among them, and scales of their blocks."""
    lead = () if experts is None else (experts,)
    w = torch.randn(lead + (n, k), generator=gen, device="cuda") * 90.0
    w = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.1, w * 1e-4, w).clamp(-448, 448).to(F8)
    s = (0.5 + torch.rand(lead + (blocks(n), blocks(k)), generator=gen, device="cuda")) * 2e-4
    return w, s


def sort(inds, experts):
    """order, inverse, offsets, by Python's own sort."""
    flat = [int(e) if 0 <= int(e) < experts else experts for e in inds.reshape(-1).tolist()]
    order = sorted(range(len(flat)), key=lambda p: flat[p])
    inverse = [0] * len(flat)
    for r, p in enumerate(order):
        inverse[p] = r if flat[p] < experts else -1 - r
    offsets = [sum(f < e for f in flat) for e in range(experts + 1)]
    return order, inverse, offsets

"""include/mi_moe_f8.h without a GPU: what it declares is exported, bound and mirrored in Rust, and bad arguments come back as a status with a message before anything is
launched."""
import ctypes as C
import os
import re

import pytest

import test_rust_shim_abi as abi
from test_layer_host import P, lib, refused  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mi_moe_f8.h")
RUST = os.path.join(ROOT, "mlx-rs_amd", "rust", "mi-moe-sys", "src", "f8.rs")


def test_the_header_is_exported_and_bound(lib):  # noqa: F811
    import mlx_rs_amd as m
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(mi_moe_[a-z_0-9]+)\s*\(", text)))
    assert names == sorted(m.capi.F8_EXPORTS) and not set(names) & set(m.capi.EXPORTS + m.capi.LAYER_EXPORTS)
    for n in names:
        assert getattr(lib, n).argtypes, n


def test_the_rust_declarations_are_the_header_s(monkeypatch):
    monkeypatch.setattr(abi, "HEADER", HEADER)
    monkeypatch.setattr(abi, "RUST", RUST)
    monkeypatch.setitem(abi.C_TO_RUST, "mi_moe_f8_experts", "mi_moe_f8_experts")
    header, rust = abi.parse_header(), abi.parse_rust()
    assert len(header[0]) == 13 and rust[0] == header[0] and rust[1] == header[1] and list(header[1]) == ["mi_moe_f8_experts"]
    import mlx_rs_amd as m
    assert [n for n, _ in m.capi.F8Experts._fields_] == [n for n, _ in header[1]["mi_moe_f8_experts"]]


SLOTS = [("top_k", dict(k=0)), ("top_k", dict(k=33)), ("token count", dict(T=-1)), ("token count", dict(T=(1 << 24) // 2)), ("hidden", dict(H=0)),
         ("hidden", dict(H=(1 << 22) + 1)), ("dtype", dict(dt=3))]


@pytest.mark.parametrize("needle,change", SLOTS)
def test_sorted_tokens_refusals(lib, needle, change):  # noqa: F811
    a = dict(T=4, k=2, H=8, dt=0)
    a.update(change)
    T, k, H, dt = a["T"], a["k"], a["H"], a["dt"]
    refused(lib, needle, "mi_moe_sort_tokens", P, P, T, k, 8, H, dt, P, P, P, P, None, 0, None)
    refused(lib, needle, "mi_moe_sort_tokens_grad", P, P, T, k, H, dt, P, None)
    refused(lib, needle, "mi_moe_unsort_tokens", P, P, 0, P, T, k, H, dt, P, None)
    refused(lib, needle, "mi_moe_unsort_tokens_grad", P, P, P, 0, P, T, k, H, dt, P, P, None)


def test_more_sorted_tokens_refusals(lib):  # noqa: F811
    for E in (0, 513):
        refused(lib, "n_experts", "mi_moe_sort_tokens", P, P, 4, 2, E, 8, 0, P, P, P, P, None, 0, None)
    for i in (1, 8, 9, 10):
        args = [P, P, 4, 2, 8, 8, 0, P, P, P, P, None, 0, None]
        args[i] = None
        refused(lib, "non-NULL", "mi_moe_sort_tokens", *args)
    refused(lib, "non-NULL", "mi_moe_sort_tokens", None, P, 4, 2, 8, 8, 0, P, P, P, P, None, 0, None)  # (rows of nothing)
    n = C.c_size_t()
    assert lib.mi_moe_sort_tokens_workspace_size(2000, 2, 8, C.byref(n)) == 0 and n.value
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        refused(lib, "workspace", "mi_moe_sort_tokens", P, P, 2000, 2, 8, 8, 0, P, P, P, P, ws, size, None)
    refused(lib, "bytes", "mi_moe_sort_tokens_workspace_size", 1, 1, 1, None)
    refused(lib, "dtype", "mi_moe_unsort_tokens", P, P, 7, P, 4, 2, 8, 0, P, None)
    refused(lib, "drows", "mi_moe_unsort_tokens_grad", P, P, P, 0, P, 4, 2, 8, 0, P, P, None)
    for name, args, at in (("sort_tokens_grad", [P, P, 4, 2, 8, 0, P, None], (0, 1, 6)), ("unsort_tokens", [P, P, 0, P, 4, 2, 8, 0, P, None], (0, 1, 3, 8)),
                           ("unsort_tokens_grad", [P, P, P, 0, P, 4, 2, 8, 0, P + 64, P, None], (0, 1, 2, 4, 9, 10))):
        for i in at:
            refused(lib, "non-NULL", "mi_moe_" + name, *[None if j == i else v for j, v in enumerate(args)])
    assert lib.mi_moe_sort_tokens_grad(None, None, 0, 2, 8, 0, None, None) == 0
    assert lib.mi_moe_unsort_tokens(None, None, 0, None, 0, 2, 8, 0, None, None) == 0
    assert lib.mi_moe_unsort_tokens_grad(None, None, None, 0, None, 0, 2, 8, 0, None, None, None) == 0


@pytest.mark.parametrize("needle,change", [("dtype", dict(dt=-1)), ("block_rows", dict(b=64)), ("block_rows", dict(b=0)), ("cols", dict(c=0)), ("cols", dict(c=(1 << 22) + 1)),
                                           ("row count", dict(r=-1)), ("row count", dict(r=1 << 40)), ("non-NULL", dict(x=None)), ("non-NULL", dict(q=None)), ("non-NULL", dict(s=None))])
def test_codes_refusals(lib, needle, change):  # noqa: F811
    a = dict(x=P, q=P, s=P, r=4, c=200, b=1, dt=0)
    a.update(change)
    refused(lib, needle, "mi_moe_quantize_f8", a["x"], a["dt"], a["r"], a["c"], a["b"], a["q"], a["s"], None)
    refused(lib, needle, "mi_moe_dequantize_f8", a["q"], a["s"], a["r"], a["c"], a["b"], a["dt"], a["x"], None)


@pytest.mark.parametrize("needle,change", [
    ("dtype", dict(dt=3)), ("N and K", dict(N=0)), ("N and K", dict(K=0)), ("N and K", dict(N=(1 << 22) + 16)), ("multiple of 16", dict(K=120)), ("multiple of 16", dict(t=0, N=120)),
    ("row count", dict(M=-1)), ("row count", dict(M=(1 << 30) + 1, N=1, K=16)), ("row count", dict(M=1 << 30)), ("non-NULL", dict(x=None)), ("non-NULL", dict(w=None)),
    ("non-NULL", dict(s=None)), ("non-NULL", dict(y=None)), ("16-byte", dict(w=P + 8)), ("workspace", dict(ws=None)), ("workspace", dict(ws=P + 8)), ("workspace", dict(short=1))])
def test_linear_refusals(lib, needle, change):  # noqa: F811
    a = dict(x=P, w=P, s=P, M=5, N=48, K=128, t=1, dt=0, y=P, ws=P, short=0)
    a.update(change)
    n = C.c_size_t()
    assert lib.mi_moe_linear_f8_workspace_size(5, max(a["N"], 1) % (1 << 22), 128, C.byref(n)) == 0
    size = n.value - a["short"]
    refused(lib, needle, "mi_moe_linear_f8", a["x"], a["w"], a["s"], None, a["M"], a["N"], a["K"], a["t"], a["dt"], a["y"], a["ws"], size, None)
    refused(lib, needle, "mi_moe_grouped_linear_f8", a["x"], a["w"], a["s"], P, a["M"], 2, a["N"], a["K"], a["t"], a["dt"], a["y"], a["ws"], size, None)


def test_more_linear_refusals(lib):  # noqa: F811
    refused(lib, "transpose", "mi_moe_linear_f8", P, P, P, P, 5, 48, 128, 0, 0, P, P, 1 << 20, None)
    refused(lib, "offsets", "mi_moe_grouped_linear_f8", P, P, P, None, 5, 2, 48, 128, 1, 0, P, P, 1 << 20, None)
    for E in (0, 513):
        refused(lib, "n_experts", "mi_moe_grouped_linear_f8", P, P, P, P, 5, E, 48, 128, 1, 0, P, P, 1 << 20, None)
    refused(lib, "bytes", "mi_moe_linear_f8_workspace_size", 1, 16, 16, None)
    refused(lib, "bad sizes", "mi_moe_linear_f8_workspace_size", -1, 16, 16, C.byref(C.c_size_t()))
    assert lib.mi_moe_linear_f8(None, None, None, None, 0, 48, 128, 1, 0, None, None, 0, None) == 0
    assert lib.mi_moe_grouped_linear_f8(None, None, None, None, 0, 3, 48, 128, 1, 0, None, None, 0, None) == 0
    assert lib.mi_moe_quantize_f8(None, 0, 0, 8, 1, None, None, None) == 0 and lib.mi_moe_dequantize_f8(None, None, 0, 8, 1, 0, None, None) == 0


@pytest.mark.parametrize("needle,change", SLOTS + [
    ("F16", dict(dt=2)), ("multiples of 16", dict(H=120)), ("multiples of 16", dict(I=40)), ("multiples of 16", dict(I=0)), ("n_experts", dict(E=0)), ("2^32", dict(T=1 << 20, k=1, H=4096)),
    ("n_experts", dict(E=513)), ("dtype", dict(wt=4)), ("weights and scales", dict(banks=None)), ("weights and scales", dict(up=None)), ("16-byte", dict(up=P + 8)),
    ("non-NULL", dict(x=None)), ("non-NULL", dict(idx=None)), ("non-NULL", dict(w=None)), ("non-NULL", dict(out=None)), ("workspace", dict(ws=None)), ("workspace", dict(short=1))])
def test_experts_refusals(lib, needle, change):  # noqa: F811
    import mlx_rs_amd as m
    a = dict(x=P, idx=P, w=P, wt=0, up=P, T=4, H=256, I=128, E=8, k=2, dt=0, out=P, ws=P, short=0)
    a.update(change)
    banks = m.capi.F8Experts(P, a["up"], P, P, P, P)
    banks = None if "banks" in a else C.byref(banks)
    for grad in (0, 1):
        n = C.c_size_t()
        assert lib.mi_moe_switch_glu_f8_workspace_size(4, 256, 128, 8, 2, grad, C.byref(n)) == 0
        rest = (a["x"], a["idx"], a["w"], a["wt"], banks, a["T"], a["H"], a["I"], a["E"], a["k"], a["dt"], a["out"])
        ws = (a["ws"], n.value - a["short"], None)
        if grad:
            refused(lib, needle, "mi_moe_switch_glu_f8_grad", P, *rest, P, *ws)
        else:
            refused(lib, needle, "mi_moe_switch_glu_f8", *rest, *ws)
    assert lib.mi_moe_switch_glu_f8(None, None, None, 0, None, 0, 256, 128, 8, 2, 0, None, None, 0, None) == 0
    assert lib.mi_moe_switch_glu_f8_grad(None, None, None, None, 0, None, 0, 256, 128, 8, 2, 0, None, None, None, 0, None) == 0


def test_workspaces_grow_with_the_batch(lib):  # noqa: F811
    counts = list(range(0, 700)) + [1000, 4096, 5000, 16384, 100000]

    def sizes(fn, *rest, tokens=counts):
        n = C.c_size_t()
        for t in tokens:
            assert getattr(lib, fn)(t, *rest, C.byref(n)) == 0
            yield n.value

    for fn, rest in (("mi_moe_sort_tokens_workspace_size", (8, 128)), ("mi_moe_linear_f8_workspace_size", (4096, 2048)), ("mi_moe_linear_f8_workspace_size", (1, 16)),
                     ("mi_moe_switch_glu_f8_workspace_size", (2048, 768, 128, 8, 0)), ("mi_moe_switch_glu_f8_workspace_size", (2048, 768, 128, 8, 1)),
                     ("mi_moe_switch_glu_f8_workspace_size", (272, 400, 2, 1, 0))):
        got = list(sizes(fn, *rest))
        assert got == sorted(got), fn


def test_python_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    import mlx_rs_amd as m
    x, ids = torch.zeros(2, 16, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32)
    w, s = torch.zeros(16, 16).to(torch.float8_e4m3fn), torch.ones(1, 1)
    rows = torch.zeros(4, 16)
    bank = (w[None], s[None])
    for call in (lambda: m.ops.sort_tokens(x, ids, 4), lambda: m.ops.sort_tokens_grad(rows, ids), lambda: m.ops.unsort_tokens(rows, x[:, :2].contiguous(), ids),
                 lambda: m.ops.unsort_tokens_grad(x.float(), rows, x[:, :2].contiguous(), ids), lambda: m.ops.quantize_f8(x), lambda: m.ops.dequantize_f8(w, s),
                 lambda: m.ops.linear_f8(x, w, s), lambda: m.ops.grouped_linear_f8(x, *bank, ids[0]), lambda: m.ops.switch_glu_f8(x, ids, x[:, :2].contiguous(), bank, bank, bank),
                 lambda: m.ops.switch_glu_f8_grad(x, x, ids, x[:, :2].contiguous(), bank, bank, bank)):
        with pytest.raises(m.MoeError, match="device tensor"):
            call()

"""include/mi_moe_layer.h without a GPU: what it declares is exported, bound and mirrored in Rust, and bad arguments come back as a status with a
message before anything is launched."""
import ctypes as C
import os
import re

import pytest

import test_rust_shim_abi as abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mi_moe_layer.h")
RUST = os.path.join(ROOT, "mlx-rs_amd", "rust", "mi-moe-sys", "src", "layer.rs")


@pytest.fixture(scope="module")
def lib():
    import mlx_rs_amd as m
    return m.load_library()


def test_the_header_is_exported_and_bound(lib):
    import mlx_rs_amd as m
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(mi_moe_[a-z_0-9]+)\s*\(", text)))
    assert names == sorted(m.capi.LAYER_EXPORTS) and not set(names) & set(m.capi.EXPORTS)
    for n in names:
        assert getattr(lib, n).argtypes, n


def test_the_rust_declarations_are_the_header_s(monkeypatch):
    monkeypatch.setattr(abi, "HEADER", HEADER)
    monkeypatch.setattr(abi, "RUST", RUST)
    header, rust = abi.parse_header(), abi.parse_rust()
    assert len(header[0]) == 9 and rust[0] == header[0]
    values = {a: int(b) for a, b in re.findall(r"(MI_MOE_(?:SCORING|GROUP_SCORE)_\w+)\s*=\s*(\d+)", open(HEADER).read())}
    assert len(values) == 4 and rust[2] == values
    import mlx_rs_amd as m
    for name, v in values.items():
        assert getattr(m.capi, name[len("MI_MOE_"):]) == v


P = 64  # an address that nothing follows: the calls below end before a launch


def refused(lib, needle, fn, *args):
    import mlx_rs_amd as m
    assert getattr(lib, fn)(*args) != 0
    assert needle in m.capi.last_error(), m.capi.last_error()


@pytest.mark.parametrize("needle,change", [
    ("row count", dict(T=-1)), ("row count", dict(T=(1 << 30) + 1)), ("hidden", dict(H=0)), ("hidden", dict(H=32769)), ("eps", dict(eps=-1.0)),
    ("eps", dict(eps=float("nan"))), ("dtype", dict(dt=3)), ("dtype", dict(dt=-1)), ("non-NULL", dict(x=None)), ("non-NULL", dict(w=None)),
    ("sum", dict(sum=None)), ("non-NULL", dict(y=None))])
def test_norm_refusals(lib, needle, change):
    a = dict(x=P, r=P, w=P, eps=1e-5, T=4, H=128, dt=0, sum=P, y=P)
    a.update(change)
    refused(lib, needle, "mi_moe_add_rms_norm", a["x"], a["r"], a["w"], a["eps"], a["T"], a["H"], a["dt"], a["sum"], a["y"], None)
    refused(lib, needle, "mi_moe_add_rms_norm_rows8", a["x"], a["r"], a["w"], a["eps"], a["T"], a["H"], a["dt"], a["sum"], a["y"], P, None)
    if needle != "sum":
        refused(lib, needle, "mi_moe_add_rms_norm_grad", a["x"], P, None, a["w"], a["eps"], a["T"], a["H"], a["dt"], a["y"], P, P, 1 << 30, None)


def test_norm_scales_workspace_and_empty_batches(lib):
    refused(lib, "row_scales", "mi_moe_add_rms_norm_rows8", P, P, P, 1e-5, 4, 128, 0, P, P, None, None)
    n = C.c_size_t(7)
    assert lib.mi_moe_add_rms_norm_grad_workspace_size(4, 128, C.byref(n)) == 0 and n.value >= 512
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        refused(lib, "workspace", "mi_moe_add_rms_norm_grad", P, P, None, P, 1e-5, 4, 128, 0, P, P, ws, size, None)
    refused(lib, "dweight", "mi_moe_add_rms_norm_grad", P, P, None, P, 1e-5, 4, 128, 0, P, None, P, n.value, None)
    refused(lib, "bad sizes", "mi_moe_add_rms_norm_grad_workspace_size", -1, 128, C.byref(n))
    refused(lib, "bytes", "mi_moe_add_rms_norm_grad_workspace_size", 1, 128, None)
    assert lib.mi_moe_add_rms_norm(None, None, None, 1e-5, 0, 128, 0, None, None, None) == 0
    assert lib.mi_moe_add_rms_norm_rows8(None, None, None, 1e-5, 0, 128, 0, None, None, None, None) == 0


@pytest.mark.parametrize("needle,change", [
    ("dtype", dict(dt=9)), ("dtype", dict(wt=3)), ("token count", dict(T=-1)), ("n_experts", dict(E=0)), ("n_experts", dict(E=513)), ("top_k", dict(k=0)),
    ("top_k", dict(k=33, E=64)), ("top_k", dict(k=17)), ("scoring", dict(scoring=2)), ("scale", dict(scale=float("inf"))),
    ("scale", dict(scale=float("nan"))), ("non-NULL", dict(l=None)), ("non-NULL", dict(idx=None)), ("non-NULL", dict(w=None)),
    ("n_groups", dict(groups=0)), ("n_groups", dict(groups=3)), ("n_groups", dict(groups=65, E=65)), ("top_groups", dict(open=0)), ("top_groups", dict(open=5)),
    ("open groups", dict(k=5, open=1)), ("group_score", dict(gs=2))])
def test_select_refusals(lib, needle, change):
    a = dict(l=P, dt=0, T=3, E=16, k=2, scoring=0, groups=4, open=2, gs=0, scale=1.0, idx=P, w=P, wt=0)
    a.update(change)
    refused(lib, needle, "mi_moe_select_experts", a["l"], a["dt"], None, a["T"], a["E"], a["k"], a["scoring"], a["groups"], a["open"], a["gs"], 1, a["scale"],
            a["idx"], a["w"], a["wt"], None)
    if not set(change) & {"groups", "open", "gs"}:
        refused(lib, needle, "mi_moe_select_experts_grad", a["w"], a["wt"], a["l"], a["dt"], a["idx"], a["T"], a["E"], a["k"], a["scoring"], 1, a["scale"], P, None)


def test_select_of_no_tokens(lib):
    assert lib.mi_moe_select_experts(None, 0, None, 0, 16, 2, 0, 1, 1, 0, 1, 1.0, None, None, 0, None) == 0
    assert lib.mi_moe_select_experts_grad(None, 0, None, 0, None, 0, 16, 2, 0, 1, 1.0, None, None) == 0


@pytest.mark.parametrize("needle,change", [
    ("dtype", dict(dt=3)), ("bits", dict(bits=2)), ("bits", dict(bits=3)), ("group_size", dict(group=16)), ("multiple of group_size", dict(K=96)),
    ("N must", dict(N=0)), ("N must", dict(K=0)), ("row count", dict(M=-1)), ("non-NULL", dict(x=None)), ("non-NULL", dict(sx=None)), ("non-NULL", dict(w=None)),
    ("non-NULL", dict(s=None)), ("non-NULL", dict(b=None)), ("non-NULL", dict(y=None))])
def test_linear_refusals(lib, needle, change):
    a = dict(x=P, sx=P, w=P, s=P, b=P, M=2, N=8, K=128, group=64, bits=4, dt=0, y=P)
    a.update(change)
    refused(lib, needle, "mi_moe_quantized_linear_rows8", a["x"], a["sx"], a["w"], a["s"], a["b"], None, a["M"], a["N"], a["K"], a["group"], a["bits"], a["dt"],
            a["y"], None, 0, None)


def test_linear_of_no_rows_and_its_workspace(lib):
    n = C.c_size_t(7)
    assert lib.mi_moe_quantized_linear_rows8(None, None, None, None, None, None, 0, 8, 128, 64, 4, 0, None, None, 0, None) == 0
    assert lib.mi_moe_quantized_linear_rows8_workspace_size(1000, 4096, C.byref(n)) == 0
    refused(lib, "bad sizes", "mi_moe_quantized_linear_rows8_workspace_size", 1, 0, C.byref(n))
    refused(lib, "bytes", "mi_moe_quantized_linear_rows8_workspace_size", 1, 128, None)


def test_routed_refusals(lib):
    refused(lib, "topk_idx", "mi_moe_forward_routed", None, P, None, P, 2, P, P, 1 << 20, None, None)
    refused(lib, "handle", "mi_moe_forward_routed", None, P, P, P, 2, P, P, 1 << 20, None, None)


def test_python_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    import mlx_rs_amd as m
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.ones(8, dtype=torch.bfloat16)
    for call in (lambda: m.ops.add_rms_norm(x, x, w), lambda: m.ops.add_rms_norm_rows8(x, x, w), lambda: m.ops.add_rms_norm_grad(x, x, w),
                 lambda: m.ops.select_experts(x, 2), lambda: m.ops.select_experts_grad(x, x, torch.zeros(2, 8, dtype=torch.int32)),
                 lambda: m.ops.quantized_linear_rows8(x.to(torch.int8), torch.ones(2), torch.zeros(2, 1, dtype=torch.int32), w, w)):
        with pytest.raises(m.MoeError, match="device tensor"):
            call()


@pytest.mark.parametrize("hidden", [1, 512, 1000, 1025, 2048, 4096, 8192, 32768])
def test_a_workspace_is_enough_for_every_smaller_batch(lib, hidden):
    def sizes(fn, rows):
        need = C.c_size_t()
        for t in rows:
            assert getattr(lib, fn)(t, hidden, C.byref(need)) == 0
            yield need.value

    rows = list(range(0, 1400)) + [4096, 5000, 16384, 100000, 1 << 24]
    for fn in ("mi_moe_add_rms_norm_grad_workspace_size", "mi_moe_quantized_linear_rows8_workspace_size"):
        got = list(sizes(fn, rows))
        assert got == sorted(got), fn

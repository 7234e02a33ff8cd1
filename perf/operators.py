"""Operators around the experts of a decoder layer, as a list of cases and a generator of more of the same ranges.

``norm``         the residual's addition and the RMS norm behind it in one pass (``ops.add_rms_norm``): what stands between
                 two sublayers.
``norm_grad``    its backward pass (``ops.add_rms_norm_grad``): gradients of the two summands and of the weight.
``select``       experts of every token from the router's logits (``ops.select_experts``): softmax or sigmoid scores, a bias
                 that balances the load, groups of experts, top-k, renormalised weights.
``select_grad``  the gradient of those weights with respect to the logits (``ops.select_experts_grad``).
``linear8``      a quantized linear layer on rows in 8 bits (``ops.quantized_linear_rows8``).
``norm_linear8`` the norm with its rows in 8 bits and scales (``ops.add_rms_norm_rows8``), and the layer that reads them.

The plain forms are elementary torch operations.
"""
import math

import torch

own = False  # True: the package's operators in place of the plain forms

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}
EPS = 1e-6


def _norm(name, rows, hidden, dtype):
    return {"name": name, "kind": "norm", "rows": rows, "hidden": hidden, "dtype": dtype}


def _norm_grad(name, rows, hidden, dtype, through=True):
    return {"name": name, "kind": "norm_grad", "rows": rows, "hidden": hidden, "dtype": dtype, "through": through}


def _select(name, kind, rows, experts, top_k, scoring, dtype, bias=False, groups=1, top_groups=1, group_score="max",
            renormalize=True, scale=1.0, weights="bfloat16"):
    return {"name": name, "kind": kind, "rows": rows, "experts": experts, "top_k": top_k, "scoring": scoring, "dtype": dtype,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": group_score, "renormalize": renormalize,
            "scale": scale, "weights": weights}


def _linear8(name, kind, rows, n, k, bits, group, dtype, bias=False):
    return {"name": name, "kind": kind, "rows": rows, "n": n, "k": k, "bits": bits, "group": group, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one user's next token between two sublayers: the latency of a launch
        _norm("norm 1", 1, 2048, "bfloat16"),
        # a long prompt
        _norm("norm 8192", 8192, 4096, "bfloat16"),
        # fine-tuning: rows that fill no whole vector, no gradient past the norm
        _norm_grad("norm gradient 1000 odd", 1000, 2045, "float16", through=False),
        # a training batch, with the gradient that arrives along the residual
        _norm_grad("norm gradient 4096", 4096, 4096, "bfloat16"),
        # a serving batch's routing
        _select("select 32", "select", 32, 128, 8, "softmax", "bfloat16"),
        # a prompt's routing over many experts: sigmoid scores, a bias for balance, half of the groups
        _select("select 8192 groups", "select", 8192, 256, 8, "sigmoid", "float32", True, 8, 4, "top2", True, 2.5, "float32"),
        # training: weights that are not renormalised reach every logit
        _select("select gradient 203", "select_grad", 203, 128, 8, "softmax", "bfloat16", renormalize=False, weights="float32"),
        _select("select gradient 8192", "select_grad", 8192, 256, 8, "sigmoid", "float32", True, 8, 4, "top2", True, 2.5, "float32"),
        # the projections of one token, and of a prompt
        _linear8("norm and linear 1", "norm_linear8", 1, 4096, 2048, 4, 64, "bfloat16"),
        _linear8("norm and linear 4096", "norm_linear8", 4096, 4096, 4096, 4, 64, "bfloat16"),
        # a projection with a bias over a ragged prompt, in half precision
        _linear8("linear f16 777", "linear8", 777, 4096, 4096, 8, 64, "float16", True),
        # the widest layer: few groups, many columns
        _linear8("linear 2048 wide", "linear8", 2048, 14336, 4096, 4, 128, "bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "select", "select_grad", "linear8", "linear8", "norm_linear8"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("norm", "norm_grad"):
        hidden = _log_int(rng, 128, 8192)
        if rng.random() < 0.7:
            hidden = (hidden + 7) // 8 * 8
        most = (8192 if kind == "norm" else 4096) * 4096 // hidden // (2 if dtype == "float32" else 1)
        rows = _log_int(rng, 1, min(16384, most))
        case = _norm("", rows, hidden, dtype) if kind == "norm" else _norm_grad("", rows, hidden, dtype, rng.random() < 0.6)
    elif kind in ("select", "select_grad"):
        groups = rng.choice([1, 1, 2, 4, 8, 8, 16])
        experts = groups * rng.randint(max(2, 8 // groups), 256 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, experts // groups * top_groups))
        case = _select("", kind, _log_int(rng, 1, 8192), experts, top_k, rng.choice(["softmax", "sigmoid"]), dtype, rng.random() < 0.5,
                       groups, top_groups, rng.choice(["max", "top2"]), rng.random() < 0.6, rng.choice([1.0, 2.5]),
                       rng.choice(["bfloat16", "float32"]) if kind == "select" else "float32")
    else:
        k = 128 * rng.randint(4, 32)
        n = 16 * rng.randint(16, 896) - (rng.randint(1, 15) if rng.random() < 0.3 else 0)
        rows = _log_int(rng, 1, 2048 if n > 4096 else 4096)
        case = _linear8("", kind, rows, n, k, rng.choice([4, 4, 8]), rng.choice([64, 64, 32, 128]), dtype, rng.random() < 0.3)
    case.pop("name", None)
    return case


# ---------------------------------------------------------------- inputs
def _pack(codes, bits):
    """Codes [N, K] to words [N, K * bits / 32], low bits first."""
    per = 32 // bits
    shifts = torch.arange(per, device=codes.device, dtype=torch.int64) * bits
    words = (codes.to(torch.int64).reshape(codes.shape[0], -1, per) << shifts).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows = case["rows"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std

    state = {"case": case}
    if case["kind"] in ("norm", "norm_grad", "norm_linear8"):
        hidden = case["hidden"] if "hidden" in case else case["k"]
        state["weight"] = (1.0 + normal(hidden, std=0.1)).to(dtype)
        if case["kind"] == "norm_grad":
            state["h"], state["dy"] = normal(rows, hidden, std=1.5).to(dtype), normal(rows, hidden).to(dtype)
            state["dh"] = normal(rows, hidden).to(dtype) if case["through"] else None
        else:
            state["x"], state["residual"] = normal(rows, hidden).to(dtype), normal(rows, hidden, std=1.5).to(dtype)
    if case["kind"] in ("select", "select_grad"):
        state["logits"] = normal(rows, case["experts"], std=1.3).to(dtype)
        state["bias"] = normal(case["experts"], std=0.05) if case["bias"] else None
        if case["kind"] == "select_grad":
            state["inds"] = _select_plain(state["logits"], state["bias"], case)[0]
            state["dweights"] = normal(rows, case["top_k"])
    if case["kind"] in ("linear8", "norm_linear8"):
        n, k, bits, group = case["n"], case["k"], case["bits"], case["group"]
        most = 2 ** bits - 1
        state["q"] = _pack((normal(n, k, std=most / 4.6) + most / 2).round().clamp(0, most), bits)
        scales = 0.092 / most * (1.0 + normal(n, k // group, std=0.1).clamp(-0.5, 0.5))
        state["s"], state["b"] = scales.to(dtype), (-scales * most / 2 + normal(n, k // group, std=0.002)).to(dtype)
        state["linear_bias"] = normal(n, std=0.5).to(dtype) if case["bias"] else None
        if case["kind"] == "linear8":
            state["x8"] = normal(rows, k, std=127 / 3.8).round().clamp(-127, 127).to(torch.int8)
            state["x_scales"] = 0.03 * (1.0 + 0.2 * normal(rows).clamp(-3, 3))
    return state


# ---------------------------------------------------------------- plain forms
def _add_plain(x, residual):
    return (x.float() + residual.float()).to(x.dtype)


def _norm_plain(h, weight):
    h = h.float()
    return weight.float() * (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS))


def _norm_grad_plain(dy, h, weight, dh):
    dy32, h32 = dy.float(), h.float()
    rstd = torch.rsqrt(h32.square().mean(-1, keepdim=True) + EPS)
    hat = h32 * rstd
    wdy = weight.float() * dy32
    dx = rstd * (wdy - hat * (wdy * hat).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.float()
    return dx.to(h.dtype), (dy32 * hat).sum(0).to(weight.dtype)


def _scores(logits, scoring):
    wide = logits.double()
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-wide))
    e = torch.exp(wide - wide.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _select_plain(logits, bias, case):
    """Scores and keys in 64 bits: what lies next to a border has to fall on its side of it."""
    s = _scores(logits, case["scoring"])
    biased = s if bias is None else s + bias.double()
    key = logits.double() if bias is None else biased  # (without a bias the logits' own order, which the scores' is where they differ)
    groups = case["groups"]
    if groups > 1:
        by_group = key.reshape(key.shape[0], groups, -1)
        if case["group_score"] == "max":
            rank = by_group.amax(-1)
        else:
            rank = torch.sort(biased.reshape(by_group.shape), dim=-1, descending=True)[0][..., :2].sum(-1)
        order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, :case["top_groups"]]
        open_ = torch.zeros_like(rank, dtype=torch.bool).scatter(1, order, True)
        key = torch.where(open_[..., None], by_group, torch.full_like(by_group, -math.inf)).reshape(key.shape)
    inds = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :case["top_k"]]
    w = s.gather(1, inds)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return inds.to(torch.int32), (w * case["scale"]).to(DTYPES[case["weights"]])


def _select_grad_plain(dweights, logits, inds, case):
    x, at = logits.float(), inds.long()
    if case["scoring"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    picked, g = s.gather(1, at), dweights.float() * case["scale"]
    if case["renormalize"]:
        share = picked / picked.sum(-1, keepdim=True)
        inner = share * (g - (share * g).sum(-1, keepdim=True))  # s times the gradient with respect to s
    else:
        inner = picked * g
    if case["scoring"] == "sigmoid":
        out = torch.zeros_like(x).scatter(1, at, inner * (1.0 - picked))
    elif case["renormalize"]:
        out = torch.zeros_like(x).scatter(1, at, inner)
    else:
        out = torch.zeros_like(x).scatter(1, at, inner) - s * inner.sum(-1, keepdim=True)
    return out.to(logits.dtype)


def _rows8_plain(h, weight):
    """The normalised rows in steps of a 127th of their largest value.  A row's own factor has no part in the codes; they are
    in 64 bits, where the products are exact, so that what lies halfway between two codes is seen to."""
    p = h.double() * weight.double()
    largest = p.abs().amax(-1, keepdim=True)
    codes = torch.where(largest > 0, (127.0 * p / largest).round(), torch.zeros_like(p))
    rstd = torch.rsqrt(h.double().square().mean(-1, keepdim=True) + EPS)
    return codes, (largest * rstd / 127.0).float()


def _dense(state, wide):
    """The layer's weights: scale * code + bias of every group."""
    case = state["case"]
    n, k, bits, group = case["n"], case["k"], case["bits"], case["group"]
    shifts = torch.arange(32 // bits, device="cuda", dtype=torch.int32) * bits
    codes = (state["q"][..., None] >> shifts & (2 ** bits - 1)).to(wide).reshape(n, k // group, group)
    return (state["s"].to(wide)[..., None] * codes + state["b"].to(wide)[..., None]).reshape(n, k)


def _linear8_plain(x8, x_scales, state):
    y = torch.matmul(x8.float(), _dense(state, torch.float32).t()) * x_scales.reshape(-1, 1)
    if state["linear_bias"] is not None:
        y = y + state["linear_bias"].float()
    return y.to(state["s"].dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        h = _add_plain(state["x"], state["residual"])
        return _norm_plain(h, state["weight"]).to(h.dtype), h
    if kind == "norm_grad":
        return _norm_grad_plain(state["dy"], state["h"], state["weight"], state["dh"])
    if kind == "select":
        return _select_plain(state["logits"], state["bias"], case)
    if kind == "select_grad":
        return _select_grad_plain(state["dweights"], state["logits"], state["inds"], case)
    if kind == "linear8":
        return _linear8_plain(state["x8"], state["x_scales"], state)
    h = _add_plain(state["x"], state["residual"])
    x8, scales = _rows8_plain(h, state["weight"])
    return _linear8_plain(x8, scales, state), h


def run(state):
    if not own:
        return _plain(state)
    from mlx_rs_amd import ops
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        return ops.add_rms_norm(state["x"], state["residual"], state["weight"], EPS)
    if kind == "norm_grad":
        return ops.add_rms_norm_grad(state["dy"], state["h"], state["weight"], EPS, state["dh"])
    if kind == "select":
        return ops.select_experts(state["logits"], case["top_k"], case["scoring"], state["bias"], case["groups"], case["top_groups"],
                                  case["group_score"], case["renormalize"], case["scale"], DTYPES[case["weights"]])
    if kind == "select_grad":
        return ops.select_experts_grad(state["dweights"], state["logits"], state["inds"], case["scoring"], case["renormalize"],
                                       case["scale"])
    if kind == "linear8":
        return ops.quantized_linear_rows8(state["x8"], state["x_scales"], state["q"], state["s"], state["b"], state["linear_bias"],
                                          case["group"], case["bits"])
    x8, scales, h = ops.add_rms_norm_rows8(state["x"], state["residual"], state["weight"], EPS)
    return ops.quantized_linear_rows8(x8, scales, state["q"], state["s"], state["b"], state["linear_bias"], case["group"], case["bits"]), h


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_norm(h, weight):
    wide = h.double()
    rms = (wide.pow(2).sum(-1, keepdim=True) / wide.shape[-1] + EPS).sqrt()
    return wide / rms * weight.double()


def _exact_picks(logits, bias, case):
    wide = logits.double()
    s = torch.sigmoid(wide) if case["scoring"] == "sigmoid" else torch.softmax(wide, -1)
    rows, experts = wide.shape
    key = wide if bias is None else s + bias.double()
    open_ = torch.ones_like(key, dtype=torch.bool)
    if case["groups"] > 1:
        of = (key if case["group_score"] == "max" else s if bias is None else key).reshape(rows, case["groups"], -1)
        if case["group_score"] == "max":
            score = of.max(-1).values
        else:
            score = of.topk(2, -1).values.sum(-1) if of.shape[-1] > 1 else of[..., 0]
        # a group is open where fewer than top_groups groups stand before it: a larger score, or the same and a lower number
        number = torch.arange(case["groups"], device="cuda")
        first = (score[:, None, :] > score[:, :, None]) | ((score[:, None, :] == score[:, :, None]) & (number[None, :] < number[:, None]))
        open_ = (first.sum(-1) < case["top_groups"]).repeat_interleave(experts // case["groups"], 1)
    inds = torch.argsort(torch.where(open_, -key, math.inf), dim=-1, stable=True)[:, :case["top_k"]]
    return s, inds


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        total = state["x"].double() + state["residual"].double()
        return _exact_norm(total.to(state["x"].dtype), state["weight"]), total
    if kind == "norm_grad":
        h, dy, w = state["h"].double(), state["dy"].double(), state["weight"].double()
        var = h.pow(2).mean(-1, keepdim=True) + EPS
        dot = (w * dy * h).sum(-1, keepdim=True)
        dx = w * dy / var.sqrt() - h * dot / (h.shape[-1] * var.pow(1.5))
        return dx if state["dh"] is None else dx + state["dh"].double(), (dy * h / var.sqrt()).sum(0)
    if kind == "select":
        s, inds = _exact_picks(state["logits"], state["bias"], case)
        w = torch.take_along_dim(s, inds, -1)
        if case["renormalize"]:
            w = w / w.sum(-1, keepdim=True)
        return inds.to(torch.int32), case["scale"] * w
    if kind == "select_grad":
        wide = state["logits"].double()
        s = torch.sigmoid(wide) if case["scoring"] == "sigmoid" else torch.softmax(wide, -1)
        at = state["inds"].long()
        w, g = torch.take_along_dim(s, at, -1), case["scale"] * state["dweights"].double()
        if case["renormalize"]:
            total = w.sum(-1, keepdim=True)
            g = g / total - (g * w).sum(-1, keepdim=True) / total.square()
        ds = torch.zeros_like(s).scatter_(1, at, g)  # with respect to the scores
        return ds * s * (1 - s) if case["scoring"] == "sigmoid" else s * (ds - (ds * s).sum(-1, keepdim=True))
    if kind == "linear8":
        x8, scales, total = state["x8"].double(), state["x_scales"].double()[:, None], None
    else:
        total = state["x"].double() + state["residual"].double()
        h = total.to(state["x"].dtype)
        scales = _exact_norm(h, state["weight"]).abs().amax(-1, keepdim=True) / 127
        z = h.double() * state["weight"].double()  # (the norm but for the row's factor)
        x8 = torch.round(z * 127 / z.abs().amax(-1, keepdim=True))
    y = torch.matmul(x8, _dense(state, torch.float64).t()) * scales
    if state["linear_bias"] is not None:
        y = y + state["linear_bias"].double()
    return y if total is None else (y, total)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, size, kind = case["rows"], SIZES[case["dtype"]], case["kind"]
    if kind == "norm":
        return {"bytes": size * case["hidden"] * (4 * rows + 1), "flops": 6 * rows * case["hidden"]}
    if kind == "norm_grad":
        return {"bytes": size * case["hidden"] * ((4 if case["through"] else 3) * rows + 2), "flops": 13 * rows * case["hidden"]}
    if kind == "select":
        out = (4 + SIZES[case["weights"]]) * case["top_k"]
        return {"bytes": rows * (size * case["experts"] + out) + (4 * case["experts"] if case["bias"] else 0), "flops": 4 * rows * case["experts"]}
    if kind == "select_grad":
        # renormalised weights and sigmoid scores go by the chosen experts' logits alone
        read = case["experts"] if case["scoring"] == "softmax" and not case["renormalize"] else case["top_k"]
        return {"bytes": rows * (size * (read + case["experts"]) + 8 * case["top_k"]), "flops": 4 * rows * read}
    n, k = case["n"], case["k"]
    weights = n * k * case["bits"] // 8 + 2 * size * n * k // case["group"]
    out = size * (rows * n + (n if case["bias"] else 0))
    if kind == "linear8":
        return {"bytes": weights + out + rows * (k + 4), "flops": 2 * rows * n * k}
    return {"bytes": weights + out + size * k * (3 * rows + 1), "flops": 2 * rows * n * k}

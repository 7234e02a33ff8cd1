"""Operators of experts whose weights are 8-bit floating point, as a list of cases and a generator of more of the same ranges.

``sort``          tokens to rows sorted by expert (``ops.sort_tokens``): the rows, the order of the (token, slot) pairs, every slot's row, and where
                  every expert's rows begin.
``sort_grad``     its gradient (``ops.sort_tokens_grad``): a token's gradient is the sum over its rows.
``unsort``        rows back to tokens, weighted (``ops.unsort_tokens``).
``unsort_grad``   its gradients with respect to the rows and the weights (``ops.unsort_tokens_grad``).
``linear``        a linear layer on e4m3 weights with a scale for each block of 128 x 128 (``ops.linear_f8``): rows are rounded to e4m3 with a scale for
                  each run of 128 values on the way in.
``linear_grad``   the gradient with respect to its input, in the same way (``ops.linear_f8`` with ``transpose=False``).
``grouped``, ``grouped_grad``  the same for rows sorted by expert, a matrix for every expert (``ops.grouped_linear_f8``).
``experts``       SwiGLU experts on such weights, from tokens to tokens (``ops.switch_glu_f8``).
``experts_grad``  their gradients with respect to the tokens and to the routing weights (``ops.switch_glu_f8_grad``); roundings to e4m3 pass a gradient
                  on as it is.

The plain forms are elementary torch operations.
"""
import math

import torch

own = False  # True: the package's operators in place of the plain forms

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}
F8 = torch.float8_e4m3fn
F8_MOST = 448.0  # the type's largest value
BLOCK = 128


def _tokens(name, kind, rows, hidden, experts, top_k, dtype, padded=False, weights="bfloat16"):
    return {"name": name, "kind": kind, "rows": rows, "hidden": hidden, "experts": experts, "top_k": top_k, "dtype": dtype, "padded": padded,
            "weights": weights}


def _linear(name, kind, rows, n, k, dtype, bias=False):
    return {"name": name, "kind": kind, "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _grouped(name, kind, rows, experts, n, k, dtype):
    return {"name": name, "kind": kind, "rows": rows, "experts": experts, "n": n, "k": k, "dtype": dtype}


def _experts(name, kind, rows, hidden, intermediate, experts, top_k, dtype, padded=False, weights="bfloat16"):
    return {"name": name, "kind": kind, "rows": rows, "hidden": hidden, "intermediate": intermediate, "experts": experts, "top_k": top_k, "dtype": dtype,
            "padded": padded, "weights": weights}


def listed():
    return [
        # a serving batch's tokens, some of the batch padding: the latency of a launch or two
        _tokens("sort 32 padded", "sort", 32, 2048, 128, 8, "bfloat16", padded=True),
        # training: a long batch's gradient back at its tokens
        _tokens("sort gradient 8192", "sort_grad", 8192, 2048, 128, 8, "bfloat16"),
        # a prompt's rows back at their tokens
        _tokens("unsort 4096", "unsort", 4096, 2048, 128, 8, "bfloat16"),
        # fine-tuning in half precision, a ragged padded batch of rows that fill no whole vector
        _tokens("unsort gradient 1000 odd", "unsort_grad", 1000, 2045, 64, 6, "float16", padded=True, weights="float32"),
        # a projection of one token
        _linear("linear 1", "linear", 1, 4096, 2048, "bfloat16"),
        # the same of a prompt
        _linear("linear 4096", "linear", 4096, 4096, 4096, "bfloat16"),
        # fine-tuning on frozen weights: a ragged batch's gradient with respect to the input
        _linear("linear gradient 1000", "linear_grad", 1000, 4096, 4096, "float16"),
        # a decode batch's rows at their experts, two or three rows each
        _grouped("grouped 300", "grouped", 300, 128, 768, 2048, "bfloat16"),
        # a training batch's gradient through a bank of matrices
        _grouped("grouped gradient 16384", "grouped_grad", 16384, 64, 2048, 1408, "bfloat16"),
        # one user's next token through its experts
        _experts("experts 1", "experts", 1, 2048, 768, 128, 8, "bfloat16"),
        # a prompt through its experts: the largest call
        _experts("experts 4096", "experts", 4096, 2048, 768, 128, 8, "bfloat16"),
        # fine-tuning: the way back, a few wide experts
        _experts("experts gradient 1000", "experts_grad", 1000, 2048, 1792, 16, 2, "bfloat16", weights="float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo, hi):
    """A layer's extent: often whole blocks of 128, else a multiple of 16."""
    step = BLOCK if rng.random() < 0.6 else 16
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(["sort", "sort_grad", "unsort", "unsort_grad", "linear", "linear", "linear_grad", "grouped", "grouped_grad", "experts", "experts",
                       "experts_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("sort", "sort_grad", "unsort", "unsort_grad"):
        hidden = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            hidden = (hidden + 7) // 8 * 8
        experts = _log_int(rng, 2, 256)
        top_k = rng.randint(1, min(8, experts))
        rows = _log_int(rng, 1, min(8192, 134217728 // (hidden * top_k) * 2 // SIZES[dtype]))
        case = _tokens("", kind, rows, hidden, experts, top_k, dtype, rng.random() < 0.4, rng.choice(["bfloat16", "float32"]))
    elif kind in ("linear", "linear_grad"):
        n = _width(rng, 256, 8192) - (rng.randint(1, 15) if kind == "linear" and rng.random() < 0.3 else 0)
        k = _width(rng, 256, 8192)
        case = _linear("", kind, _log_int(rng, 1, min(8192, 68719476736 // (n * k))), n, k, dtype, kind == "linear" and rng.random() < 0.4)
    elif kind in ("grouped", "grouped_grad"):
        n, k = _width(rng, 256, 4096), _width(rng, 256, 4096)
        experts = _log_int(rng, 1, min(256, 300000000 // (n * k)))
        case = _grouped("", kind, _log_int(rng, 1, min(32768, 50000000000 // (n * k))), experts, n, k, dtype)
    else:
        dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
        hidden, intermediate = _width(rng, 256, 4096), _width(rng, 128, 4096)
        experts = _log_int(rng, 2, min(256, 200000000 // (hidden * intermediate)))
        top_k = rng.randint(1, min(8, experts))
        pairs = (50000000000 if kind == "experts" else 16000000000) // (hidden * intermediate)
        case = _experts("", kind, _log_int(rng, 1, min(4096, pairs // top_k)), hidden, intermediate, experts, top_k, dtype, rng.random() < 0.3,
                        rng.choice(["bfloat16", "float32"]))
    case.pop("name", None)
    return case


# ---------------------------------------------------------------- inputs
def _blocks(n):
    return -(-n // BLOCK)


def _bank(normal, n, k, experts=None, spread=1.0):
    """Matrices [experts, n, k] as a checkpoint holds them: codes over the type's range and a scale a block, so that a row's weights have about the
    length `spread`."""
    lead = () if experts is None else (experts,)
    codes = torch.empty(lead + (n, k), dtype=F8, device="cuda")
    for part in [codes] if experts is None else codes:  # (a bank's float32 values would be four times the bank)
        part.copy_((normal(n, k) * (F8_MOST / 4.5)).clamp(-F8_MOST, F8_MOST))
    scales = spread * 4.5 / F8_MOST / math.sqrt(k) * (1.0 + 0.2 * normal(*lead, _blocks(n), _blocks(k)).clamp(-3, 3))
    return codes, scales.contiguous()


def _routing(gen, case):
    """Different experts for the slots of a token, some experts more popular than others; in a padded batch some tokens and slots name none."""
    rows, experts, top_k = case["rows"], case["experts"], case["top_k"]
    liked = 0.7 * torch.randn(experts, generator=gen, device="cuda")
    score = liked + torch.randn((rows, experts), generator=gen, device="cuda")
    inds = torch.sort(score, dim=-1, descending=True)[1][:, :top_k].to(torch.int32)
    if case["padded"]:
        u = torch.rand((rows, 1), generator=gen, device="cuda")
        v = torch.rand((rows, top_k), generator=gen, device="cuda")
        inds = torch.where(u < 0.1, torch.full_like(inds, experts), torch.where(v < 0.05, torch.full_like(inds, -1), inds))
    w = torch.rand((rows, top_k), generator=gen, device="cuda") + 0.1
    return inds.contiguous(), (w / w.sum(-1, keepdim=True)).to(DTYPES[case["weights"]])


def _plan(offsets, pairs):
    """What the plain form goes by: the experts that have rows, and their rows' numbers, filled up with `pairs` to the most that one has."""
    counts = (offsets[1:] - offsets[:-1]).long()
    active = counts.nonzero()[:, 0]
    step = torch.arange(int(counts.max()), device=counts.device)
    at = torch.where(step < counts[active, None], offsets[active, None].long() + step, pairs)
    return active, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, rows = DTYPES[case["dtype"]], case["kind"], case["rows"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    state = {"case": case}
    if kind in ("sort", "sort_grad", "unsort", "unsort_grad"):
        hidden, pairs = case["hidden"], rows * case["top_k"]
        state["inds"], state["weights"] = _routing(gen, case)
        if kind == "sort":
            state["x"] = normal(rows, hidden).to(dtype)
        else:
            state["inverse"] = _order_plain(state["inds"], case["experts"])[1]
            if kind != "unsort_grad":
                state["sorted"] = normal(pairs, hidden).to(dtype)
            else:
                state["sorted"], state["dout"] = normal(pairs, hidden).to(dtype), normal(rows, hidden).to(dtype)
    elif kind in ("linear", "linear_grad"):
        n, k = case["n"], case["k"]
        state["w"], state["s"] = _bank(normal, n, k)
        state["x"] = normal(rows, k if kind == "linear" else n).to(dtype)
        state["bias"] = (0.5 * normal(n)).to(dtype) if case["bias"] else None
    elif kind in ("grouped", "grouped_grad"):
        n, k, experts = case["n"], case["k"], case["experts"]
        state["w"], state["s"] = _bank(normal, n, k, experts)
        state["x"] = normal(rows, k if kind == "grouped" else n).to(dtype)
        pick = torch.randint(0, experts, (rows,), generator=gen, device="cuda")
        counts = (pick[None] == torch.arange(experts, device="cuda")[:, None]).sum(-1)
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        state["plan"] = _plan(state["offsets"], rows)
    else:
        hidden, inter, experts = case["hidden"], case["intermediate"], case["experts"]
        state["x"] = normal(rows, hidden).to(dtype)
        state["inds"], state["weights"] = _routing(gen, case)
        state["gate"] = _bank(normal, inter, hidden, experts)
        state["up"] = _bank(normal, inter, hidden, experts)
        state["down"] = _bank(normal, hidden, inter, experts)
        state["plan"] = _plan(_order_plain(state["inds"], experts)[2], state["inds"].numel())
        if kind == "experts_grad":
            state["dout"] = normal(rows, hidden).to(dtype)
    return state


# ---------------------------------------------------------------- plain forms
def _order_plain(inds, experts):
    """The pairs sorted by expert, those that name none last; every slot's row (-1 - row where it names none); where every expert's rows begin."""
    flat = inds.reshape(-1).long()
    named = (flat >= 0) & (flat < experts)
    flat = torch.where(named, flat, torch.full_like(flat, experts))
    order = torch.sort(flat, stable=True)[1]
    place = torch.zeros_like(order).scatter(0, order, torch.arange(order.numel(), device=order.device))
    inverse = torch.where(named, place, -1 - place).reshape(inds.shape)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=order.device).scatter_add(0, flat, torch.ones_like(flat))[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return order.to(torch.int32), inverse.to(torch.int32), offsets.to(torch.int32)


def _sort_plain(x, inds, experts):
    order, inverse, offsets = _order_plain(inds, experts)
    rows = x[order.long() // inds.shape[1]]
    named = torch.arange(rows.shape[0], device=x.device) < offsets[-1]
    return torch.where(named[:, None], rows, torch.zeros_like(rows)), order, inverse, offsets


def _sort_grad_plain(drows, inverse):
    at = inverse.long()
    picked = drows.float()[at.clamp(min=0)]
    return torch.where((at >= 0)[..., None], picked, torch.zeros_like(picked)).sum(1).to(drows.dtype)


def _unsort_plain(rows, weights, inverse):
    at = inverse.long()
    picked = rows.float()[at.clamp(min=0)] * weights.float()[..., None]
    return torch.where((at >= 0)[..., None], picked, torch.zeros_like(picked)).sum(1).to(rows.dtype)


def _unsort_grad_plain(dout, rows, weights, inverse):
    at = inverse.long()
    named = (at >= 0)[..., None]
    g = dout.float()[:, None, :]
    part = torch.where(named, g * weights.float()[..., None], torch.zeros_like(g))
    drows = torch.zeros(rows.shape, dtype=torch.float32, device=rows.device)
    drows[torch.where(at >= 0, at, -1 - at).reshape(-1)] = part.reshape(-1, rows.shape[1])
    picked = rows.float()[at.clamp(min=0)]
    dweights = torch.where(named, g * picked, torch.zeros_like(picked)).sum(-1)
    return drows.to(rows.dtype), dweights.to(weights.dtype)


def _e4m3_plain(x):
    """Rows in e4m3 with a scale for each run of 128 values: the values that they stand for, in 32 bits.  The scale is the run's largest value over
    448, a code is the e4m3 value nearest to the quotient of value and scale, both rounded to float32 (by way of 64 bits: values of 16 bits often lie
    halfway between two codes, where a division that is off in its last bit goes to the other one)."""
    rows, cols = x.shape
    runs = torch.zeros(rows, _blocks(cols) * BLOCK, device=x.device)
    runs[:, :cols] = x.float()
    runs = runs.reshape(rows, _blocks(cols), BLOCK)
    scale = (runs.abs().amax(-1, keepdim=True).double() / F8_MOST).float()
    codes = torch.where(scale > 0, (runs.double() / scale.double()).float(), torch.zeros_like(runs)).clamp(-F8_MOST, F8_MOST).to(F8)
    return (codes.float() * scale).reshape(rows, _blocks(cols) * BLOCK)[:, :cols]


def _dense_plain(codes, scales):
    spread = scales.repeat_interleave(BLOCK, -2)[..., :codes.shape[-2], :].repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]
    return codes.float() * spread


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _padded(rows, at):
    """Rows by number; the number behind the last is a row of zeros."""
    return torch.cat([rows, rows.new_zeros((1,) + rows.shape[1:])])[at]


def _back(parts, at, count):
    """Padded rows where they came from; rows that none came from are zeros."""
    out = torch.zeros((count + 1,) + parts.shape[2:], device=parts.device)
    out[at.reshape(-1)] = parts.reshape((-1,) + parts.shape[2:])
    return out[:count]


def _times(rows, dense, transpose):
    return torch.bmm(rows, dense.transpose(1, 2).contiguous() if transpose else dense)


def _grouped_plain(x, w, s, plan, transpose):
    active, at = plan
    y = _times(_padded(_e4m3_plain(x), at), _dense_plain(w[active], s[active]), transpose)
    return _back(y, at, x.shape[0]).to(x.dtype)


def _experts_plain(state):
    case, (active, at) = state["case"], state["plan"]
    order, inverse, _ = _order_plain(state["inds"], case["experts"])
    token = torch.cat([order.long() // case["top_k"], order.new_full((1,), case["rows"])])[at]
    gate, up, down = (_dense_plain(codes[active], scales[active]) for codes, scales in (state["gate"], state["up"], state["down"]))
    rows = _padded(_e4m3_plain(state["x"]), token)
    g, u = _times(rows, gate, True), _times(rows, up, True)
    if case["kind"] == "experts":
        h = _e4m3_plain((_silu(g) * u).reshape(-1, g.shape[2])).reshape(g.shape)
        return _unsort_plain(_back(_times(h, down, True), at, order.numel()), state["weights"], inverse).to(state["x"].dtype)
    dh = _times(_padded(_e4m3_plain(state["dout"]), token), down, False)  # (but for the slot's weight)
    dweights = _back((dh * (_silu(g) * u)).sum(-1), at, order.numel())
    dh = dh * _padded(state["weights"].float().reshape(-1)[order.long()], at)[..., None]
    sigma = 1.0 / (1.0 + torch.exp(-g))
    dg, du = (_e4m3_plain(d.reshape(-1, d.shape[2])).reshape(d.shape) for d in (dh * u * sigma * (1.0 + g * (1.0 - sigma)), dh * g * sigma))
    dx = _sort_grad_plain(_back(_times(dg, gate, False) + _times(du, up, False), at, order.numel()), inverse)
    dweights = torch.zeros_like(dweights).scatter(0, order.long(), dweights).reshape(inverse.shape)
    return dx.to(state["x"].dtype), dweights.to(state["weights"].dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "sort":
        return _sort_plain(state["x"], state["inds"], case["experts"])
    if kind == "sort_grad":
        return _sort_grad_plain(state["sorted"], state["inverse"])
    if kind == "unsort":
        return _unsort_plain(state["sorted"], state["weights"], state["inverse"])
    if kind == "unsort_grad":
        return _unsort_grad_plain(state["dout"], state["sorted"], state["weights"], state["inverse"])
    if kind in ("linear", "linear_grad"):
        dense = _dense_plain(state["w"], state["s"])
        y = torch.matmul(_e4m3_plain(state["x"]), dense.t() if kind == "linear" else dense)
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(state["x"].dtype)
    if kind in ("grouped", "grouped_grad"):
        return _grouped_plain(state["x"], state["w"], state["s"], state["plan"], kind == "grouped")
    return _experts_plain(state)


def run(state):
    if not own:
        return _plain(state)
    from mlx_rs_amd import ops
    case = state["case"]
    kind = case["kind"]
    if kind == "sort":
        return ops.sort_tokens(state["x"], state["inds"], case["experts"])
    if kind == "sort_grad":
        return ops.sort_tokens_grad(state["sorted"], state["inverse"])
    if kind == "unsort":
        return ops.unsort_tokens(state["sorted"], state["weights"], state["inverse"])
    if kind == "unsort_grad":
        return ops.unsort_tokens_grad(state["dout"], state["sorted"], state["weights"], state["inverse"])
    if kind in ("linear", "linear_grad"):
        return ops.linear_f8(state["x"], state["w"], state["s"], state["bias"], transpose=kind == "linear")
    if kind in ("grouped", "grouped_grad"):
        return ops.grouped_linear_f8(state["x"], state["w"], state["s"], state["offsets"], transpose=kind == "grouped")
    if kind == "experts":
        return ops.switch_glu_f8(state["x"], state["inds"], state["weights"], state["gate"], state["up"], state["down"])
    return ops.switch_glu_f8_grad(state["dout"], state["x"], state["inds"], state["weights"], state["gate"], state["up"], state["down"])


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_e4m3(x):
    """e4m3's grid: four significant bits down to 2^-6, steps of 2^-9 below.  Scales and quotients are float32 numbers by definition."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], BLOCK):
        run = x[:, c:c + BLOCK].double()
        scale = (run.abs().max(-1, keepdim=True).values / F8_MOST).float().double()
        q = torch.nan_to_num((run / scale).float().double(), nan=0.0)
        step = torch.exp2(torch.frexp(q)[1].double().sub(1).clamp(min=-6) - 3)
        out[:, c:c + BLOCK] = torch.clamp(torch.round(q / step) * step, -F8_MOST, F8_MOST) * scale
    return out


def _exact_matrix(codes, scales):
    out = codes.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            out[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j].double()
    return out


def _exact_rows(x, codes, scales, transpose):
    """x . W^T or x . W by runs of the summed axis, so that a bank's matrix is not spread out block by block."""
    out = torch.zeros(x.shape[0], codes.shape[0] if transpose else codes.shape[1], dtype=torch.float64, device=x.device)
    w = codes.double() if transpose else codes.double().t()
    s = scales.double() if transpose else scales.double().t()
    for j in range(s.shape[1]):
        each = s[:, j].repeat_interleave(BLOCK)[:w.shape[0]]
        out += torch.matmul(x[:, j * BLOCK:(j + 1) * BLOCK], w[:, j * BLOCK:(j + 1) * BLOCK].t()) * each
    return out


def _exact_slots(rows, inverse):
    at = inverse.long()
    return rows.double()[at.clamp(min=0)] * (at >= 0)[..., None]


def _exact_sorted(state):
    case = state["case"]
    flat = state["inds"].reshape(-1)
    named = (flat >= 0) & (flat < case["experts"])
    key = torch.where(named, flat, case["experts"])
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(case["experts"] + 1, device=key.device, dtype=key.dtype))
    return order, torch.where(named, place, -1 - place).reshape(state["inds"].shape), offsets


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "sort":
        order, inverse, offsets = _exact_sorted(state)
        rows = state["x"].double()[torch.div(order, case["top_k"], rounding_mode="floor")]
        rows[int(offsets[-1]):] = 0
        return rows, order.to(torch.int32), inverse.to(torch.int32), offsets.to(torch.int32)
    if kind == "sort_grad":
        return _exact_slots(state["sorted"], state["inverse"]).sum(1)
    if kind == "unsort":
        return (_exact_slots(state["sorted"], state["inverse"]) * state["weights"].double()[..., None]).sum(1)
    if kind == "unsort_grad":
        at, g = state["inverse"].long(), state["dout"].double()
        drows = torch.zeros(state["sorted"].shape, dtype=torch.float64, device=g.device)
        for s in range(case["top_k"]):
            named = at[:, s] >= 0
            drows[at[named, s]] = g[named] * state["weights"][named, s].double()[:, None]
        return drows, (_exact_slots(state["sorted"], state["inverse"]) * g[:, None]).sum(-1)
    if kind in ("linear", "linear_grad"):
        y = _exact_rows(_exact_e4m3(state["x"]), state["w"], state["s"], kind == "linear")
        return y if state["bias"] is None else y + state["bias"].double()
    if kind in ("grouped", "grouped_grad"):
        x, ends = _exact_e4m3(state["x"]), state["offsets"].tolist()
        return torch.cat([_exact_rows(x[ends[e]:ends[e + 1]], state["w"][e], state["s"][e], kind == "grouped") for e in range(case["experts"])])
    order, inverse, offsets = _exact_sorted(state)
    token, ends = torch.div(order, case["top_k"], rounding_mode="floor"), offsets.tolist()
    x, w = _exact_e4m3(state["x"]), state["weights"].double().reshape(-1)[order][:, None]
    dout = _exact_e4m3(state["dout"]) if kind == "experts_grad" else None
    out = torch.zeros(order.numel(), case["hidden"], dtype=torch.float64, device=x.device)
    dw = torch.zeros(order.numel(), dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        at = slice(ends[e], ends[e + 1])
        if ends[e] == ends[e + 1]:
            continue
        gate, up, down = (_exact_matrix(state[name][0][e], state[name][1][e]) for name in ("gate", "up", "down"))
        g, u = torch.matmul(x[token[at]], gate.t()), torch.matmul(x[token[at]], up.t())
        h = torch.nn.functional.silu(g) * u
        if dout is None:
            out[at] = torch.matmul(_exact_e4m3(h), down.t())
            continue
        dh = torch.matmul(dout[token[at]], down)
        dw[at] = (dh * h).sum(-1)
        dh = dh * w[at]
        sigma = torch.sigmoid(g)
        dg, du = dh * u * (sigma + g * sigma * (1 - sigma)), dh * g * sigma
        out[at] = torch.matmul(_exact_e4m3(dg), gate) + torch.matmul(_exact_e4m3(du), up)
    if dout is None:
        return (_exact_slots(out, inverse) * state["weights"].double()[..., None]).sum(1)
    back = torch.empty_like(dw)
    back[order] = dw
    return _exact_slots(out, inverse).sum(1), back.reshape(inverse.shape)


# ---------------------------------------------------------------- what a pass cannot do without
def _bank_bytes(n, k):
    return n * k + 4 * _blocks(n) * _blocks(k)


def _named(experts, pairs, distinct=1):
    """Experts that `pairs` pairs name, `distinct` different ones a token, if all are as likely."""
    return min(experts, math.ceil(experts * (1.0 - (1.0 - distinct / experts) ** (pairs / distinct))))


def work(case):
    rows, size, kind = case["rows"], SIZES[case["dtype"]], case["kind"]
    if kind in ("sort", "sort_grad", "unsort", "unsort_grad"):
        hidden, pairs, ids = case["hidden"], rows * case["top_k"], 4 * rows * case["top_k"]
        wide = SIZES[case["weights"]] * pairs
        if kind == "sort":
            return {"bytes": size * hidden * (rows + pairs) + 3 * ids + 4 * case["experts"], "flops": 0}
        if kind == "unsort_grad":
            return {"bytes": size * hidden * (rows + 2 * pairs) + ids + 2 * wide, "flops": 3 * pairs * hidden}
        return {"bytes": size * hidden * (rows + pairs) + ids + (wide if kind == "unsort" else 0), "flops": (2 if kind == "unsort" else 1) * pairs * hidden}
    if kind in ("linear", "linear_grad"):
        n, k = case["n"], case["k"]
        return {"bytes": _bank_bytes(n, k) + size * (rows * (n + k) + (n if case["bias"] else 0)), "flops": 2 * rows * n * k}
    if kind in ("grouped", "grouped_grad"):
        n, k = case["n"], case["k"]
        return {"bytes": _named(case["experts"], rows) * _bank_bytes(n, k) + size * rows * (n + k), "flops": 2 * rows * n * k}
    hidden, inter, pairs = case["hidden"], case["intermediate"], rows * case["top_k"]
    bank = _named(case["experts"], pairs, case["top_k"]) * (2 * _bank_bytes(inter, hidden) + _bank_bytes(hidden, inter))
    ids = pairs * (4 + SIZES[case["weights"]])
    if kind == "experts":
        return {"bytes": bank + 2 * size * rows * hidden + ids, "flops": 6 * pairs * hidden * inter}
    return {"bytes": bank + 3 * size * rows * hidden + ids + SIZES[case["weights"]] * pairs, "flops": 10 * pairs * hidden * inter}

"""Performance cases of the operators around a trained and a served MoE layer: the gate, tokens sorted by expert and back
with their gradients, and the experts' products in 8-bit floating point.

A case is one pass of a program:

``gate``    softmax and top-k of the scores, and the gradient of the scores
``sort``    cells copied to the rows of their paths (weighted or not), and the gradients of the cells and the weights
``back``    rows added up to their cells by weight, and the gradients of the rows and the weights
``train``   gate, route, sort and back in one step with identity experts, and the gradients of cells and scores
``fp8``     rows quantized in blocks of 128, multiplied with experts' e4m3 weights that have one scale per 128 x 128 block
``serve``   gate, route, sort, an expert FFN of two such products, and back

``listed`` holds sizes of the repository's configurations and benchmark and generic ones beside them; ``draw`` gives more of
the ranges they stand for: 1 to 65536 cells of 8 to 4096 elements, 4 to 128 paths, one to four of them per cell, fp32 / fp16 /
bf16, products of 1 to 16384 rows of 128 to 8192 elements over 1 to 128 experts, odd and ragged sizes among them.
"""
import math

import torch

#: False: the plain form, elementary operations in 32 bits.  True: this framework's operators.
own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_F8 = torch.float8_e4m3fn
_F8_MAX = 448.0       # the largest e4m3 value
_LEAST = 2.0 ** -100  # blocks whose largest value is below this are scaled as if it were this
_B = 128              # elements of a row, and rows and columns of a weight, that share a scale


def _gate(name, tokens, experts, top_k, dtype):
    return {"name": name, "kind": "gate", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype}


def _rows(name, kind, tokens, d, experts, top_k, dtype, weighted=True, capacity_factor=0.0):
    """``capacity_factor`` 0: no entry is dropped."""
    return {"name": name, "kind": kind, "tokens": tokens, "d": d, "experts": experts, "top_k": top_k, "dtype": dtype,
            "weighted": weighted, "capacity_factor": capacity_factor}


def _fp8(name, rows, d_in, d_out, experts, dtype="bf16", activation="none", bias=False, skew=0.0):
    return {"name": name, "kind": "fp8", "rows": rows, "d_in": d_in, "d_out": d_out, "experts": experts, "dtype": dtype,
            "activation": activation, "bias": bias, "skew": skew}


def listed():
    return [
        # the gate of a small training step, one path per cell
        _gate("gate_1k_top1", 1024, 16, 1, "fp32"),
        # ... and of a large batch with many fine experts, from 16-bit scores
        _gate("gate_64k_top2", 65536, 128, 2, "bf16"),
        # cells to their rows in a small fp32 step: every cell on one path, nothing dropped
        _rows("sort_1k_fp32", "sort", 1024, 512, 16, 1, "fp32", weighted=False),
        # a large batch on two paths per cell, rows behind a path's capacity dropped, weights applied on the way out
        _rows("sort_16k_top2", "sort", 16384, 1024, 32, 2, "bf16", capacity_factor=1.25),
        # rows back to their cells in a short odd batch, rows of 65 units
        _rows("back_999_fp16", "back", 999, 520, 12, 2, "fp16"),
        # a large training batch on its way back, two rows to a cell, some dropped
        _rows("back_32k_top2", "back", 32768, 1024, 32, 2, "bf16", capacity_factor=1.25),
        # gate to gradient of the benchmark's batch (8192 cells, 64 paths) with two paths per cell
        _rows("train_8k_top2", "train", 8192, 768, 64, 2, "bf16", capacity_factor=1.25),
        # one token in decode: one expert of eight streams its weights
        _fp8("fp8_one_token", 1, 2048, 8192, 8),
        # a decode batch: few rows on every expert
        _fp8("fp8_decode_48", 48, 1024, 4096, 8, dtype="fp16", activation="gelu", bias=True),
        # the benchmark's number of tokens and experts, ragged: 128 rows an expert in the mean
        _fp8("fp8_8k_64e", 8192, 1024, 4096, 64, activation="gelu", skew=0.6),
        # prefill: thousands of rows per expert
        _fp8("fp8_prefill_16k", 16384, 4096, 4096, 8),
        # a whole routed layer in serving, experts in 8 bits
        {"name": "serve_4k_top2", "kind": "serve", "tokens": 4096, "d": 1024, "d_ff": 4096, "experts": 32, "top_k": 2,
         "dtype": "bf16", "capacity_factor": 1.25},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gate", "sort", "sort", "back", "back", "train", "fp8", "fp8", "fp8", "fp8", "serve"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "gate":
        experts = rng.choice([4, 8, 12, 16, 32, 60, 64, 128])
        return _gate(None, _log_int(rng, 1, 65536), experts, rng.choice([1, 2, 2, 4]), dtype)
    if kind in ("sort", "back", "train"):
        unit = 4 if dtype == "fp32" else 8  # rows are whole 16-byte units
        d = max(8, _log_int(rng, 8, 4096) // unit * unit)
        tokens = min(_log_int(rng, 1, 65536), (1 << 25) // d)
        return _rows(None, kind, tokens, d, rng.choice([4, 8, 12, 16, 32, 64, 128]), rng.choice([1, 2, 2, 4]), dtype,
                     weighted=kind != "sort" or rng.random() < 0.5, capacity_factor=rng.choice([0.0, 1.25, 2.0]))
    experts = rng.choice([1, 2, 4, 8, 16, 32, 64, 128])
    while True:
        d_in = _log_int(rng, 128, 8192) // 16 * 16
        d_out = _log_int(rng, 64, 8192)
        d_out = d_out if rng.random() < 0.25 else max(64, d_out // 64 * 64)
        if experts * d_in * d_out <= 1 << 28:
            break
    if kind == "fp8":
        most = int(min(16384, 5.4e11 / (2.0 * d_in * d_out)))
        return _fp8(None, _log_int(rng, 1, most), d_in, d_out, experts, dtype=dtype,
                    activation=rng.choice(["none", "relu"] if dtype == "fp32" else ["none", "relu", "gelu"]),
                    bias=rng.random() < 0.4, skew=rng.choice([0.0, 0.0, 0.6]))
    d_in, d_out = max(128, d_in // 2 // 16 * 16), max(128, d_out // 16 * 16)
    experts = max(4, experts)
    top_k = rng.choice([1, 2])
    most = int(min(16384, 5.4e11 / (5.0 * d_in * d_out * top_k)))
    return {"kind": "serve", "tokens": _log_int(rng, 1, most), "d": d_in, "d_ff": d_out, "experts": experts, "top_k": top_k,
            "dtype": "bf16", "capacity_factor": rng.choice([1.25, 2.0])}


# ------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def _capacity(case):
    """Rows a path keeps; as many as there are cells where nothing is dropped."""
    if not case["capacity_factor"]:
        return case["tokens"]
    return min(case["tokens"], max(4, int(case["capacity_factor"] * case["tokens"] * case["top_k"] / case["experts"])))


def _row_count(case):
    """Rows of the path-major buffer: what the layout can need at most, known without reading the loads."""
    return min(case["tokens"] * case["top_k"], case["experts"] * _capacity(case))


def _plain_route(ids, experts, capacity, rows):
    """Seats in ascending order of the entries: the 1-based row of every entry (0: dropped), the 1-based entry of every row
    (0: padding) and the kept rows per path."""
    entry_paths = ids.reshape(-1).long()
    n = entry_paths.numel()
    order = torch.sort(entry_paths, stable=True).indices
    counts = torch.bincount(entry_paths, minlength=experts)
    loads = counts.clamp(max=capacity)
    sorted_paths = entry_paths[order]
    rank = torch.arange(n, device=ids.device) - (counts.cumsum(0) - counts)[sorted_paths]
    row = (loads.cumsum(0) - loads)[sorted_paths] + rank + 1
    row = torch.where(rank < capacity, row, 0)
    seat_rows = torch.zeros(n, dtype=torch.int64, device=ids.device).scatter_(0, order, row)
    row_entries = torch.zeros(rows + 1, dtype=torch.int64, device=ids.device).scatter_(
        0, seat_rows, torch.arange(1, n + 1, device=ids.device))[1:]
    return seat_rows.view(ids.shape).int(), row_entries.int(), loads.int()


def _weights_in_blocks(gen, experts, d_out, d_in):
    """N(0, 0.02) weights as e4m3 values with one fp32 scale per 128 x 128 block."""
    n_blocks, k_blocks = -(-d_out // _B), -(-d_in // _B)
    w = torch.zeros(experts, n_blocks * _B, k_blocks * _B, device="cuda")
    w[:, :d_out, :d_in] = _normal(gen, experts, d_out, d_in, scale=0.02)
    blocks = w.view(experts, n_blocks, _B, k_blocks, _B)
    amax = blocks.abs().amax(dim=(2, 4))
    q = (blocks * (_F8_MAX / amax)[:, :, None, :, None]).to(_F8).view(torch.uint8).view(w.shape)
    return q[:, :d_out, :d_in].contiguous().view(_F8), amax / _F8_MAX


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, experts = case["kind"], _DTYPES[case["dtype"]], case["experts"]
    state = {"case": case}
    if kind == "fp8":
        share = 1.0 / torch.arange(1, experts + 1, device="cuda", dtype=torch.float32) ** case["skew"]
        share = share[torch.randperm(experts, device="cuda", generator=gen)]
        paths = torch.multinomial(share, case["rows"], replacement=True, generator=gen)
        state["loads"] = torch.bincount(paths, minlength=experts).int()
        state["most"] = int(state["loads"].max())  # (the plain form's room for one expert)
        state["x"] = _normal(gen, case["rows"], case["d_in"], dtype=dtype)
        state["w"], state["ws"] = _weights_in_blocks(gen, experts, case["d_out"], case["d_in"])
        state["bias"] = _normal(gen, experts, case["d_out"], dtype=dtype, scale=0.1) if case["bias"] else None
        return state
    tokens, k = case["tokens"], case["top_k"]
    scores = _normal(gen, tokens, experts)
    if kind == "gate":
        state["scores"] = scores.to(dtype).requires_grad_()
        state["grad"] = _normal(gen, tokens, k)
        return state
    d = case["d"]
    state["x"] = _normal(gen, tokens, d, dtype=dtype)
    if kind in ("train", "serve"):
        state["scores"] = scores
        state["capacities"] = torch.tensor([_capacity(case)], dtype=torch.int32, device="cuda")
        if kind == "train":
            state["grad"] = _normal(gen, tokens, d, dtype=dtype)
            state["x"].requires_grad_(), state["scores"].requires_grad_()
        else:
            state["w1"], state["ws1"] = _weights_in_blocks(gen, experts, case["d_ff"], d)
            state["w2"], state["ws2"] = _weights_in_blocks(gen, experts, d, case["d_ff"])
        return state
    # the route that the gate of this step has made
    rows = _row_count(case)
    top = torch.topk(scores, k, dim=1)
    state["ids"] = top.indices.int()
    state["seat_rows"], state["row_entries"], _ = _plain_route(state["ids"], experts, _capacity(case), rows)
    state["weights"] = torch.softmax(top.values, dim=1).requires_grad_() if case["weighted"] else None
    if kind == "sort":
        state["x"].requires_grad_()
        state["grad"] = _normal(gen, rows, d, dtype=dtype)
    else:
        state["y"] = _normal(gen, rows, d, dtype=dtype).requires_grad_()
        state["grad"] = _normal(gen, tokens, d, dtype=dtype)
    return state


# ----------------------------------------------------------------------------- the plain forms
def _plain_gate(scores, k):
    """Softmax over the row; the k largest, the lowest path first among equals."""
    s = scores.float()
    e = torch.exp(s - s.amax(dim=1, keepdim=True))
    p = e / e.sum(dim=1, keepdim=True)
    ids = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :k]
    return ids, p.gather(1, ids), p


def _plain_gate_grad(ids, weights, p, grad):
    picked = torch.zeros_like(p).scatter_(1, ids, grad)
    return p * (picked - (grad * weights).sum(dim=1, keepdim=True))


def _of_entries(rows, seat_rows):
    """``[cells, k, d]``: the row of every entry in 32 bits, zeros for entries without one."""
    padded = torch.cat([rows.new_zeros(1, rows.shape[1]), rows]).float()
    return padded[seat_rows.long()]


def _to_rows(cells, row_entries, k, weights):
    """``[rows, d]``: the cell behind every row (times the weight of its entry), zeros for padding rows."""
    filled = (row_entries > 0)[:, None]
    entry = (row_entries.long() - 1).clamp(min=0)
    rows = cells.float()[entry // k]
    if weights is not None:
        rows = rows * weights.reshape(-1)[entry][:, None]
    return torch.where(filled, rows, 0.0)


def _plain_sort(state):
    x, grad, weights = state["x"].detach(), state["grad"], state["weights"]
    weights = None if weights is None else weights.detach()
    k = state["case"]["top_k"]
    rows = _to_rows(x, state["row_entries"], k, weights)
    of_entries = _of_entries(grad, state["seat_rows"])
    found = {"rows": rows.to(x.dtype)}
    if weights is None:
        found["dx"] = of_entries.sum(dim=1).to(x.dtype)
    else:
        found["dx"] = (of_entries * weights[:, :, None]).sum(dim=1).to(x.dtype)
        found["dweights"] = (of_entries * x.float()[:, None]).sum(dim=2)
    return found


def _plain_back(state):
    y, grad, weights = state["y"].detach(), state["grad"], state["weights"].detach()
    of_entries = _of_entries(y, state["seat_rows"])
    return {"out": (of_entries * weights[:, :, None]).sum(dim=1).to(y.dtype),
            "dy": _to_rows(grad, state["row_entries"], state["case"]["top_k"], weights).to(y.dtype),
            "dweights": (of_entries * grad.float()[:, None]).sum(dim=2)}


def _plain_train(state):
    case, x, grad = state["case"], state["x"].detach(), state["grad"]
    ids, weights, p = _plain_gate(state["scores"].detach(), case["top_k"])
    seat_rows, row_entries, _ = _plain_route(ids, case["experts"], _capacity(case), _row_count(case))
    rows = _to_rows(x, row_entries, case["top_k"], None)
    of_entries = _of_entries(rows, seat_rows)
    out = (of_entries * weights[:, :, None]).sum(dim=1)
    dweights = (of_entries * grad.float()[:, None]).sum(dim=2)
    drows = _to_rows(grad, row_entries, case["top_k"], weights)
    return {"ids": ids.int(), "out": out.to(x.dtype), "dx": _of_entries(drows, seat_rows).sum(dim=1).to(x.dtype),
            "dscores": _plain_gate_grad(ids, weights, p, dweights)}


def _dequantized(x):
    """The values that rows stand for once they are rounded to e4m3 with one fp32 scale per 128 elements."""
    rows, d = x.shape
    padded = torch.zeros(rows, -(-d // _B) * _B, device=x.device)
    padded[:, :d] = x
    blocks = padded.view(rows, -1, _B)
    amax = blocks.abs().amax(dim=2, keepdim=True).clamp(min=_LEAST)
    return ((blocks * (_F8_MAX / amax)).to(_F8).float() * (amax / _F8_MAX)).view(rows, -1)[:, :d]


def _weight_values(w, scales):
    """``[experts, d_in, d_out]``: the values that the e4m3 weights stand for."""
    spread = scales.repeat_interleave(_B, dim=1)[:, :w.shape[1]].repeat_interleave(_B, dim=2)[:, :, :w.shape[2]]
    return (w.float() * spread).transpose(1, 2).contiguous()


def _plain_product(x, w, scales, loads, most, bias, activation):
    """Rows of ``x`` (packed by expert) times their expert's weights, in 32 bits: every expert has room for ``most`` rows."""
    experts = w.shape[0]
    starts = loads.cumsum(0) - loads
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(loads.cumsum(0), row, right=True)
    expert = expert.clamp(max=experts - 1)  # (rows behind the last expert's are nobody's)
    seat = (row - starts[expert]).clamp(max=most)
    room = torch.zeros(experts, most + 1, x.shape[1], device=x.device)
    room[expert, seat] = _dequantized(x)
    out = torch.matmul(room, _weight_values(w, scales))
    if bias is not None:
        out = out + bias.float()[:, None]
    if activation == "gelu":
        out = out * 0.5 * (1.0 + torch.erf(out * math.sqrt(0.5)))
    elif activation == "relu":
        out = out.clamp(min=0.0)
    return out[expert, seat]


def _plain_serve(state):
    case, x = state["case"], state["x"]
    ids, weights, _ = _plain_gate(state["scores"], case["top_k"])
    capacity = _capacity(case)
    seat_rows, row_entries, loads = _plain_route(ids, case["experts"], capacity, _row_count(case))
    rows = _to_rows(x, row_entries, case["top_k"], None)
    # the hidden rows are held in the cells' type: that is what is quantized for the second product
    hidden = _plain_product(rows, state["w1"], state["ws1"], loads, capacity, None, "gelu").to(x.dtype)
    y = _plain_product(hidden, state["w2"], state["ws2"], loads, capacity, None, "none")
    return {"out": (_of_entries(y, seat_rows) * weights[:, :, None]).sum(dim=1).to(x.dtype), "loads": loads}


# ------------------------------------------------------------------------------------ a pass
def _own_serve(state):
    from brainstorm_amd._C import router as c_router
    from brainstorm_amd.jit import grouped_linear_fp8

    case, x = state["case"], state["x"]
    ids, weights = c_router.gate_topk(state["scores"], case["top_k"], softmax=True)
    loads, _, seat_rows, row_entries = c_router.route_by_path(ids, case["experts"], state["capacities"], rows=_row_count(case))
    rows = c_router.dispatch_by_rows(x, row_entries, case["top_k"])
    hidden, scales = grouped_linear_fp8(rows, state["w1"], state["ws1"], loads, activation="gelu", out_blocks=True)
    # (the experts' rows stay in 32 bits until they are added up)
    y = grouped_linear_fp8(hidden, state["w2"], state["ws2"], loads, x_scales=scales, out_dtype=torch.float32, exact=False)
    return {"out": c_router.combine_by_rows(y, ids, seat_rows, weights, out_dtype=x.dtype), "loads": loads}


def _own(state):
    from brainstorm_amd._C import router as c_router

    case = state["case"]
    kind = case["kind"]
    if kind == "fp8":
        from brainstorm_amd.jit import grouped_linear_fp8

        return {"out": grouped_linear_fp8(state["x"], state["w"], state["ws"], state["loads"], bias=state["bias"],
                                          activation=case["activation"])}
    if kind == "gate":
        scores = state["scores"]
        ids, weights = c_router.gate_topk(scores, case["top_k"], softmax=True, differentiable=True)
        (dscores,) = torch.autograd.grad(weights, scores, state["grad"])
        return {"ids": ids, "weights": weights.detach(), "dscores": dscores}
    if kind == "sort":
        x, weights = state["x"], state["weights"]
        rows = c_router.dispatch_by_rows(x, state["row_entries"], case["top_k"], weights, seat_rows=state["seat_rows"])
        found = torch.autograd.grad(rows, [x] if weights is None else [x, weights], state["grad"])
        return {"rows": rows.detach(), **dict(zip(("dx", "dweights"), found))}
    if kind == "back":
        y, weights = state["y"], state["weights"]
        out = c_router.combine_by_rows(y, state["ids"], state["seat_rows"], weights, row_entries=state["row_entries"])
        dy, dweights = torch.autograd.grad(out, [y, weights], state["grad"])
        return {"out": out.detach(), "dy": dy, "dweights": dweights}
    x, scores, k = state["x"], state["scores"], case["top_k"]
    ids, weights = c_router.gate_topk(scores, k, softmax=True, differentiable=True)
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, case["experts"], state["capacities"], rows=_row_count(case))
    rows = c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows)
    out = c_router.combine_by_rows(rows, ids, seat_rows, weights, row_entries=row_entries)
    dx, dscores = torch.autograd.grad(out, [x, scores], state["grad"])
    return {"ids": ids, "out": out.detach(), "dx": dx, "dscores": dscores}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _own_serve(state) if kind == "serve" else _own(state)
    if kind == "gate":
        ids, weights, p = _plain_gate(state["scores"].detach(), case["top_k"])
        return {"ids": ids.int(), "weights": weights,
                "dscores": _plain_gate_grad(ids, weights, p, state["grad"]).to(state["scores"].dtype)}
    if kind == "fp8":
        out = _plain_product(state["x"].float(), state["w"], state["ws"], state["loads"], state["most"], state["bias"],
                             case["activation"])
        return {"out": out.to(state["x"].dtype)}
    return {"sort": _plain_sort, "back": _plain_back, "train": _plain_train, "serve": _plain_serve}[kind](state)


# ------------------------------------------------------------------------- the same in 64 bits
def _exact_gate(scores, k):
    s = scores.detach().double()
    ids = torch.argsort(-s, dim=1, stable=True)[:, :k]
    return ids, torch.log_softmax(s, dim=1).exp()


def _exact_route(ids, experts, capacity):
    """The 0-based row of every entry, -1 where it is dropped, from the one-hot matrix of the route."""
    hot = torch.nn.functional.one_hot(ids.reshape(-1).long(), experts)
    rank = (hot.cumsum(0) - hot).gather(1, ids.reshape(-1, 1).long())[:, 0]
    kept = hot.sum(0).clamp(max=capacity)
    first = torch.nn.functional.pad(kept.cumsum(0), (1, 0))[:-1]
    return torch.where(rank < capacity, first[ids.reshape(-1).long()] + rank, -1), kept


def _exact_rows(cells, row_of_entry, rows, k, weights=None):
    """Entries written to their rows one after the other, in 64 bits."""
    keep = torch.nonzero(row_of_entry >= 0)[:, 0]
    out = torch.zeros(rows, cells.shape[1], dtype=torch.float64, device=cells.device)
    values = cells.double()[keep // k]
    out[row_of_entry[keep]] = values if weights is None else values * weights.detach().double().reshape(-1, 1)[keep]
    return out


def _exact_cells(rows, row_of_entry, cells, k, weights=None):
    keep = torch.nonzero(row_of_entry >= 0)[:, 0]
    values = rows.double()[row_of_entry[keep]]
    if weights is not None:
        values = values * weights.detach().double().reshape(-1, 1)[keep]
    return torch.zeros(cells, rows.shape[1], dtype=torch.float64, device=rows.device).index_add_(0, keep // k, values)


def _exact_dots(rows, cells, row_of_entry, k):
    keep = torch.nonzero(row_of_entry >= 0)[:, 0]
    dots = torch.zeros(row_of_entry.numel(), dtype=torch.float64, device=rows.device)
    dots[keep] = torch.linalg.vecdot(rows.double()[row_of_entry[keep]], cells.double()[keep // k])
    return dots.view(-1, k)


def _exact_quantized(x):
    """What the rows stand for: the scale and the product with its inverse are fp32 by definition, then e4m3."""
    columns = torch.split(x.float(), _B, dim=1)
    found = []
    for part in columns:
        largest = torch.clamp(part.abs().max(dim=1, keepdim=True).values, min=_LEAST)
        found.append((part * (448.0 / largest)).to(_F8).double() * (largest / 448.0).double())
    return torch.cat(found, dim=1)


def _exact_product(x, w, scales, loads, bias, activation):
    values = _exact_quantized(x)
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    first = 0
    n = torch.arange(w.shape[1], device=x.device) // _B
    k = torch.arange(w.shape[2], device=x.device) // _B
    for e, load in enumerate(loads.tolist()):
        if load:
            weight = w[e].double() * scales[e].double()[n][:, k]
            out[first:first + load] = values[first:first + load] @ weight.t()
            if bias is not None:
                out[first:first + load] += bias[e].double()
            first += load
    return {"gelu": torch.nn.functional.gelu, "relu": torch.relu, "none": lambda v: v}[activation](out)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "fp8":
        return {"out": _exact_product(state["x"], state["w"], state["ws"], state["loads"], state["bias"], case["activation"])}
    k, experts = case["top_k"], case["experts"]
    if kind == "gate":
        ids, p = _exact_gate(state["scores"], k)
        grad = torch.zeros_like(p).scatter_(1, ids, state["grad"].double())
        return {"ids": ids.int(), "weights": p.gather(1, ids), "dscores": p * grad - p * (p * grad).sum(1, keepdim=True)}
    tokens, rows = case["tokens"], _row_count(case)
    if kind in ("sort", "back"):
        row, _ = _exact_route(state["ids"], experts, _capacity(case))
        weights, grad = state["weights"], state["grad"]
        if kind == "back":
            return {"out": _exact_cells(state["y"].detach(), row, tokens, k, weights), "dy": _exact_rows(grad, row, rows, k, weights),
                    "dweights": _exact_dots(state["y"].detach(), grad, row, k)}
        x = state["x"].detach()
        found = {"rows": _exact_rows(x, row, rows, k, weights), "dx": _exact_cells(grad, row, tokens, k, weights)}
        return found if weights is None else {**found, "dweights": _exact_dots(grad, x, row, k)}
    ids, p = _exact_gate(state["scores"], k)
    weights = p.gather(1, ids)
    row, kept = _exact_route(ids, experts, _capacity(case))
    x = state["x"].detach()
    if kind == "train":
        of_rows, grad = _exact_rows(x, row, rows, k), state["grad"]
        dots = torch.zeros_like(p).scatter_(1, ids, _exact_dots(of_rows, grad, row, k))
        return {"ids": ids.int(), "out": _exact_cells(of_rows, row, tokens, k, weights),
                "dx": _exact_cells(_exact_rows(grad, row, rows, k, weights), row, tokens, k),
                "dscores": p * dots - p * (p * dots).sum(1, keepdim=True)}
    of_rows = _exact_rows(x, row, rows, k)
    hidden = _exact_product(of_rows, state["w1"], state["ws1"], kept, None, "gelu").to(x.dtype)
    y = _exact_product(hidden, state["w2"], state["ws2"], kept, None, "none")
    return {"out": _exact_cells(y, row, tokens, k, weights), "loads": kept.int()}


# ------------------------------------------------------------------------------------- work
def work(case):
    """Every input read once, every output written once."""
    kind, experts, size = case["kind"], case["experts"], _DTYPES[case["dtype"]].itemsize

    def used(entries):  # experts that get a row at all, each as likely as the others
        return experts * (1.0 - (1.0 - 1.0 / experts) ** entries)

    if kind == "fp8":
        rows, d_in, d_out = case["rows"], case["d_in"], case["d_out"]
        weights = used(rows) * d_in * d_out * (1.0 + 4.0 / _B ** 2)
        return {"bytes": weights + rows * (d_in + d_out) * size, "flops": 2.0 * rows * d_in * d_out}
    tokens, k = case["tokens"], case["top_k"]
    entries = tokens * k
    if kind == "gate":
        # scores and their gradient, the gradient of the weights, ids and weights
        return {"bytes": 2 * tokens * experts * size + 12 * entries, "flops": 8.0 * tokens * experts}
    d, rows = case["d"], _row_count(case)
    kept = min(entries, experts * _capacity(case))
    cells = tokens * d * size
    if kind == "sort":
        # cells, their gradient, rows and the kept rows of theirs; the route, the weights and their gradient
        return {"bytes": 2 * cells + (rows + kept) * d * size + 4 * (rows + entries) + (8 * entries if case["weighted"] else 0),
                "flops": (3.0 if case["weighted"] else 1.0) * kept * d}
    if kind == "back":
        return {"bytes": 2 * cells + (rows + kept) * d * size + 4 * (rows + 2 * entries) + 8 * entries, "flops": 5.0 * kept * d}
    if kind == "train":
        # scores, cells, their gradients, the result and its gradient; what lies between need not leave the chip
        return {"bytes": 2 * tokens * experts * 4 + 4 * cells, "flops": 6.0 * kept * d}
    weights = 2 * used(entries) * d * case["d_ff"] * (1.0 + 4.0 / _B ** 2)
    return {"bytes": tokens * experts * 4 + 2 * cells + weights, "flops": 4.0 * kept * d * case["d_ff"]}

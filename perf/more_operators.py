"""Performance cases of the router's losses and of expert products with 4-bit weights.

A case is one pass of a program:

``balance``  the balance and z losses of a batch of scores with the entries per expert, and the gradient of the scores
``train``    gate, losses, route, cells to their rows and back in one step with identity experts, and the gradients of cells and scores
``int4``     rows packed by expert times their expert's weights, which are held in 4 bits with a scale (and zero point) per group
``serve``    gate, route, an expert FFN of two such products on the routed cells, and back

``listed`` holds sizes of the repository's configurations and benchmark and generic ones beside them; ``draw`` gives more of
the ranges they stand for: 1 to 65536 cells, 4 to 256 paths, one to eight of them per cell, fp32 / fp16 / bf16; products of 1 to
16384 rows of 64 to 8192 elements over 1 to 128 experts, groups of 32, 64 and 128, odd and ragged sizes among them.

The layout of the weights: ``values`` uint8 ``[experts, tiles of 16 rows, blocks of 128 columns, 1024]``; byte ``16 * (16 * g + r) + 4
* j + m`` of a block belongs to row ``r`` of the tile and holds column ``32 * j + 8 * g + m`` in its low and ``+ 4`` in its high four bits.
``scales`` and ``zeros`` are ``[experts, tiles of 16 rows, groups, 16]``.  A weight stands for ``(value - zero) * scale``, with a zero of 8
where there are none.
"""
import math

import torch

#: False: the plain form, elementary operations in 32 bits.  True: this framework's operators.
own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_B = 128  # columns of a block of the weights' layout
_R = 16   # rows of a tile of it


def _balance(name, tokens, experts, top_k, dtype, padded=0.0):
    """``padded``: the share of cells that are padding and do not count."""
    return {"name": name, "kind": "balance", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "padded": padded}


def _train(name, tokens, d, experts, top_k, dtype, capacity_factor=1.25):
    return {"name": name, "kind": "train", "tokens": tokens, "d": d, "experts": experts, "top_k": top_k, "dtype": dtype,
            "capacity_factor": capacity_factor}


def _int4(name, rows, d_in, d_out, experts, group=128, zeros=False, dtype="bf16", activation="none", bias=False, skew=0.0):
    return {"name": name, "kind": "int4", "rows": rows, "d_in": d_in, "d_out": d_out, "experts": experts, "group": group,
            "zeros": zeros, "dtype": dtype, "activation": activation, "bias": bias, "skew": skew}


def _serve(name, tokens, d, d_ff, experts, top_k, group, zeros, capacity_factor=2.0):
    return {"name": name, "kind": "serve", "tokens": tokens, "d": d, "d_ff": d_ff, "experts": experts, "top_k": top_k,
            "group": group, "zeros": zeros, "dtype": "bf16", "capacity_factor": capacity_factor}


def listed():
    return [
        # the losses of a small fp32 step (the smallest configuration's cells and paths)
        _balance("balance_1k_top1", 1024, 16, 1, "fp32"),
        # ... of a short odd batch of padded sequences, four of 60 paths per cell
        _balance("balance_4099_padded", 4099, 60, 4, "fp16", padded=0.3),
        # ... of a large batch with many fine experts, from 16-bit scores
        _balance("balance_64k_top2", 65536, 128, 2, "bf16"),
        # gate, losses and route of the benchmark's batch (8192 cells, 64 paths) in one training step, two paths per cell
        _train("train_8k_losses", 8192, 768, 64, 2, "bf16"),
        # one token in decode: one expert of eight streams its weights
        _int4("int4_one_token", 1, 2048, 8192, 8),
        # a decode batch: few rows on every expert, short groups with zero points
        _int4("int4_decode_48", 48, 1024, 4096, 8, group=64, zeros=True, dtype="fp16", activation="gelu", bias=True),
        # a larger decode batch over many experts: four rows an expert in the mean, some with none
        _int4("int4_decode_256", 256, 4096, 1024, 64, skew=0.6),
        # fp32 rows of odd lengths on the shortest groups, a dozen experts
        _int4("int4_odd_fp32", 333, 776, 1001, 12, group=32, dtype="fp32", bias=True),
        # the benchmark's number of tokens and experts, ragged: 128 rows an expert in the mean
        _int4("int4_8k_64e", 8192, 1024, 4096, 64, activation="gelu", skew=0.6),
        # prefill: thousands of rows per expert
        _int4("int4_prefill_16k", 16384, 4096, 4096, 8, group=64, zeros=True),
        # a routed layer in decode, experts in 4 bits
        _serve("serve_64_top2", 64, 1024, 4096, 32, 2, 128, False),
        # ... and of a short prefill
        _serve("serve_2k_top2", 2048, 1024, 4096, 32, 2, 64, True, capacity_factor=1.25),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["balance", "balance", "balance", "train", "int4", "int4", "int4", "int4", "int4", "serve"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "balance":
        experts = rng.choice([4, 8, 12, 16, 32, 60, 64, 128, 160, 256])
        tokens = min(_log_int(rng, 1, 65536), (1 << 23) // experts)
        return _balance(None, tokens, experts, min(experts, rng.choice([1, 2, 2, 4, 8])), dtype, padded=rng.choice([0.0, 0.0, 0.2, 0.6]))
    if kind == "train":
        unit = 4 if dtype == "fp32" else 8  # rows are whole 16-byte units
        d = max(8, _log_int(rng, 8, 2048) // unit * unit)
        tokens = min(_log_int(rng, 1, 32768), (1 << 23) // d)
        return _train(None, tokens, d, rng.choice([4, 8, 12, 16, 32, 64, 128]), rng.choice([1, 2, 2, 4]), dtype,
                      capacity_factor=rng.choice([1.25, 2.0]))
    experts = rng.choice([1, 2, 4, 8, 16, 32, 64, 128])
    while True:
        d_in = _log_int(rng, 64, 8192) // 8 * 8
        d_out = _log_int(rng, 64, 8192)
        d_out = d_out if rng.random() < 0.25 else max(64, d_out // 64 * 64)
        if experts * d_in * d_out <= 1 << 28:
            break
    group, zeros = rng.choice([32, 64, 128, 128]), rng.random() < 0.5
    if kind == "int4":
        most = int(min(16384, 5.4e11 / (2.0 * d_in * d_out)))
        return _int4(None, _log_int(rng, 1, most), d_in, d_out, experts, group=group, zeros=zeros, dtype=dtype,
                     activation=rng.choice(["none", "relu", "gelu"]), bias=rng.random() < 0.4, skew=rng.choice([0.0, 0.0, 0.6]))
    d, d_ff, experts = max(64, d_in // 2 // 8 * 8), max(64, d_out // 8 * 8), max(4, experts)
    top_k = rng.choice([1, 2])
    most = int(min(4096, 1.0e11 / (4.0 * d * d_ff * top_k)))
    return _serve(None, _log_int(rng, 1, max(1, most)), d, d_ff, experts, top_k, group, zeros, capacity_factor=rng.choice([1.25, 2.0]))


# ------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def _capacity(case):
    """Rows a path keeps."""
    return min(case["tokens"], max(4, int(case["capacity_factor"] * case["tokens"] * case["top_k"] / case["experts"])))


def _row_count(case):
    """Rows of the path-major buffer: what the layout can need at most, known without reading the loads."""
    return min(case["tokens"] * case["top_k"], case["experts"] * _capacity(case))


def _weights(gen, experts, d_out, d_in, group, zeros):
    """Values as the quantization of N(0, 0.02) weights leaves them (a group's largest one near the end of the range), packed;
    scales in bf16, zero points a little off the middle."""
    tiles, blocks, groups = -(-d_out // _R), -(-d_in // _B), -(-d_in // group)
    q = torch.randn(experts, tiles * _R, blocks * _B, device="cuda", generator=gen).mul_(2.7).round_().add_(8).clamp_(0, 15).to(torch.uint8)
    q[:, d_out:], q[:, :, d_in:] = 0, 0
    # [e, tile, r, block, j, g, half, m] -> [e, tile, block, g, r, j, m]
    q = q.view(experts, tiles, _R, blocks, 4, 4, 2, 4).permute(0, 1, 3, 5, 2, 4, 7, 6)
    values = (q[..., 0] | (q[..., 1] << 4)).reshape(experts, tiles, blocks, 1024)
    shape = (experts, tiles, groups, _R)
    scales = torch.empty(shape, device="cuda").uniform_(0.004, 0.012, generator=gen).to(torch.bfloat16)
    points = torch.randint(6, 11, shape, device="cuda", generator=gen).to(torch.uint8) if zeros else None
    return {"values": values, "scales": scales, "zeros": points, "d_in": d_in, "d_out": d_out, "group": group}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, experts = case["kind"], _DTYPES[case["dtype"]], case["experts"]
    state = {"case": case}
    if kind == "int4":
        share = 1.0 / torch.arange(1, experts + 1, device="cuda", dtype=torch.float32) ** case["skew"]
        share = share[torch.randperm(experts, device="cuda", generator=gen)]
        paths = torch.multinomial(share, case["rows"], replacement=True, generator=gen)
        state["loads"] = torch.bincount(paths, minlength=experts).int()
        state["most"] = int(state["loads"].max())  # (the plain form's room for one expert)
        state["x"] = _normal(gen, case["rows"], case["d_in"], dtype=dtype)
        state["w"] = _weights(gen, experts, case["d_out"], case["d_in"], case["group"], case["zeros"])
        state["bias"] = _normal(gen, experts, case["d_out"], dtype=dtype, scale=0.1) if case["bias"] else None
        return state
    tokens, k = case["tokens"], case["top_k"]
    # some paths are preferred, as in a router that is not balanced yet
    scores = _normal(gen, tokens, experts) + _normal(gen, 1, experts, scale=0.5)
    if kind in ("balance", "train"):
        # what a training step multiplies the two losses by; with fp16 scores the loss is scaled up, or their gradient would vanish
        state["by"] = (torch.tensor([1e-2, 1e-3], device="cuda") * (65536.0 if kind == "balance" and case["dtype"] == "fp16" else 1.0)).unbind()
    if kind == "balance":
        scores = scores.to(dtype)
        state["ids"] = torch.sort(scores.float(), dim=1, descending=True, stable=True).indices[:, :k].int().contiguous()
        state["scores"] = scores.requires_grad_()
        state["counted"] = torch.rand(tokens, device="cuda", generator=gen) >= case["padded"] if case["padded"] else None
        return state
    state["x"] = _normal(gen, tokens, case["d"], dtype=dtype)
    state["scores"] = scores
    state["capacities"] = torch.tensor([_capacity(case)], dtype=torch.int32, device="cuda")
    if kind == "train":
        state["grad"] = _normal(gen, tokens, case["d"], dtype=dtype)
        state["x"].requires_grad_(), state["scores"].requires_grad_()
    else:
        state["w1"] = _weights(gen, experts, case["d_ff"], case["d"], case["group"], case["zeros"])
        state["w2"] = _weights(gen, experts, case["d"], case["d_ff"], case["group"], case["zeros"])
    return state


# ----------------------------------------------------------------------------- the plain forms
def _plain_losses(scores, ids, counted, by):
    """(balance, z, counts, gradient of the scores in 32 bits).  ``p`` the softmax of a cell, n the cells that count, f the share of
    their entries that go to a path: balance = experts * sum over paths of f * mean(p), z = mean(log(sum(exp(scores)))^2)."""
    s = scores.float()
    tokens, experts = s.shape
    k = ids.shape[1]
    use = torch.ones(tokens, device=s.device) if counted is None else counted.float()
    top = s.amax(dim=1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(dim=1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total))[:, 0]
    counts = torch.zeros(experts, device=s.device).index_add_(0, ids.reshape(-1).long(), use.repeat_interleave(k))
    n = use.sum().clamp(min=1.0)
    f = counts / (n * k)
    mean_p = (p * use[:, None]).sum(dim=0) / n
    balance = experts * (f * mean_p).sum()
    z = (use * lse * lse).sum() / n
    inner = experts * f - (experts * p * f).sum(dim=1, keepdim=True)
    grad = p * (use / n)[:, None] * (by[0] * inner + by[1] * 2.0 * lse[:, None])
    return balance, z, counts.int(), grad


def _plain_gate(scores, k):
    """Softmax over the row; the k largest, the lowest path first among equals."""
    s = scores.float()
    e = torch.exp(s - s.amax(dim=1, keepdim=True))
    p = e / e.sum(dim=1, keepdim=True)
    ids = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :k]
    return ids, p.gather(1, ids), p


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
    return seat_rows.view(ids.shape), row_entries, loads.int()


def _of_entries(rows, seat_rows):
    """``[cells, k, d]``: the row of every entry in 32 bits, zeros for entries without one."""
    padded = torch.cat([rows.new_zeros(1, rows.shape[1]), rows]).float()
    return padded[seat_rows]


def _to_rows(cells, row_entries, k, weights=None):
    """``[rows, d]``: the cell behind every row (times the weight of its entry), zeros for padding rows."""
    entry = (row_entries - 1).clamp(min=0)
    rows = cells.float()[entry // k]
    if weights is not None:
        rows = rows * weights.reshape(-1)[entry][:, None]
    return torch.where((row_entries > 0)[:, None], rows, 0.0)


def _plain_train(state):
    case, x, grad, scores = state["case"], state["x"].detach(), state["grad"], state["scores"].detach()
    k = case["top_k"]
    ids, weights, p = _plain_gate(scores, k)
    balance, z, counts, dlosses = _plain_losses(scores, ids, None, state["by"])
    seat_rows, row_entries, _ = _plain_route(ids, case["experts"], _capacity(case), _row_count(case))
    rows = _to_rows(x, row_entries, k)
    of_entries = _of_entries(rows, seat_rows)
    out = (of_entries * weights[:, :, None]).sum(dim=1)
    dweights = (of_entries * grad.float()[:, None]).sum(dim=2)
    drows = _to_rows(grad, row_entries, k, weights)
    dgate = p * (torch.zeros_like(p).scatter_(1, ids, dweights) - (dweights * weights).sum(dim=1, keepdim=True))
    return {"ids": ids.int(), "out": out.to(x.dtype), "balance": balance, "z": z, "counts": counts,
            "dx": _of_entries(drows, seat_rows).sum(dim=1).to(x.dtype), "dscores": dgate + dlosses}


def _weight_values(w):
    """``[experts, d_in, d_out]``: what the packed weights stand for, in 32 bits."""
    experts, tiles, blocks, _ = w["values"].shape
    q = w["values"].view(experts, tiles, blocks, 4, _R, 4, 4)  # [e, tile, block, g, r, j, m]
    q = torch.stack([q & 15, q >> 4], dim=-2)                 # [e, tile, block, g, r, j, half, m]
    q = q.permute(0, 2, 5, 3, 6, 7, 1, 4).reshape(experts, blocks * _B, tiles * _R)[:, :w["d_in"], :w["d_out"]].float()

    def spread(t):  # [e, tile, group, r] -> [e, d_in, d_out]
        t = t.permute(0, 2, 1, 3).reshape(experts, t.shape[2], tiles * _R)[:, :, :w["d_out"]].float()
        return t.repeat_interleave(w["group"], dim=1)[:, :w["d_in"]]

    return (q - (8.0 if w["zeros"] is None else spread(w["zeros"]))) * spread(w["scales"])


def _plain_product(x, w, loads, most, bias, activation):
    """Rows of ``x`` (packed by expert) times their expert's weights, in 32 bits: every expert has room for ``most`` rows."""
    experts = w["values"].shape[0]
    starts = loads.cumsum(0) - loads
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(loads.cumsum(0), row, right=True)
    expert = expert.clamp(max=experts - 1)  # (rows behind the last expert's are nobody's)
    seat = (row - starts[expert]).clamp(max=most)
    room = torch.zeros(experts, most + 1, x.shape[1], device=x.device)
    room[expert, seat] = x.float()
    out = torch.matmul(room, _weight_values(w))
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
    rows = _to_rows(x, row_entries, case["top_k"])
    # the hidden rows are held in the cells' type between the two products
    hidden = _plain_product(rows, state["w1"], loads, capacity, None, "gelu").to(x.dtype)
    y = _plain_product(hidden, state["w2"], loads, capacity, None, "none")
    return {"out": (_of_entries(y, seat_rows) * weights[:, :, None]).sum(dim=1).to(x.dtype), "loads": loads}


# ------------------------------------------------------------------------------------ a pass
def _own_weight(w):
    from brainstorm_amd.jit import Int4Weight

    return Int4Weight(w["values"], w["scales"], w["zeros"], w["d_in"], w["d_out"], w["group"])


def _own(state):
    from brainstorm_amd._C import router as c_router

    case = state["case"]
    kind = case["kind"]
    if kind in ("int4", "serve"):
        from brainstorm_amd.jit import grouped_linear_int4
    if kind == "int4":
        return {"out": grouped_linear_int4(state["x"], _own_weight(state["w"]), state["loads"], bias=state["bias"],
                                           activation=case["activation"])}
    scores = state["scores"]
    if kind == "balance":
        balance, z, counts = c_router.balance_loss(scores, state["ids"], counted=state["counted"])
        (dscores,) = torch.autograd.grad([balance, z], scores, state["by"])
        return {"balance": balance.detach(), "z": z.detach(), "counts": counts, "dscores": dscores}
    x, k = state["x"], case["top_k"]
    if kind == "serve":
        ids, weights = c_router.gate_topk(scores, k, softmax=True)
        loads, _, seat_rows, row_entries = c_router.route_by_path(ids, case["experts"], state["capacities"], rows=_row_count(case))
        hidden = grouped_linear_int4(x, _own_weight(state["w1"]), loads, activation="gelu", row_entries=row_entries, entries_per_cell=k)
        # (the experts' rows stay in 32 bits until they are added up)
        y = grouped_linear_int4(hidden, _own_weight(state["w2"]), loads, out_dtype=torch.float32)
        return {"out": c_router.combine_by_rows(y, ids, seat_rows, weights, out_dtype=x.dtype), "loads": loads}
    ids, weights = c_router.gate_topk(scores, k, softmax=True, differentiable=True)
    balance, z, counts = c_router.balance_loss(scores, ids)
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, case["experts"], state["capacities"], rows=_row_count(case))
    rows = c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows)
    out = c_router.combine_by_rows(rows, ids, seat_rows, weights, row_entries=row_entries)
    dx, dscores = torch.autograd.grad([out, balance, z], [x, scores], [state["grad"], *state["by"]])
    return {"ids": ids, "out": out.detach(), "balance": balance.detach(), "z": z.detach(), "counts": counts, "dx": dx, "dscores": dscores}


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "balance":
        scores = state["scores"].detach()
        balance, z, counts, grad = _plain_losses(scores, state["ids"], state["counted"], state["by"])
        return {"balance": balance, "z": z, "counts": counts, "dscores": grad.to(scores.dtype)}
    if kind == "int4":
        out = _plain_product(state["x"], state["w"], state["loads"], state["most"], state["bias"], case["activation"])
        return {"out": out.to(state["x"].dtype)}
    return {"train": _plain_train, "serve": _plain_serve}[kind](state)


# ------------------------------------------------------------------------- the same in 64 bits
def _exact_losses(scores, ids, counted, by):
    """The losses of the cells that count, and their gradient from the derivative of each."""
    s = scores.detach().double()
    experts = s.shape[1]
    keep = torch.ones(s.shape[0], dtype=torch.bool, device=s.device) if counted is None else counted
    part, chosen = s[keep], ids[keep].long()
    counts = torch.bincount(chosen.reshape(-1), minlength=experts)
    dscores = torch.zeros_like(s)
    n = part.shape[0]
    if n == 0:
        return s.new_zeros(()), s.new_zeros(()), counts.int(), dscores
    p, lse = torch.softmax(part, dim=1), torch.logsumexp(part, dim=1)
    weight = counts.double() * (experts / (n * n * ids.shape[1]))  # d balance / d p, the same for every cell
    inner = p @ weight
    dscores[keep] = p * (float(by[0]) * (weight - inner[:, None]) + float(by[1]) * (2.0 / n) * lse[:, None])
    return inner.sum(), lse.square().mean(), counts.int(), dscores


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
    keep = torch.nonzero(row_of_entry >= 0)[:, 0]
    out = torch.zeros(rows, cells.shape[1], dtype=torch.float64, device=cells.device)
    values = cells.double()[keep // k]
    out[row_of_entry[keep]] = values if weights is None else values * weights.reshape(-1, 1)[keep]
    return out


def _exact_cells(rows, row_of_entry, cells, k, weights=None):
    keep = torch.nonzero(row_of_entry >= 0)[:, 0]
    values = rows.double()[row_of_entry[keep]]
    if weights is not None:
        values = values * weights.reshape(-1, 1)[keep]
    return torch.zeros(cells, rows.shape[1], dtype=torch.float64, device=rows.device).index_add_(0, keep // k, values)


def _exact_weight(w, e):
    """``[d_out, d_in]`` of one expert, byte by byte of the layout."""
    tiles, blocks = w["values"].shape[1:3]
    at = torch.arange(1024, device="cuda")
    r, g, j, m = at // 16 % 16, at // 256, at // 4 % 4, at % 4
    q = torch.zeros(tiles, _R, blocks, _B, dtype=torch.float64, device="cuda")
    q[:, r, :, 32 * j + 8 * g + m] = (w["values"][e] & 15).double().permute(2, 0, 1)
    q[:, r, :, 32 * j + 8 * g + m + 4] = (w["values"][e] >> 4).double().permute(2, 0, 1)
    q = q.view(tiles * _R, blocks * _B)[:w["d_out"], :w["d_in"]]
    of = torch.arange(w["d_in"], device="cuda") // w["group"]
    scale = w["scales"][e].double().transpose(1, 2).reshape(tiles * _R, -1)[:w["d_out"]][:, of]
    zero = 8.0 if w["zeros"] is None else w["zeros"][e].double().transpose(1, 2).reshape(tiles * _R, -1)[:w["d_out"]][:, of]
    return (q - zero) * scale


def _exact_product(x, w, loads, bias, activation):
    out = torch.zeros(x.shape[0], w["d_out"], dtype=torch.float64, device=x.device)
    first = 0
    for e, load in enumerate(loads.tolist()):
        if load:
            out[first:first + load] = x[first:first + load].double() @ _exact_weight(w, e).t()
            if bias is not None:
                out[first:first + load] += bias[e].double()
            first += load
    return {"gelu": torch.nn.functional.gelu, "relu": torch.relu, "none": lambda v: v}[activation](out)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "int4":
        return {"out": _exact_product(state["x"], state["w"], state["loads"], state["bias"], case["activation"])}
    if kind == "balance":
        return dict(zip(("balance", "z", "counts", "dscores"), _exact_losses(state["scores"], state["ids"], state["counted"], state["by"])))
    k, experts, tokens, rows = case["top_k"], case["experts"], case["tokens"], _row_count(case)
    ids, p = _exact_gate(state["scores"], k)
    weights = p.gather(1, ids)
    row, kept = _exact_route(ids, experts, _capacity(case))
    x = state["x"].detach()
    of_rows = _exact_rows(x, row, rows, k)
    if kind == "serve":
        hidden = _exact_product(of_rows, state["w1"], kept, None, "gelu").to(x.dtype)
        y = _exact_product(hidden, state["w2"], kept, None, "none")
        return {"out": _exact_cells(y, row, tokens, k, weights), "loads": kept.int()}
    grad = state["grad"]
    keep = torch.nonzero(row >= 0)[:, 0]
    dots = torch.zeros(row.numel(), dtype=torch.float64, device="cuda")
    dots[keep] = torch.linalg.vecdot(of_rows[row[keep]], grad.double()[keep // k])
    dots = torch.zeros_like(p).scatter_(1, ids, dots.view(-1, k))
    balance, z, counts, dlosses = _exact_losses(state["scores"], ids, None, state["by"])
    return {"ids": ids.int(), "out": _exact_cells(of_rows, row, tokens, k, weights), "balance": balance, "z": z, "counts": counts,
            "dx": _exact_cells(_exact_rows(grad, row, rows, k, weights), row, tokens, k),
            "dscores": p * dots - p * (p * dots).sum(1, keepdim=True) + dlosses}


# ------------------------------------------------------------------------------------- work
def work(case):
    """Every input read once, every output written once."""
    kind, experts, size = case["kind"], case["experts"], _DTYPES[case["dtype"]].itemsize

    def used(entries):  # experts that get a row at all, each as likely as the others
        return experts * (1.0 - (1.0 - 1.0 / experts) ** entries)

    def weight_bytes(d_in, d_out):
        groups = -(-d_in // case["group"])
        return d_in * d_out / 2 + groups * d_out * (3 if case["zeros"] else 2)

    if kind == "int4":
        rows, d_in, d_out = case["rows"], case["d_in"], case["d_out"]
        return {"bytes": used(rows) * weight_bytes(d_in, d_out) + rows * (d_in + d_out) * size, "flops": 2.0 * rows * d_in * d_out}
    tokens, k = case["tokens"], case["top_k"]
    entries = tokens * k
    if kind == "balance":
        # scores and their gradient, ids, the mask and the counts
        return {"bytes": 2 * tokens * experts * size + 4 * entries + (tokens if case["padded"] else 0) + 4 * experts,
                "flops": 12.0 * tokens * experts}
    d = case["d"]
    kept = min(entries, experts * _capacity(case))
    cells = tokens * d * size
    if kind == "train":
        # scores, cells, their gradients, the result and its gradient; what lies between need not leave the chip
        return {"bytes": 2 * tokens * experts * 4 + 4 * cells, "flops": 6.0 * kept * d + 12.0 * tokens * experts}
    weights = used(entries) * (weight_bytes(d, case["d_ff"]) + weight_bytes(case["d_ff"], d))
    return {"bytes": tokens * experts * 4 + 2 * cells + weights, "flops": 4.0 * kept * d * case["d_ff"]}

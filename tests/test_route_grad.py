"""Gradients of the compact route's ops against the formulas in 64 bits, against differences, and their refusals.

Tolerances: a result is a sum of n fp32 products, each rounded once and added in fp32, then rounded to its type.  The sum is
within n * 2^-23 of the sum of the terms' magnitudes (n roundings of products and n of sums, half a step of 2^-23 each), the
last rounding within half a step of the value (``torch.finfo(t).eps / 2``, and half of the smallest subnormal).
"""
import pytest
import torch

import brt._C.router as c_router

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make_route(cells, paths, k, capacity, seed, keep=1.0):
    """Random distinct paths per cell (some entries without one where ``keep`` < 1) and the route that route_by_path lays out."""
    gen = torch.Generator().manual_seed(seed)
    ids = torch.rand(cells, paths, generator=gen).argsort(1)[:, :k].int()
    if keep < 1.0:
        ids = torch.where(torch.rand(cells, k, generator=gen) < keep, ids, -1)
    ids = ids.contiguous().cuda()
    caps = torch.tensor([capacity], dtype=torch.int32, device="cuda")
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, paths, caps, rows=min(cells * k, paths * capacity) + 3)
    return ids, seat_rows, row_entries


def normal(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def near(got, want, magnitude, terms):
    info = torch.finfo(got.dtype)
    bound = terms * 2.0 ** -23 * magnitude + info.eps / 2 * (want.abs() + terms * 2.0 ** -23 * magnitude) + info.tiny * info.eps
    off = (got.detach().double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound.clamp(min=1e-300)).max())} of the bound"


def of_entries(rows, seat_rows):
    padded = torch.cat([rows.new_zeros(1, rows.shape[1]), rows]).double()
    return padded[seat_rows.long()]


SHAPES = [  # cells, paths, k, capacity, elements
    (1, 4, 1, 1, 8), (1, 4, 4, 1, 16), (3, 5, 2, 2, 24), (64, 8, 1, 100, 64), (65, 8, 2, 12, 136), (257, 16, 3, 40, 264),
    (999, 12, 2, 200, 520), (130, 9, 8, 90, 1032), (515, 64, 4, 20, 72), (77, 6, 2, 20, 4104), (2048, 32, 2, 100, 1024),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("cells,paths,k,capacity,d", SHAPES)
def test_dispatch_gradients(cells, paths, k, capacity, d, weighted, dtype):
    dtype = TYPES[dtype]
    ids, seat_rows, row_entries = make_route(cells, paths, k, capacity, cells, keep=0.8)
    x = normal(1, cells, d, dtype=dtype).requires_grad_()
    w = normal(2, cells, k).requires_grad_() if weighted else None
    rows = c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows)
    plain = c_router.dispatch_by_rows(x.detach(), row_entries, k, None if w is None else w.detach())
    assert torch.equal(rows, plain) and rows.requires_grad and not plain.requires_grad
    grad = normal(3, *rows.shape, dtype=dtype)
    found = torch.autograd.grad(rows, [x] + ([w] if weighted else []), grad)
    terms = of_entries(grad, seat_rows)
    if weighted:
        terms_x = terms * w.detach().double()[:, :, None]
        products = terms * x.detach().double()[:, None]
        near(found[1], products.sum(2), products.abs().sum(2), d)
        assert not found[1][seat_rows == 0].any()
    else:
        terms_x = terms
    near(found[0], terms_x.sum(1), terms_x.abs().sum(1), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("cells,paths,k,capacity,d", SHAPES)
def test_combine_gradients(cells, paths, k, capacity, d, weighted, dtype, out):
    dtype, out = TYPES[dtype], TYPES[out]
    ids, seat_rows, row_entries = make_route(cells, paths, k, capacity, cells + 1, keep=0.8)
    y = normal(1, row_entries.numel(), d, dtype=dtype).requires_grad_()
    w = normal(2, cells, k).requires_grad_() if weighted else None
    got = c_router.combine_by_rows(y, ids, seat_rows, w, out_dtype=out, row_entries=row_entries)
    plain = c_router.combine_by_rows(y.detach(), ids, seat_rows, None if w is None else w.detach(), out_dtype=out)
    assert torch.equal(got, plain) and got.dtype == out and got.requires_grad
    grad = normal(3, cells, d, dtype=out)
    found = torch.autograd.grad(got, [y] + ([w] if weighted else []), grad)
    entry = (row_entries.long() - 1).clamp(min=0)
    want = grad.double()[entry // k] * (1.0 if w is None else w.detach().double().reshape(-1)[entry][:, None])
    want = torch.where((row_entries > 0)[:, None], want, 0.0)
    assert found[0].dtype == dtype
    near(found[0], want, want.abs(), 1)
    assert not found[0][row_entries == 0].any()
    if weighted:
        products = of_entries(y.detach(), seat_rows) * grad.double()[:, None]
        near(found[1], products.sum(2), products.abs().sum(2), d)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("cells,paths,k,capacity,d", SHAPES)
def test_fp32_rows_combined_into_16_bits(cells, paths, k, capacity, d, weighted, out):
    """The fp32 sum of the rows, rounded once; and its gradients."""
    out = TYPES[out]
    ids, seat_rows, row_entries = make_route(cells, paths, k, capacity, cells + 2, keep=0.8)
    y, w = normal(1, row_entries.numel(), d).requires_grad_(), normal(2, cells, k) if weighted else None
    got = c_router.combine_by_rows(y, ids, seat_rows, w, out_dtype=out, row_entries=row_entries)
    wide = c_router.combine_by_rows(y.detach(), ids, seat_rows, w)
    assert got.dtype == out and torch.equal(got, wide.to(out))
    kept = torch.full((cells, d), 3.0, dtype=out, device="cuda")
    c_router.combine_by_rows(y.detach(), ids, seat_rows, w, kept)
    has = (seat_rows > 0).any(1)
    assert torch.equal(kept[has], got[has]) and bool((kept[~has] == 3.0).all())
    grad = normal(3, cells, d, dtype=out)
    (dy,) = torch.autograd.grad(got, y, grad)
    entry = (row_entries.long() - 1).clamp(min=0)
    want = grad.double()[entry // k] * (1.0 if w is None else w.double().reshape(-1)[entry][:, None])
    near(dy, torch.where((row_entries > 0)[:, None], want, 0.0), want.abs(), 1)


GATES = [(1, 1, 1), (1, 4, 4), (5, 3, 2), (63, 8, 2), (130, 60, 3), (257, 64, 1), (33, 100, 4), (70, 128, 2), (9, 1000, 8), (17, 1024, 2), (12, 513, 13)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("cells,paths,k", GATES)
def test_gate_gradient(cells, paths, k, softmax, dtype):
    """p is the softmax in fp32: exp within 2 steps of 2^-23, the sum within paths steps, the quotient within one; the bracket's
    sum over j within k + 1 steps more, and twice the weights' own error."""
    dtype = TYPES[dtype]
    scores = (3 * normal(cells, cells, paths)).to(dtype).requires_grad_()
    ids, weights, mask = c_router.gate_topk(scores, k, softmax, True, differentiable=True)
    plain = c_router.gate_topk(scores.detach(), k, softmax, True)
    assert all(torch.equal(a, b) for a, b in zip((ids, weights, mask), plain))
    assert weights.requires_grad and not ids.requires_grad and not mask.requires_grad
    grad = normal(2, cells, k)
    (got,) = torch.autograd.grad(weights, scores, grad)
    picked = torch.zeros(cells, paths, dtype=torch.float64, device="cuda").scatter_(1, ids.long(), grad.double())
    if not softmax:
        return near(got, picked, picked.abs(), 0)
    p = torch.softmax(scores.detach().double(), 1)
    parts = p.gather(1, ids.long()) * grad.double()
    want = p * (picked - parts.sum(1, keepdim=True))
    near(got, want, p * (picked.abs() + parts.abs().sum(1, keepdim=True)), 2 * paths + k + 8)


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32 operands of a few bits and steps of 2^-3: every op is linear in each operand, so a difference quotient is the
    derivative but for the fp32 roundings of the two values."""
    cells, paths, k, d = 13, 4, 2, 8
    ids, seat_rows, row_entries = make_route(cells, paths, k, 5, 1)
    x, w = normal(1, cells, d).round(), normal(2, cells, k).round()
    up = normal(3, row_entries.numel(), d).round()

    def of_dispatch(x, w):
        return (c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows).double() * up).sum()

    y, back = normal(4, row_entries.numel(), d).round(), normal(5, cells, d).round()

    def of_combine(y, w):
        return (c_router.combine_by_rows(y, ids, seat_rows, w, row_entries=row_entries).double() * back).sum()

    for op, operands in ((of_dispatch, (x, w)), (of_combine, (y, w))):
        leaves = [t.clone().requires_grad_() for t in operands]
        grads = torch.autograd.grad(op(*leaves), leaves)
        for n, grad in enumerate(grads):
            flat = operands[n].reshape(-1)
            for i in range(0, flat.numel(), 7):
                moved = []
                for step in (0.125, -0.125):
                    other = [t.clone() for t in operands]
                    other[n].view(-1)[i] += step
                    moved.append(op(*other))
                assert float((moved[0] - moved[1]) / 0.25) == float(grad.reshape(-1)[i])


@pytest.mark.gpu
def test_a_path_named_twice_by_a_cell():
    """The dispatch copies the cell to both rows, the combine adds the first of them only: so do their gradients."""
    ids = torch.tensor([[1, 1], [0, 1], [-1, -1]], dtype=torch.int32, device="cuda")
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, 2)
    d = 8
    x, w = normal(1, 3, d).requires_grad_(), normal(2, 3, 2).requires_grad_()
    rows = c_router.dispatch_by_rows(x, row_entries, 2, w, seat_rows=seat_rows)
    grad = normal(3, *rows.shape)
    dx, dw = torch.autograd.grad(rows, [x, w], grad)
    terms = of_entries(grad, seat_rows)
    near(dx, (terms * w.detach().double()[:, :, None]).sum(1), (terms * w.detach().double()[:, :, None]).abs().sum(1), 2)
    y = normal(4, *rows.shape).requires_grad_()
    out = c_router.combine_by_rows(y, ids, seat_rows, w, row_entries=row_entries)
    g = normal(5, 3, d)
    dy, dw = torch.autograd.grad(out, [y, w], g)
    first, second = seat_rows[0].tolist()
    assert not dy[second - 1].any() and float(dw[0, 1]) == 0.0
    near(dy[first - 1], w[0, 0].detach().double() * g[0].double(), (w[0, 0] * g[0]).detach().double().abs(), 1)
    assert not dw[2].any() and not dx[2].any()


@pytest.mark.gpu
def test_what_belongs_to_no_entry_is_not_looked_at():
    """NaN in rows without an entry and in weights of entries without a row do not reach the gradients."""
    ids = torch.tensor([[0, -1], [1, 0], [0, 1]], dtype=torch.int32, device="cuda")
    caps = torch.tensor([2], dtype=torch.int32, device="cuda")
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, 2, caps, rows=6)
    w = normal(1, 3, 2)
    w[seat_rows == 0] = float("nan")
    w.requires_grad_()
    x = normal(2, 3, 32).requires_grad_()
    grad = normal(3, 6, 32)
    grad[row_entries == 0] = float("nan")
    dx, dw = torch.autograd.grad(c_router.dispatch_by_rows(x, row_entries, 2, w, seat_rows=seat_rows), [x, w], grad)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    y = normal(4, 6, 32)
    y[row_entries == 0] = float("nan")
    y.requires_grad_()
    out = c_router.combine_by_rows(y, ids, seat_rows, w, row_entries=row_entries)
    dy, dw = torch.autograd.grad(out, [y, w], normal(5, 3, 32))
    assert torch.isfinite(out).all() and torch.isfinite(dy).all() and torch.isfinite(dw).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("k,d", [(1, 8), (2, 32), (3, 264), (8, 1032)])
def test_cells_that_are_not_finite_and_entries_without_a_row(k, d, dtype):
    """The weight of an entry without a row has the gradient zero, whatever its cell and the gradient of its result hold."""
    cells, paths, dtype = 24, 9, TYPES[dtype]
    ids, _, _ = make_route(cells, paths, k, 40, 1)
    ids[:3], ids[3:9, ::2] = -1, -1  # all entries of some cells have no row, every other one of some
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, paths, rows=cells * k)
    given = normal(2, cells, d, dtype=dtype)
    x = given.clone()
    x[0], x[1, 5], x[3, 0], x[4], x[5, d - 1] = float("nan"), float("inf"), float("inf"), float("nan"), float("-inf")
    w = normal(3, cells, k).requires_grad_()
    grad = normal(4, row_entries.numel(), d, dtype=dtype)

    def of_dispatch(x):
        return torch.autograd.grad(c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows), w, grad)[0]

    dw, sound = of_dispatch(x), of_dispatch(given)
    assert not dw[seat_rows == 0].any()
    assert not torch.isfinite(dw[3:6][seat_rows[3:6] > 0]).any()
    finite = torch.isfinite(x).all(1)
    assert torch.equal(dw[finite], sound[finite])
    # the combine's: rows and gradients that are not finite beside entries without a row
    y = normal(5, row_entries.numel(), d, dtype=dtype)
    out = c_router.combine_by_rows(y, ids, seat_rows, w, row_entries=row_entries)
    (dw,) = torch.autograd.grad(out, w, x)
    assert not dw[seat_rows == 0].any() and not torch.isfinite(dw[3:6][seat_rows[3:6] > 0]).any()


@pytest.mark.gpu
def test_gate_gradient_of_masked_scores():
    """Scores of -inf have no probability and no gradient; a row of nothing else is NaN, as its softmax is."""
    scores = normal(1, 4, 40)
    scores[0, 3:] = float("-inf")
    scores[1, ::2] = torch.finfo(torch.float32).min
    scores[2] = float("-inf")
    scores.requires_grad_()
    ids, weights = c_router.gate_topk(scores, 2, True, differentiable=True)
    (got,) = torch.autograd.grad(weights, scores, torch.ones_like(weights))
    p = torch.softmax(scores.detach().double(), 1)
    sums = p.gather(1, ids.long()).sum(1, keepdim=True)
    want = p * (torch.zeros_like(p).scatter_(1, ids.long(), 1.0) - sums)
    assert not got[0, 3:].any() and not got[1, ::2].any() and got[2].isnan().all()
    rows = [0, 1, 3]
    near(got[rows], want[rows], p[rows] * (1 + sums[rows]), 2 * 40 + 10)


@pytest.mark.gpu
def test_what_a_gate_without_softmax_keeps():
    """Its gradient reads neither scores nor weights: both may be written to before the backward pass; with softmax that is an error."""
    given = normal(1, 20, 8).requires_grad_()
    for softmax in (False, True):
        scores = given * 1.0
        ids, weights = c_router.gate_topk(scores, 2, softmax, differentiable=True)
        weights /= 2.0
        with torch.no_grad():
            scores.zero_()
        if softmax:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(weights.sum(), given)
        else:
            (got,) = torch.autograd.grad(weights.sum(), given)
            assert torch.equal(got, torch.zeros_like(given).scatter_(1, ids.long(), 0.5))


@pytest.mark.gpu
def test_only_what_is_asked_for():
    cells, k, d = 50, 2, 64
    ids, seat_rows, row_entries = make_route(cells, 4, k, 20, 1)
    x, w = normal(1, cells, d), normal(2, cells, k)
    assert not c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows).requires_grad
    with torch.no_grad():
        assert not c_router.dispatch_by_rows(x.requires_grad_(), row_entries, k, w, seat_rows=seat_rows).requires_grad
    x = x.detach()
    grad = normal(3, row_entries.numel(), d)
    both = [t.clone().requires_grad_() for t in (x, w)]
    want = torch.autograd.grad(c_router.dispatch_by_rows(both[0], row_entries, k, both[1], seat_rows=seat_rows), both, grad)
    for n in range(2):
        pair = [x.clone(), w.clone()]
        pair[n].requires_grad_()
        (got,) = torch.autograd.grad(c_router.dispatch_by_rows(pair[0], row_entries, k, pair[1], seat_rows=seat_rows), pair[n], grad)
        assert torch.equal(got, want[n])
    y, back = normal(4, row_entries.numel(), d), normal(5, cells, d)
    both = [t.clone().requires_grad_() for t in (y, w)]
    want = torch.autograd.grad(c_router.combine_by_rows(both[0], ids, seat_rows, both[1], row_entries=row_entries), both, back)
    for n in range(2):
        pair = [y.clone(), w.clone()]
        pair[n].requires_grad_()
        (got,) = torch.autograd.grad(c_router.combine_by_rows(pair[0], ids, seat_rows, pair[1], row_entries=row_entries), pair[n], back)
        assert torch.equal(got, want[n])


@pytest.mark.gpu
def test_strides_shapes_and_broadcast_gradients():
    """Cells of several dimensions, operands that are views, a gradient without strides (that of a sum)."""
    cells, k = 40, 2
    ids, seat_rows, row_entries = make_route(cells, 6, k, 30, 1)
    base = normal(1, cells, 4, 24)
    x = base.transpose(1, 2)[:, ::2].requires_grad_()  # [cells, 12, 4], not contiguous
    w = normal(2, k, cells).t().requires_grad_()
    rows = c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows)
    assert rows.shape == (row_entries.numel(), 12, 4)
    dx, dw = torch.autograd.grad(rows.sum(), [x, w])
    has = (seat_rows > 0).double()
    near(dx, (has * w.detach().double()).sum(1)[:, None, None].expand(cells, 12, 4), (has * w.detach().double().abs()).sum(1)[:, None, None], k)
    sums = x.detach().double().sum((1, 2))[:, None] * has
    near(dw, sums, x.detach().double().abs().sum((1, 2))[:, None] * has, 48)
    out = c_router.combine_by_rows(rows.detach().requires_grad_(), ids, seat_rows, row_entries=row_entries)
    assert out.shape == x.shape
    wide = normal(3, 30, 16)[:, ::2].requires_grad_()
    _, weights = c_router.gate_topk(wide, 2, True, differentiable=True)
    (got,) = torch.autograd.grad(weights.sum(), wide)
    assert got.shape == wide.shape and torch.isfinite(got).all()


@pytest.mark.gpu
def test_gates_of_a_differentiable_combine():
    cells, paths, k, d = 33, 5, 2, 16
    ids, seat_rows, row_entries = make_route(cells, paths, k, 40, 1)
    y, gates = normal(1, row_entries.numel(), d).requires_grad_(), normal(2, cells, paths).requires_grad_()
    out = c_router.combine_by_rows(y, ids, seat_rows, gates=gates, row_entries=row_entries)
    assert torch.equal(out, c_router.combine_by_rows(y.detach(), ids, seat_rows, gates=gates.detach()))
    back = normal(3, cells, d)
    _, dgates = torch.autograd.grad(out, [y, gates], back)
    products = of_entries(y.detach(), seat_rows) * back.double()[:, None]
    want = torch.zeros(cells, paths, dtype=torch.float64, device="cuda").scatter_(1, ids.long(), products.sum(2))
    near(dgates, want, torch.zeros_like(want).scatter_(1, ids.long(), products.abs().sum(2)), d)


def test_gates_are_not_read_at_ids_outside_the_paths(monkeypatch):
    """An id below zero or beyond the paths names no path: the weight handed to the kernel comes from the row of the cell all the same,
    and so does its gradient's place."""
    from brainstorm_amd import _lib

    class Handed:
        @staticmethod
        def combine_by_rows(in_data, path_ids, seat_rows, weights, out_data, out_dtype, gates, row_entries):
            return weights

    monkeypatch.setattr(_lib, "native", lambda: Handed)
    ids = torch.tensor([[-1, 2], [3, 0], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    entries = torch.zeros(2, dtype=torch.int32)
    for gates, row_entries in ((torch.arange(9.0).view(3, 3), entries), (torch.arange(9.0, dtype=torch.float64).view(3, 3), None),
                               (torch.arange(12.0).view(4, 3), None)):
        gates.requires_grad_()
        weights = c_router.combine_by_rows(None, ids, None, gates=gates, row_entries=row_entries)
        assert weights.dtype == torch.float32 and weights[0, 1] == 2.0 and weights[1, 1] == 3.0
        (found,) = torch.autograd.grad(weights, gates, torch.tensor([[0.0, 1.0], [0.0, 1.0], [0.0, 0.0]]))
        assert found[0, 2] == 1.0 and found[1, 0] == 1.0 and found.sum() == 2.0
    with pytest.raises(RuntimeError, match="at least one path"):
        c_router.combine_by_rows(None, ids, None, gates=torch.zeros(3, 0), row_entries=entries)
    with pytest.raises(RuntimeError, match="at least one path"):
        c_router.combine_by_rows(None, ids, None, gates=torch.zeros(9), row_entries=entries)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_of_entries_without_a_path(dtype):
    """Ids of -1 and beyond the paths, in the first cell and the last: result and gradients of the entries that have a path."""
    cells, paths, k, d = 33, 5, 3, 16
    ids, _, _ = make_route(cells, paths, k, 40, 1, keep=0.7)
    ids[0, 0], ids[0, 1], ids[-1] = -1, paths, torch.tensor([2 ** 31 - 1, -2 ** 31, paths + 3])
    _, _, seat_rows, row_entries = c_router.route_by_path(ids, paths, rows=cells * k)
    assert not seat_rows[(ids < 0) | (ids >= paths)].any()
    y = normal(1, row_entries.numel(), d).requires_grad_()
    gates = normal(2, cells, paths, dtype=TYPES[dtype]).requires_grad_()
    out = c_router.combine_by_rows(y, ids, seat_rows, gates=gates, row_entries=row_entries)
    assert torch.equal(out, c_router.combine_by_rows(y.detach(), ids, seat_rows, gates=gates.detach()))
    wide = gates.detach().double()  # (weights from outside the kernel)
    assert torch.equal(out, c_router.combine_by_rows(y.detach(), ids, seat_rows, gates=wide))
    back = normal(3, cells, d)
    dy, dgates = torch.autograd.grad(out, [y, gates], back)
    column = ids.long().clamp(0, paths - 1)
    products = of_entries(y.detach(), seat_rows) * back.double()[:, None]
    zero = torch.zeros(cells, paths, dtype=torch.float64, device="cuda")
    near(dgates, zero.scatter_add(1, column, products.sum(2)), zero.scatter_add(1, column, products.abs().sum(2)), d)
    entry = (row_entries.long() - 1).clamp(min=0)
    want = back.double()[entry // k] * gates.detach().double().gather(1, column).reshape(-1)[entry][:, None]
    near(dy, torch.where((row_entries > 0)[:, None], want, 0.0), want.abs(), 1)


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused():
    cells, k, d = 20, 1, 16
    ids, seat_rows, row_entries = make_route(cells, 4, k, 20, 1)
    x = normal(1, cells, d).requires_grad_()
    rows = c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows)
    (dx,) = torch.autograd.grad((rows * rows).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(dx.sum(), x)


@pytest.mark.gpu
def test_forward_mode_gradients_are_refused():
    """A tangent is never dropped without an error; tensors without one go through, and duals through ops that are cut off anyway."""
    import torch.autograd.forward_ad as forward

    cells, k, d = 20, 2, 16
    ids, seat_rows, row_entries = make_route(cells, 4, k, 20, 1)
    x, w, scores = normal(1, cells, d), normal(2, cells, k), normal(3, cells, 4)
    y, gates = normal(4, row_entries.numel(), d), normal(5, cells, 4)
    calls = [
        (lambda t: c_router.gate_topk(t, k, True, differentiable=True)[1], scores),
        (lambda t: c_router.gate_topk(t, k, differentiable=True)[1], scores),
        (lambda t: c_router.dispatch_by_rows(t, row_entries, k, w, seat_rows=seat_rows), x),
        (lambda t: c_router.dispatch_by_rows(x, row_entries, k, t, seat_rows=seat_rows), w),
        (lambda t: c_router.combine_by_rows(t, ids, seat_rows, w, row_entries=row_entries), y),
        (lambda t: c_router.combine_by_rows(y, ids, seat_rows, t, row_entries=row_entries), w),
        (lambda t: c_router.combine_by_rows(y, ids, seat_rows, gates=t, row_entries=row_entries), gates),
    ]
    for call, given in calls:
        want = call(given)
        with forward.dual_level():
            dual = forward.make_dual(given, torch.ones_like(given))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward.make_dual(given.clone().requires_grad_(), torch.ones_like(given)))
            assert torch.equal(call(forward.unpack_dual(dual).primal), want) and torch.equal(call(given), want)
            assert torch.equal(c_router.gate_topk(forward.make_dual(scores, scores), k, True)[1], c_router.gate_topk(scores, k, True)[1])


@pytest.mark.gpu
def test_refusals_of_the_differentiable_forms():
    cells, k, d = 20, 2, 16
    ids, seat_rows, row_entries = make_route(cells, 4, k, 20, 1)
    x, w = normal(1, cells, d).requires_grad_(), normal(2, cells, k)
    y = normal(3, row_entries.numel(), d).requires_grad_()
    room = torch.empty(row_entries.numel(), d, device="cuda")
    with pytest.raises(RuntimeError, match="not both"):
        c_router.dispatch_by_rows(x, row_entries, k, out=room, seat_rows=seat_rows)
    with pytest.raises(RuntimeError, match=r"\[cells, k\]"):
        c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows[:-1])
    with pytest.raises(RuntimeError, match="int32"):
        c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows.long())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows.cpu())
    with pytest.raises(RuntimeError, match="another device"):
        c_router.dispatch_by_rows(x, row_entries, k, w.cpu(), seat_rows=seat_rows)
    with pytest.raises(NotImplementedError):
        c_router.dispatch_by_rows(x, row_entries, 9, seat_rows=torch.ones(cells, 9, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="neither out_data nor gates"):
        c_router.combine_by_rows(y, ids, seat_rows, out_data=torch.zeros(cells, d, device="cuda"), row_entries=row_entries)
    with pytest.raises(RuntimeError, match="one entry for every row"):
        c_router.combine_by_rows(y, ids, seat_rows, row_entries=row_entries[:-1])
    with pytest.raises(RuntimeError, match="fp32"):
        c_router.combine_by_rows(y, ids, seat_rows, w.double(), row_entries=row_entries)
    with pytest.raises(NotImplementedError):
        c_router.combine_by_rows(y[:, :3], ids, seat_rows, row_entries=row_entries)
    saved = x * 1
    rows = c_router.dispatch_by_rows(saved, row_entries, k, w.requires_grad_(), seat_rows=seat_rows)
    with torch.no_grad():
        saved.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        rows.sum().backward()


@pytest.mark.gpu
def test_no_cells_and_no_rows():
    none = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    entries = torch.zeros(3, dtype=torch.int32, device="cuda")
    rows = c_router.dispatch_by_rows(x, entries, 2, seat_rows=none)
    (dx,) = torch.autograd.grad(rows.sum(), x)
    assert dx.shape == x.shape
    y = normal(1, 3, 16).requires_grad_()
    out = c_router.combine_by_rows(y, none, none, row_entries=entries)
    (dy,) = torch.autograd.grad(out.sum(), y)
    assert out.shape == (0, 16) and dy.shape == y.shape and not dy.any()
    bare = torch.zeros(5, 1, dtype=torch.int32, device="cuda")
    nothing = torch.zeros(0, dtype=torch.int32, device="cuda")
    x = normal(2, 5, 16).requires_grad_()
    w = normal(3, 5, 1).requires_grad_()
    rows = c_router.dispatch_by_rows(x, nothing, 1, w, seat_rows=bare)
    dx, dw = torch.autograd.grad(rows.sum(), [x, w])
    assert rows.shape == (0, 16) and not dx.any() and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_results_of_no_cells_and_of_no_rows_are_zeros(dtype):
    """Rows of a dispatch without cells, cells of a combine without rows; memory that held something else before."""
    d, dtype = 24, TYPES[dtype]
    none = torch.zeros(0, 2, dtype=torch.int32, device="cuda")

    def used(rows, kind):
        torch.full((rows, d), 7.0, dtype=kind, device="cuda")  # (what the allocator hands out next)

    for seat_rows in (None, none):
        x = torch.zeros(0, d, dtype=dtype, device="cuda", requires_grad=True)
        used(3, dtype)
        rows = c_router.dispatch_by_rows(x, torch.zeros(3, dtype=torch.int32, device="cuda"), 2, seat_rows=seat_rows)
        assert rows.shape == (3, d) and not rows.any()
    ids = torch.tensor([[0, 1], [1, 2], [-1, 0], [2, 1], [0, 2]], dtype=torch.int32, device="cuda")
    bare, nothing = torch.zeros(5, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    gates, w = normal(1, 5, 3).requires_grad_(), normal(2, 5, 2).requires_grad_()
    y = torch.zeros(0, d, dtype=dtype, device="cuda", requires_grad=True)
    for entries in (None, nothing):
        for kind in {dtype, torch.float32}:
            for operand in ({}, {"weights": w}, {"gates": gates}):
                used(5, kind)
                out = c_router.combine_by_rows(y, ids, bare, out_dtype=kind, row_entries=entries, **operand)
                assert out.shape == (5, d) and out.dtype == kind and not out.any()
                if entries is not None:
                    found = torch.autograd.grad(out, [y] + list(operand.values()), torch.ones_like(out))
                    assert found[0].shape == y.shape and not any(g.any() for g in found)
    kept = torch.full((5, d), 7.0, dtype=dtype, device="cuda")
    assert bool((c_router.combine_by_rows(y.detach(), ids, bare, None, kept) == 7.0).all())


@pytest.mark.gpu
def test_a_training_step_of_all_three_on_a_stream_and_replayed():
    """Gate, route, sort and back with identity experts: against autograd over plain torch in 64 bits, on a stream of its own,
    and captured once and replayed for other inputs."""
    cells, paths, k, d = 96, 8, 2, 64
    caps = torch.tensor([20], dtype=torch.int32, device="cuda")

    def step(x, scores, back):
        ids, weights = c_router.gate_topk(scores, k, True, differentiable=True)
        _, _, seat_rows, row_entries = c_router.route_by_path(ids, paths, caps, rows=paths * 20)
        rows = c_router.dispatch_by_rows(x, row_entries, k, seat_rows=seat_rows)
        out = c_router.combine_by_rows(rows, ids, seat_rows, weights, row_entries=row_entries)
        return (seat_rows, ids, out) + torch.autograd.grad(out, [x, scores], back)

    def inputs(seed):
        return normal(seed, cells, d).requires_grad_(), normal(seed + 1, cells, paths).requires_grad_(), normal(seed + 2, cells, d)

    def check(made, x, scores, back):
        seat_rows, ids, out, dx, dscores = made
        x64, s64 = x.detach().double().requires_grad_(), scores.detach().double().requires_grad_()
        w64 = torch.softmax(s64, 1).gather(1, ids.long()) * (seat_rows > 0)
        want = x64 * w64.sum(1, keepdim=True)
        gx, gs = torch.autograd.grad(want, [x64, s64], back.double())
        torch.testing.assert_close(out.double(), want.detach(), rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(dx.double(), gx, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(dscores.double(), gs, rtol=1e-4, atol=2e-5)

    first = inputs(1)
    check(step(*first), *first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = inputs(11)
        made = step(*second)
    torch.cuda.current_stream().wait_stream(stream)
    check(made, *second)
    del made
    x, scores, back = inputs(21)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x, scores, back)
    for seed in (31, 41, 51):
        new = inputs(seed)
        with torch.no_grad():
            for to, of in zip((x, scores, back), new):
                to.copy_(of)
        graph.replay()
        eager = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
        check(held, *new)


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [24, 9])
@pytest.mark.parametrize("k,weighted", [(1, False), (1, True), (2, True)])
def test_a_layer_of_routers_that_trains(k, weighted, capacity):
    """Scatter router, experts of plain torch modules on their rows, gather router: the gradients of cells, score and experts against
    autograd over a loop in 64 bits; cells without a row keep the residual."""
    from brt import Annotator, to_grid_tensor, to_torch_tensor
    from brt.router import GatherRouter, ScatterRouter

    cells, paths, d = 70, 4, 16
    scatter = ScatterRouter(protocol_type="topk", protocol_kwargs={"top_k": k}, fabric_type="fused_dispatch",
                            fabric_kwargs={"compact_route": True, "differentiable": True, "supported_capacities": capacity}).cuda()
    gather = GatherRouter(fabric_type="fused_combine", fabric_kwargs={"transform": weighted}).cuda()
    experts = [normal(10 + e, d, d).requires_grad_() for e in range(paths)]
    x = normal(1, cells, d).requires_grad_()
    score = torch.softmax(normal(2, cells, paths), 1).requires_grad_()
    residual = normal(3, cells, d).requires_grad_()
    routed = scatter(Annotator([0])(x), score)
    rows, tags, loads, extra = to_torch_tensor(routed, retrieve_attr=True)
    counts = loads[-1].tolist()
    parts = torch.split(rows, counts + [rows.shape[0] - sum(counts)])
    y = torch.cat([part @ expert for part, expert in zip(parts, experts)] + [parts[-1]])
    out = to_torch_tensor(gather(to_grid_tensor(y, tags, loads, extra), residual, score))
    back = normal(4, cells, d)
    leaves = [x, residual] + experts + ([score] if weighted else [])
    found = torch.autograd.grad(out, leaves, back)

    x64, r64, s64 = (t.detach().double().requires_grad_() for t in (x, residual, score))
    e64 = [t.detach().double().requires_grad_() for t in experts]
    top = torch.topk(score.detach(), k, dim=1).indices
    taken, want, seats = [0] * paths, [], top.tolist()
    kept = [[False] * k for _ in range(cells)]
    for t in range(cells):
        for j, e in enumerate(seats[t]):
            kept[t][j] = taken[e] < capacity
            taken[e] += 1
    for t in range(cells):
        terms = [(x64[t] @ e64[e]) * (s64[t, e] if weighted else 1.0) for j, e in enumerate(seats[t]) if kept[t][j]]
        want.append(sum(terms) if terms else r64[t])
    want = torch.stack(want) + 0 * r64  # (where every cell has a row, nothing depends on the residual)
    assert capacity == 24 or any(not any(row) for row in kept)
    wanted = torch.autograd.grad(want, [x64, r64] + e64 + ([s64] if weighted else []), back.double())
    torch.testing.assert_close(out.double(), want.detach(), rtol=1e-5, atol=2e-5)
    for a, b in zip(found, wanted):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f16")])
def test_gradients_at_any_address(dtype, out):
    """What flattens the result behind a few other values hands back a slice that starts at any element: the same gradients."""
    cells, paths, k, d = 37, 5, 2, 40
    dtype, out = TYPES[dtype], TYPES[out]
    ids, seat_rows, row_entries = make_route(cells, paths, k, 12, 1, keep=0.8)
    x, w = normal(1, cells, d, dtype=dtype).requires_grad_(), normal(2, cells, k).requires_grad_()
    y = normal(3, row_entries.numel(), d, dtype=dtype).requires_grad_()
    scores = normal(4, cells, paths, dtype=dtype).requires_grad_()
    for made, leaves in ((c_router.dispatch_by_rows(x, row_entries, k, w, seat_rows=seat_rows), [x, w]),
                         (c_router.combine_by_rows(y, ids, seat_rows, w, out_dtype=out, row_entries=row_entries), [y, w]),
                         (c_router.gate_topk(scores, k, True, differentiable=True)[1], [scores])):
        grad = normal(5, made.numel(), dtype=made.dtype)
        want = torch.autograd.grad(made, leaves, grad.view_as(made), retain_graph=True)
        for before in (1, 3):
            some = normal(6, before, dtype=made.dtype)
            long = torch.cat([some, made.reshape(-1)])
            got = torch.autograd.grad(long, leaves, torch.cat([some, grad]), retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def routed_layer(differentiable, k, weighted, capacity, x, score, residual):
    """A scatter router, experts that scale their rows and a gather router with a residual."""
    from brt import Annotator, to_grid_tensor, to_torch_tensor
    from brt.router import GatherRouter, ScatterRouter

    scatter = ScatterRouter(protocol_type="topk", protocol_kwargs={"top_k": k}, fabric_type="fused_dispatch",
                            fabric_kwargs={"compact_route": True, "differentiable": differentiable, "supported_capacities": capacity}).cuda()
    gather = GatherRouter(fabric_type="fused_combine", fabric_kwargs={"transform": weighted}).cuda()
    rows, tags, loads, extra = to_torch_tensor(scatter(Annotator([0])(x), score), retrieve_attr=True)
    return to_torch_tensor(gather(to_grid_tensor(rows * 0.75, tags, loads, extra), residual, score))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kept", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("k,weighted", [(1, False), (1, True), (2, True)])
def test_a_residual_of_another_type(k, weighted, rows, kept):
    """With or without gradients the result has the residual's type and shape, and the same bits; its gradients as the residual's."""
    cells, paths, d = 70, 4, 16
    x = normal(1, cells, d, dtype=TYPES[rows])
    score = torch.softmax(normal(2, cells, paths), 1)
    for shape in ((cells, d), (2, cells // 2, d)):
        residual = normal(3, *shape, dtype=TYPES[kept])
        want = routed_layer(False, k, weighted, 9, x, score, residual.clone())
        leaves = [x.clone().requires_grad_(), residual.clone().requires_grad_()]
        got = routed_layer(True, k, weighted, 9, leaves[0], score, leaves[1])
        assert got.dtype == residual.dtype and got.shape == want.shape and torch.equal(got, want)
        back = normal(4, *shape, dtype=TYPES[kept])
        dx, dr = torch.autograd.grad(got, leaves, back)
        bare = (want == residual).view(cells, d).all(1)
        assert bool(bare.any()) and dx.dtype == x.dtype and dr.dtype == residual.dtype
        assert torch.equal(dr.view(cells, d), torch.where(bare[:, None], back.view(cells, d), 0.0)) and not dx[bare].any() and bool(dx[~bare].any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kept", [("bf16", torch.float16), ("f16", torch.bfloat16), ("f32", torch.float64), ("bf16", torch.float64)])
def test_a_residual_of_a_type_that_the_combine_does_not_write(rows, kept):
    """The sum in fp32, rounded to the residual's type once."""
    cells, paths, d = 70, 4, 16
    x, residual = normal(1, cells, d, dtype=TYPES[rows]).requires_grad_(), normal(3, cells, d).to(kept).requires_grad_()
    score = torch.softmax(normal(2, cells, paths), 1)
    wide = routed_layer(True, 2, True, 9, x, score, residual.detach().float())
    got = routed_layer(True, 2, True, 9, x, score, residual)
    bare = (wide == residual.detach().float()).all(1, keepdim=True)
    assert got.dtype == kept and torch.equal(got, torch.where(bare, residual, wide.to(kept)))
    dx, dr = torch.autograd.grad(got.double().sum(), [x, residual])
    assert not dx[bare[:, 0]].any() and bool(dx[~bare[:, 0]].any()) and torch.equal(dr, bare.to(kept).expand(cells, d))
    with pytest.raises(NotImplementedError):
        routed_layer(True, 2, True, 9, x, score, torch.zeros(cells, d, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("differentiable", [False, True])
def test_a_residual_that_is_a_flow(differentiable):
    from brt import Annotator, to_torch_tensor

    cells, d = 70, 16
    x, score, residual = normal(1, cells, d), torch.softmax(normal(2, cells, 4), 1), normal(3, cells, d)
    want = routed_layer(False, 2, True, 9, x, score, residual.clone())
    got = routed_layer(differentiable, 2, True, 9, x, score, Annotator([0])(residual.clone()))
    assert torch.equal(to_torch_tensor(got), want)


def test_a_differentiable_fabric_needs_the_compact_route():
    from brt.router import ScatterRouter

    with pytest.raises(ValueError, match="compact_route"):
        ScatterRouter(protocol_type="topk", fabric_type="fused_dispatch", fabric_kwargs={"differentiable": True})


def test_a_differentiable_fabric_refuses_a_mask():
    """Only the decision of a top-k protocol carries gradients; a mask would cut them off without a word."""
    from brt import Annotator
    from brt.router import ScatterRouter

    kwargs = {"fabric_type": "fused_dispatch", "fabric_kwargs": {"compact_route": True, "differentiable": True}}
    x = Annotator([0])(torch.ones(4, 8, requires_grad=True))
    for protocol in ({"protocol_type": "switch_top1", "protocol_kwargs": {"one_hot": True}}, {"protocol_type": "topk"}):
        with pytest.raises(NotImplementedError, match="topk protocol"):
            ScatterRouter(**protocol, **kwargs)(x, torch.eye(4))  # (a score on the host: the protocol gives a mask)


@pytest.mark.gpu
def test_a_mask_goes_through_where_no_gradient_is_wanted():
    from brt import Annotator, to_torch_tensor
    from brt.router import ScatterRouter

    x, mask = normal(1, 6, 8), torch.eye(6, 3, device="cuda")
    made = []
    with torch.no_grad():
        for differentiable in (False, True):
            scatter = ScatterRouter(protocol_type="switch_top1", fabric_type="fused_dispatch",
                                    fabric_kwargs={"compact_route": True, "differentiable": differentiable}).cuda()
            made.append(to_torch_tensor(scatter(Annotator([0])(x), mask)))
    assert torch.equal(*made)


@pytest.mark.gpu
def test_rows_without_their_route_are_refused():
    """An expert that drops the extra attributes, or names other loads: the combine would cut the gradients off."""
    from brt import Annotator, to_grid_tensor, to_torch_tensor
    from brt.router import GatherRouter, ScatterRouter

    x, score = normal(1, 12, 8).requires_grad_(), torch.softmax(normal(2, 12, 3), 1)
    scatter = ScatterRouter(protocol_type="topk", fabric_type="fused_dispatch",
                            fabric_kwargs={"compact_route": True, "differentiable": True}).cuda()
    gather = GatherRouter(fabric_type="fused_combine").cuda()

    def rows():
        return to_torch_tensor(scatter(Annotator([0])(x), score), retrieve_attr=True)

    data, tags, loads, extra = rows()
    with pytest.raises(RuntimeError, match="without their route"):
        gather(to_grid_tensor(data, tags, loads, None))
    data, tags, loads, extra = rows()
    with pytest.raises(RuntimeError, match="without their route"):
        gather(to_grid_tensor(data, tags, loads[:-1] + [loads[-1].clone()], extra))
    with torch.no_grad():
        data, tags, loads, extra = rows()
        assert torch.equal(to_torch_tensor(gather(to_grid_tensor(data, tags, loads, None))), x)
        data, tags, loads, extra = rows()
        assert torch.equal(to_torch_tensor(gather(to_grid_tensor(data, tags, loads[:-1] + [loads[-1].clone()], extra))), x)
    data, tags, loads, extra = rows()
    (dx,) = torch.autograd.grad(to_torch_tensor(gather(to_grid_tensor(data, tags, loads, extra))).sum(), x)
    assert torch.equal(dx, torch.ones_like(x))

"""The router's losses and their gradient against the formulas in 64 bits, against differences, and their refusals.

Tolerances, in steps of u = 2^-24 (half a step of fp32).  x = s - max is off by u of itself, its product with log2(e) by 2 u more (constant and
rounding), exp2 by 2 u: an exponential is within (3 |x| + 2) u of itself.  The sum of E of them is within E u of its terms' errors, which
weighted by the terms are at most 3 * 0.37 E + 2 (|x| exp(-|x|) <= 0.37): 2.2 E + 2 in all, so p is within (3 |x| + 2.2 E + 8) u of
itself.  A column's sum in a workgroup adds at most the rows of that workgroup (T / blocks), then eight wavefronts and six exchanges; the
rest is fp64.  A term of z is lse^2, lse off by (2.2 E + 2) u from the sum, 2 u |log| and u |lse| from the addition.  A gradient p (c -
sum c p + q lse) is within the errors of its p twice, of E additions and of lse, relative to p (c + sum c p + |q lse|); its last rounding
is half a step of the type (``torch.finfo(t).eps / 2``).
"""
import pytest
import torch

import brt._C.router as c_router
from brainstorm_amd import _lib

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def normal(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def some_ids(seed, cells, paths, k, keep=1.0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, paths, (cells, k), generator=gen).int()
    return torch.where(torch.rand(cells, k, generator=gen) < keep, ids, -1).int().cuda()


def some_cells(seed, cells, share):
    return (torch.rand(cells, generator=torch.Generator().manual_seed(seed)) < share).cuda()


def in_64_bits(scores, ids, counted=None):
    """(balance, z, counts) with the gradient of the scores left to autograd over plain operations."""
    cells, paths = scores.shape
    counted = torch.ones(cells, dtype=torch.bool, device=scores.device) if counted is None else counted
    chosen = ids[counted].long()
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < paths)], minlength=paths)
    part, n = scores[counted], int(counted.sum())
    if n == 0 or ids.shape[1] == 0:
        balance = scores.new_zeros(())
    else:
        balance = paths / (n * n * ids.shape[1]) * (counts * torch.softmax(part, 1).sum(0)).sum()
    z = torch.logsumexp(part, 1).square().mean() if n else scores.new_zeros(())
    return balance, z, counts.int()


def spread(scores):
    s = scores.detach().double()
    return float((s.amax(1) - s.amin(1)).max()) if s.numel() else 0.0


def assert_losses(made, scores, ids, counted=None):
    cells, paths = scores.shape
    balance, z, counts = (t.detach() for t in made)
    want = in_64_bits(scores.detach().double(), ids, counted)
    assert counts.dtype == torch.int32 and torch.equal(counts, want[2])
    assert balance.dtype == z.dtype == torch.float32 and balance.shape == z.shape == ()
    rows = cells if cells * paths <= 1 << 15 else -(-cells // min(256, -(-cells * paths >> 11)))
    steps = 3 * spread(scores) + 2.2 * paths + 8 + rows + 16
    assert abs(float(balance) - float(want[0])) <= (steps * U + U) * float(want[0])
    part = scores.detach().double() if counted is None else scores.detach().double()[counted]
    if part.numel():
        lse = torch.logsumexp(part, 1).abs()
        off = (2.2 * paths + 4) * U + 3 * U * lse + U * part.abs().amax(1)
        assert abs(float(z) - float(want[1])) <= float((2 * lse * off + off * off).mean()) + (rows + 16) * U * float(want[1])
    else:
        assert float(z) == 0.0


def assert_gradient(got, scores, ids, counted, by):
    cells, paths = scores.shape
    s = scores.detach().double().requires_grad_()
    balance, z, counts = in_64_bits(s, ids, counted)
    total = by[0] * balance + by[1] * z
    want = torch.autograd.grad(total, s)[0] if total.requires_grad else torch.zeros_like(s)
    use = torch.ones(cells, dtype=torch.bool, device=s.device) if counted is None else counted
    n = max(1, int(use.sum()))
    p, lse = torch.softmax(s.detach(), 1), torch.logsumexp(s.detach(), 1, keepdim=True)
    c = abs(by[0]) * paths / (n * n * max(1, ids.shape[1])) * counts.double()
    size = p * (c + (c * p).sum(1, keepdim=True) + abs(by[1]) * 2 / n * lse.abs())
    steps = 2 * (3 * spread(scores) + 2.2 * paths + 8) + paths + 10
    info = torch.finfo(got.dtype)
    z_off = p * abs(by[1]) * 2 / n * ((2.2 * paths + 4) * U + U * s.detach().abs().amax(1, keepdim=True))
    off = steps * U * size + z_off
    bound = off + info.eps / 2 * (want.abs() + off) + info.tiny * info.eps
    assert got.dtype == scores.dtype and got.shape == scores.shape
    assert not got[~use].any()
    far = ((got.double() - want).abs() / bound)[use]
    assert not far.numel() or float(far.max()) <= 1.0, f"{float(far.max())} of the bound"


SHAPES = [  # cells, paths, k
    (1, 1, 1), (1, 4, 4), (2, 3, 2), (5, 8, 1), (63, 12, 2), (64, 64, 2), (257, 60, 4), (1024, 16, 1), (1025, 16, 1), (999, 100, 2), (130, 128, 8),
    (70, 160, 2), (300, 256, 2), (41, 257, 3), (33, 513, 1), (17, 1000, 8), (65, 1024, 2), (4099, 60, 4), (9000, 128, 2), (20000, 6, 1), (70000, 8, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cells,paths,k", SHAPES)
def test_losses_and_gradient(cells, paths, k, dtype):
    scores = (2 * normal(cells + paths, cells, paths)).to(TYPES[dtype]).requires_grad_()
    for share, keep in ((None, 1.0), (0.7, 0.9)):
        ids = some_ids(k, cells, paths, k, keep)
        counted = None if share is None else some_cells(2, cells, share)
        made = c_router.balance_loss(scores, ids, counted)
        assert made[0].requires_grad and made[1].requires_grad and not made[2].requires_grad
        assert_losses(made, scores, ids, counted)
        by = (float(cells * paths), 0.25 * cells)  # (gradients of about one, so that fp16 holds them)
        grads = [torch.tensor(v, device="cuda") for v in by]
        (got,) = torch.autograd.grad(made[:2], scores, grads)
        assert_gradient(got, scores, ids, counted, by)
        plain = c_router.balance_loss(scores.detach(), ids, counted)
        assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(made, plain))


@pytest.mark.gpu
def test_an_even_router_has_a_balance_of_one():
    cells, paths, k = 512, 8, 2
    ids = torch.stack([torch.arange(cells) % paths, (torch.arange(cells) + 3) % paths], 1).int().cuda()
    balance, z, counts = c_router.balance_loss(torch.zeros(cells, paths, device="cuda"), ids)
    assert abs(float(balance) - 1.0) <= 2.0 ** -22 and counts.tolist() == [cells * k // paths] * paths
    assert abs(float(z) - float(torch.tensor(8.0).double().log()) ** 2) <= 1e-6


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the losses in fp32 with steps of 2^-4: off by h^2 / 6 times a third derivative (each derivative of a softmax's
    product with c is at most c's spread times 2, of lse^2 at most 8 (1 + |lse|)) and by the losses' own error over the step."""
    cells, paths, k, h = 3, 5, 2, 2.0 ** -4
    scores, ids = normal(1, cells, paths), some_ids(2, cells, paths, k)
    for which in (0, 1):
        leaf = scores.clone().requires_grad_()
        (got,) = torch.autograd.grad(c_router.balance_loss(leaf, ids)[which], leaf)
        for t in range(cells):
            for e in range(paths):
                moved = []
                for step in (h, -h):
                    other = scores.clone()
                    other[t, e] += step
                    moved.append(float(c_router.balance_loss(other, ids)[which]))
                limit = h * h / 6 * (2 * paths if which == 0 else 8 * (1 + 4)) + 2.0 ** -18 / h
                assert abs((moved[0] - moved[1]) / (2 * h) - float(got[t, e])) <= limit


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cells,paths", [(40, 40), (3000, 64), (40, 7)])
def test_masked_scores(cells, paths, dtype):
    """Scores of -inf and of the type's lowest value have no probability and no gradient; a row of nothing but the lowest value has an
    even softmax."""
    dtype = TYPES[dtype]
    scores = normal(1, cells, paths, dtype=dtype)
    scores[0, 3:], scores[1, ::2] = float("-inf"), torch.finfo(dtype).min
    ids = some_ids(2, cells, paths, 2)
    leaf = scores.clone().requires_grad_()
    balance, z, counts = c_router.balance_loss(leaf, ids)
    want = in_64_bits(scores.double(), ids)
    assert abs(float(balance) - float(want[0])) <= 1e-4 * float(want[0]) and abs(float(z) - float(want[1])) <= 1e-4 * float(want[1])
    (got,) = torch.autograd.grad(1e3 * balance + 1e3 * z, leaf)
    assert torch.isfinite(got).all() and not got[0, 3:].any() and not got[1, ::2].any()
    scores[2] = torch.finfo(dtype).min
    leaf = scores.clone().requires_grad_()
    balance, z, counts = c_router.balance_loss(leaf, ids)
    want = in_64_bits(scores.double(), ids)
    assert abs(float(balance) - float(want[0])) <= 1e-4 * float(want[0])
    (got,) = torch.autograd.grad(1e4 * balance, leaf)
    assert torch.isfinite(got).all()
    c = 1e4 * paths / (cells * cells * 2) * counts.double()
    row = (c - c.mean()) / paths
    assert float((got[2].double() - row).abs().max()) <= 1e-5 * float(c.max()) + torch.finfo(dtype).eps * float(row.abs().max())


@pytest.mark.gpu
def test_cells_that_do_not_count_are_not_looked_at():
    """NaN and infinities in them reach neither a loss nor a gradient, and their ids are not counted."""
    for cells, paths in ((50, 8), (4000, 60)):
        scores, ids, counted = normal(1, cells, paths), some_ids(2, cells, paths, 2), some_cells(3, cells, 0.5)
        given = scores.clone()
        given[~counted] = float("nan")
        given[torch.nonzero(~counted)[0, 0]] = float("inf")
        strange = ids.clone()
        strange[~counted] = 1 << 30
        made = []
        for s, i in ((scores, ids), (given, strange)):
            leaf = s.clone().requires_grad_()
            losses = c_router.balance_loss(leaf, i, counted)
            made.append([t.detach() for t in losses] + list(torch.autograd.grad(losses[:2], leaf, [torch.tensor(2.0, device="cuda")] * 2)))
        assert all(torch.equal(a, b) for a, b in zip(*made))
        assert_losses(made[0][:3], scores, ids, counted)


@pytest.mark.gpu
def test_rows_that_are_not_finite():
    """A counted cell with NaN, with +inf or without a score above -inf makes the losses NaN, as its softmax is; other rows keep their gradients."""
    scores, ids = normal(1, 60, 8), some_ids(2, 60, 8, 1)
    sound = scores.clone().requires_grad_()
    (want,) = torch.autograd.grad(c_router.balance_loss(sound, ids)[0], sound)
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = scores.clone()
        if value == float("-inf"):
            bad[7] = value
        else:
            bad[7, 3] = value
        bad.requires_grad_()
        balance, z, counts = c_router.balance_loss(bad, ids)
        assert balance.isnan() and z.isnan() and int(counts.sum()) == 60
        (got,) = torch.autograd.grad(balance, bad)
        rows = torch.arange(60, device="cuda") != 7
        assert got[7].isnan().all() and torch.equal(got[rows], want[rows])


@pytest.mark.gpu
def test_nothing_that_counts():
    ids = some_ids(1, 30, 6, 2)
    for scores, chosen, counted in ((normal(1, 30, 6), ids, torch.zeros(30, dtype=torch.bool, device="cuda")),
                                    (torch.zeros(0, 6, device="cuda"), ids[:0], None),
                                    (torch.zeros(0, 6, device="cuda"), ids[:0], torch.zeros(0, dtype=torch.bool, device="cuda"))):
        leaf = scores.clone().requires_grad_()
        balance, z, counts = c_router.balance_loss(leaf, chosen, counted)
        assert float(balance) == 0.0 and float(z) == 0.0 and not counts.any()
        (got,) = torch.autograd.grad(balance + z, leaf)
        assert got.shape == leaf.shape and not got.any()
    leaf = normal(1, 30, 6).requires_grad_()
    for none in (ids[:, :0], torch.full_like(ids, -1)):
        balance, z, counts = c_router.balance_loss(leaf, none)
        assert float(balance) == 0.0 and float(z) > 0.0 and not counts.any()
        assert not torch.autograd.grad(balance, leaf, retain_graph=True)[0].any()


@pytest.mark.gpu
def test_a_path_named_twice_counts_twice():
    ids = torch.tensor([[1, 1], [0, 1]], dtype=torch.int32, device="cuda")
    scores = normal(1, 2, 4)
    made = c_router.balance_loss(scores, ids)
    assert made[2].tolist() == [1, 3, 0, 0]
    assert_losses(made, scores, ids)


@pytest.mark.gpu
def test_one_loss_alone_and_the_gradients_of_both_added():
    scores, ids = normal(1, 100, 16).requires_grad_(), some_ids(2, 100, 16, 2)
    for by in ((3.0, 0.0), (0.0, 2.0), (3.0, 2.0)):
        balance, z, _ = c_router.balance_loss(scores, ids)
        (got,) = torch.autograd.grad((by[0] * balance if by[0] else 0.0) + (by[1] * z if by[1] else 0.0), scores)
        assert_gradient(got, scores, ids, None, by)
    with torch.no_grad():
        assert not c_router.balance_loss(scores, ids)[0].requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("paths", [16, 60, 61])
def test_strides_and_addresses(paths):
    cells = 120
    base = normal(1, 2 * cells, paths + 3)
    ids, counted = some_ids(2, cells, paths, 2), some_cells(3, 2 * cells, 0.8)
    views = [base[::2, 1:paths + 1], base.t()[:paths].t()[cells:], base.view(-1)[1:1 + cells * paths].view(cells, paths), base[:1, :paths].expand(cells, paths)]
    for view in views:
        leaf = view.detach().requires_grad_()
        for mask in (None, counted[::2]):
            for chosen in (ids, ids.t().contiguous().t()):
                made = c_router.balance_loss(leaf, chosen, mask)
                assert_losses(made, view, ids, mask)
                (got,) = torch.autograd.grad(made[:2], leaf, [torch.tensor(100.0, device="cuda").expand(()), torch.tensor([0.0, 3.0], device="cuda")[1]])
                assert_gradient(got, view, ids, mask, (100.0, 3.0))


@pytest.mark.gpu
def test_the_same_bits_every_time_and_a_gradient_of_its_own():
    """Two calls agree; what is written to the counts afterwards changes no gradient; writing to the scores is an error."""
    scores, ids = normal(1, 5000, 64).requires_grad_(), some_ids(2, 5000, 64, 2)
    balance, z, counts = c_router.balance_loss(scores, ids)
    (want,) = torch.autograd.grad([balance, z], scores, [torch.ones((), device="cuda")] * 2)
    again = c_router.balance_loss(scores, ids)
    again[2].zero_()
    (got,) = torch.autograd.grad(list(again[:2]), scores, [torch.ones((), device="cuda")] * 2)
    assert torch.equal(balance, again[0]) and torch.equal(z, again[1]) and torch.equal(got, want)
    for change in ("scores", "counted"):
        held, mask = scores * 1, torch.ones(5000, dtype=torch.bool, device="cuda")
        balance, _, _ = c_router.balance_loss(held, ids, mask)
        with torch.no_grad():
            (held if change == "scores" else mask).zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            balance.backward()


@pytest.mark.gpu
def test_gradients_of_the_gradient_and_tangents_raise():
    scores, ids = normal(1, 20, 8).requires_grad_(), some_ids(2, 20, 8, 1)
    balance, z, _ = c_router.balance_loss(scores, ids)
    (got,) = torch.autograd.grad(balance, scores, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        got.sum().backward()
    import torch.autograd.forward_ad as forward

    with forward.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            c_router.balance_loss(forward.make_dual(scores.detach(), torch.ones_like(scores)), ids)


@pytest.mark.gpu
def test_a_step_on_a_stream_and_two_graphs_replayed_in_turn():
    """Gate, losses and their gradient: on a stream of its own, and captured twice with other sizes, replayed in turn for other inputs."""
    def step(scores):
        ids, weights = c_router.gate_topk(scores, 2, True, differentiable=True)
        balance, z, counts = c_router.balance_loss(scores, ids)
        (got,) = torch.autograd.grad(weights.sum() + balance + z, scores)
        return ids, balance.detach(), z.detach(), counts, got

    sizes = [(64, 8), (6000, 32)]
    for cells, paths in sizes:
        step(normal(1, cells, paths).requires_grad_())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        scores = normal(3, 6000, 32).requires_grad_()
        made = step(scores)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(made, step(normal(3, 6000, 32).requires_grad_())))
    del made, scores
    held = []
    for cells, paths in sizes:
        scores = normal(1, cells, paths).requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = step(scores)
        held.append((graph, scores, made))
    for seed in (31, 41, 51):
        for graph, scores, made in held:
            new = normal(seed, *scores.shape).requires_grad_()
            with torch.no_grad():
                scores.copy_(new)
            graph.replay()
            eager = step(new)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(made, eager))


@pytest.mark.gpu
def test_scores_beyond_four_gib():
    """2^31 - 64 fp32 scores: the last rows and their gradient lie past 2^33 bytes."""
    paths = 64
    cells = (1 << 31) // paths - 1
    scores = torch.zeros(cells, paths, device="cuda")
    scores[-40:] = normal(1, 40, paths)
    ids = torch.zeros(cells, 1, dtype=torch.int32, device="cuda")
    ids[-40:] = some_ids(2, 40, paths, 1)
    scores.requires_grad_()
    balance, z, counts = c_router.balance_loss(scores, ids)
    (got,) = torch.autograd.grad([balance, z], scores, [torch.tensor(1e9, device="cuda"), torch.tensor(1e9, device="cuda")])
    assert torch.equal(counts, torch.bincount(ids.view(-1), minlength=paths).int())
    s = torch.cat([scores.detach()[:1], scores.detach()[-40:]]).double()
    p, lse, c = torch.softmax(s, 1), torch.logsumexp(s, 1, keepdim=True), paths / cells ** 2 * counts.double()
    share = (cells - 40) * p[:1].sum(0) + p[1:].sum(0)
    squares = (cells - 40) * float(lse[0] ** 2) + float((lse[1:] ** 2).sum())
    # a workgroup's 131072 rows are added up in fp32, 2048 of them one behind the other in a lane; the other terms as above
    off = (2048 + 3 * spread(s) + 2 * 2.2 * paths + 40) * U
    assert abs(float(balance.detach()) - float((c * share).sum())) <= off * float((c * share).sum())
    assert abs(float(z.detach()) - squares / cells) <= off * squares / cells
    for at, row in ((0, 0), (cells // 2, 0), (cells - 41, 0), *((cells - 40 + i, 1 + i) for i in range(40))):
        want = 1e9 * p[row] * (c - (c * p[row]).sum() + 2 / cells * lse[row])
        size = 1e9 * p[row] * (c + (c * p[row]).sum() + 2 / cells * lse[row])
        assert bool(((got[at].double() - want).abs() <= (3 * spread(s) + 2.2 * paths + 20) * 4 * U * size).all()), at


@pytest.mark.gpu
def test_two_calls_at_once():
    def step(scores, ids):
        balance, z, counts = c_router.balance_loss(scores, ids)
        return [balance.detach(), z.detach(), counts, *torch.autograd.grad(balance + z, scores)]

    inputs = [(normal(i, 20000, 64).requires_grad_(), some_ids(10 + i, 20000, 64, 2)) for i in range(2)]
    want = [step(*these) for these in inputs]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*inputs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for made in got[i] for a, b in zip(made, want[i]))


@pytest.mark.gpu
def test_refusals():
    scores, ids = normal(1, 20, 8), some_ids(2, 20, 8, 2)
    mask = torch.ones(20, dtype=torch.bool, device="cuda")
    for call, error, words in (
            (lambda: c_router.balance_loss(scores, ids.long()), RuntimeError, "int32"),
            (lambda: c_router.balance_loss(scores, ids[:-1]), RuntimeError, r"\[cells, k\]"),
            (lambda: c_router.balance_loss(scores, ids[:, 0]), RuntimeError, r"\[cells, k\]"),
            (lambda: c_router.balance_loss(scores[0], ids), RuntimeError, r"\[cells, paths\]"),
            (lambda: c_router.balance_loss(scores.double(), ids), NotImplementedError, "score data type"),
            (lambda: c_router.balance_loss(scores, ids, mask.int()), RuntimeError, "bool"),
            (lambda: c_router.balance_loss(scores, ids, mask[:-1]), RuntimeError, "bool"),
            (lambda: c_router.balance_loss(scores, ids, mask.cpu()), RuntimeError, "another device"),
            (lambda: c_router.balance_loss(scores, ids.cpu()), RuntimeError, "CUDA tensor"),
            (lambda: c_router.balance_loss(normal(1, 4, 1025), ids[:4]), NotImplementedError, "1024"),
            (lambda: c_router.balance_loss(scores[:, :0], ids), RuntimeError, "bad shape")):
        with pytest.raises(error, match=words):
            call()


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_router.balance_loss(torch.zeros(4, 4), torch.zeros(4, 1, dtype=torch.int32))


def test_argument_errors_of_the_library_need_no_gpu():
    lib = _lib.lib()
    call, grad, size = lib.brt_hip_balance_loss, lib.brt_hip_balance_loss_grad, lib.brt_hip_balance_loss_workspace_bytes
    some = 16  # an address that is never read: every call ends before a launch
    assert call(some, some, None, some, some, some, None, None, -1, 4, 1, 0, None, 0, None) == -1
    assert call(some, some, None, some, some, some, None, None, 4, 0, 1, 0, None, 0, None) == -1
    assert call(some, some, None, some, some, some, None, None, 4, 4, 1, 7, None, 0, None) == -4
    assert call(some, some, None, some, some, some, None, None, 4, 1025, 1, 0, None, 0, None) == -4
    assert call(some, some, None, some, some, some, None, None, 1 << 26, 64, 1, 0, None, 0, None) == -4
    assert call(some, some, None, some, some, some, None, None, 1 << 26, 4, 64, 0, None, 0, None) == -4
    assert call(None, some, None, some, some, some, None, None, 4, 4, 1, 0, None, 0, None) == -1
    assert call(some, some, None, some, some, some, some + 4, None, 4, 4, 1, 0, None, 0, None) == -4
    assert call(some, some, None, some, some, some, None, None, 65536, 64, 2, 0, None, 0, None) == -2
    assert call(some, some, None, some, some, some, None, None, 65536, 64, 2, 0, some, size(65536, 64) - 1, None) == -2
    assert grad(some, None, some, some, None, None, None, 4, 4, 0, None) == -1
    assert grad(some, None, some, some, None, None, some, 4, 1025, 0, None) == -4
    assert grad(some, None, some + 4, some, None, None, some, 4, 4, 0, None) == -4
    assert size(4, 4) == size(0, 4) == size(4, 0) == 0 and 0 < size(65536, 128) <= 256 * 129 * 8

"""Every kernel of the products with 4-bit weights at the values, loads and layouts where it can go wrong, against the definition in 64 bits.

Bounds as in ``test_int4`` (``assert_near``), and what is left of them where numbers are tiny: the third part of an fp32 element is a multiple of
2^-133, so the element is off by at most 2^-134; sums and their products with scales are held in units of 2^-15 with the fp32 grid's 2^-149, so an
addition to a result is off by at most 2^-135 beside its relative error.
"""
import pytest
import torch

import brt._C.router as c_router
from brainstorm_amd import _lib
from brt.jit import Int4Weight, grouped_linear_int4, pack_int4
from test_int4 import TYPES, Weights, assert_near, loads_of, normal, product_in_64

CODES = {"f32": 0, "f16": 1, "bf16": 2}


def columns_of(dtype, rows, k, n, experts, group, cells=-1):
    """Columns of the tiles that take these sizes, 16 for the kernel of few rows."""
    return _lib.lib().brt_hip_grouped_gemm_int4_kernel(CODES[dtype], cells, group, experts, rows, n, k)


def rescaled(w, by, zeros=None):
    """The weights with other scales (fp32) and, given some, zero points."""
    w.s = w.s.float() * by
    w.z = w.z if zeros is None else zeros
    w.packed = pack_int4(w.q, w.s, w.z, group=w.group)
    return w


#: columns of the tiles; rows, in, out, experts, group
EACH = [(16, 20, 264, 48, 2, 64), (16, 70, 256, 100, 2, 128), (16, 33, 200, 40, 3, 32), (128, 700, 256, 2048, 3, 32), (128, 1300, 264, 1300, 2, 64),
        (128, 900, 256, 1300, 2, 128), (256, 2100, 256, 2048, 3, 32), (256, 3300, 264, 1300, 2, 64), (256, 3100, 256, 1300, 2, 128)]


def by_kernel(dtypes=tuple(TYPES)):
    """(dtype, rows, in, out, experts, group): every shape for 16-bit rows, those of few rows for fp32 ones too."""
    return [(dtype, *shape) for columns, *shape in EACH for dtype in dtypes if dtype != "f32" or columns == 16]


def test_the_shapes_below_reach_every_kernel():
    for columns, *shape in EACH:
        assert columns_of("bf16", *shape) == columns_of("f16", *shape) == columns_of("f16", *shape, cells=shape[0]) == columns, shape


@pytest.mark.gpu
@pytest.mark.parametrize("zero", [None, 0, 255])
@pytest.mark.parametrize("dtype,rows,k,n,experts,group", by_kernel(("f32", "bf16")))
def test_large_elements(dtype, rows, k, n, experts, group, zero):
    """Sums that leave the range of fp32 before the scale, and results that do not: neither infinities nor NaN, whatever the order of the sums."""
    w = Weights(rows, experts, n, k, group, zeros=zero is None)
    rescaled(w, 2.0 ** -4 if zero == 255 else 1.0, None if zero is None else torch.full(w.s.shape, zero, dtype=torch.uint8))
    largest = 3.3e38 / 64
    x = (torch.rand(rows, k, generator=torch.Generator().manual_seed(1)) * 2 - 1) * largest
    x[::3] = x[::3].abs()
    x[1::7] = largest
    x, loads = x.to(TYPES[dtype]), loads_of(rows, rows, experts)
    for activation in ("none", "relu"):
        want, size = product_in_64(x, w, loads, activation=activation)
        assert float(want.abs().max()) < 3.3e38
        got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), out_dtype=torch.float32, activation=activation)
        assert bool(got.isfinite().all())
        assert_near(got, want, size, group, k)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0, 60])
@pytest.mark.parametrize("exponent", [-90, -108, -116, -122])
@pytest.mark.parametrize("dtype,rows,k,n,experts,group", by_kernel(("f32", "bf16")))
def test_tiny_elements(dtype, rows, k, n, experts, group, exponent, scale):
    """Elements down to the smallest: what is lost is known, and far below the results (zeros in their place are seen)."""
    w = rescaled(Weights(rows, experts, n, k, group, zeros=True), 2.0 ** (scale + 7))
    x, loads = normal(1, rows, k, scale=2.0 ** exponent, dtype=TYPES[dtype]), loads_of(rows, rows, experts)
    (want, size), (_, steps) = product_in_64(x, w, loads), product_in_64(torch.ones(rows, k), w, loads)
    off = (6 * group + -(-k // group) + 20) * 2.0 ** -23 * size + (steps * 2.0 ** -134 if dtype == "f32" else 0.0) + (-(-k // group) + 20) * 2.0 ** -135
    bound = off + 2.0 ** -24 * want.abs() + 2.0 ** -150
    got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), out_dtype=torch.float32).cpu()
    assert float(bound.square().mean().sqrt()) <= 0.1 * float(want.square().mean().sqrt())
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n,experts,group", [shape[1:] for shape in by_kernel(("f16",))])
def test_subnormal_elements_of_fp16(rows, k, n, experts, group):
    w = Weights(rows, experts, n, k, group, zeros=True)
    x, loads = normal(1, rows, k, scale=2.0 ** -20, dtype=torch.float16), loads_of(rows, rows, experts)
    want, size = product_in_64(x, w, loads)
    assert bool((x.abs() < 2.0 ** -14).all()) and bool((x != 0).any())
    assert_near(grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), out_dtype=torch.float32), want, size, group, k)


# ------------------------------------------------------------------------------- the kernel of few rows
#: 100 times the 16 columns of a workgroup plus its wavefronts; rows, in, out, experts
FORMS = [(116, 20, 4104, 100, 2), (108, 70, 1096, 520, 4), (208, 24, 1032, 1001, 8), (204, 20, 600, 500, 16), (202, 300, 264, 520, 5),
         (408, 130, 1032, 1300, 2), (404, 333, 776, 1001, 12), (402, 60, 904, 2100, 40)]


def test_the_forms_below_are_reached():
    form = _lib.lib().brt_hip_grouped_gemm_int4_few_rows
    assert form(3, 1, 1, 1, 1) == form(2, 0, 1, 1, 1) == form(2, 1, 0, 1, 1) == form(2, 1, 1, 0, 1) == form(2, 1, 1, 1, 0) == -1
    for which, rows, k, n, experts in FORMS:
        assert all(form(code, experts, rows, n, k) == which for code in CODES.values())
        assert all(columns_of(dtype, rows, k, n, experts, group) == 16 for dtype in TYPES for group in (32, 64, 128))
    # one row block to an expert: 32 columns a workgroup for 16-bit rows, 64 for fp32 ones, which every workgroup splits anew
    for rows, k, n, experts, by16, by32 in ((24, 1792, 8192, 4, 204, 408), (72, 768, 512, 24, 204, 404), (16, 3584, 1000, 16, 208, 408)):
        assert [form(code, experts, rows, n, k) for code in (2, 1, 0)] == [by16, by16, by32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("group,zeros,scales", [(32, False, "f16"), (32, True, "f32"), (64, True, "bf16"), (128, False, "f32"), (128, True, "f16")])
@pytest.mark.parametrize("form,rows,k,n,experts", FORMS)
def test_products_of_every_form_for_few_rows(form, rows, k, n, experts, group, zeros, scales, dtype):
    w = Weights(form, experts, n, k, group, zeros, scale_dtype=TYPES[scales])
    x, loads = normal(1, rows, k, dtype=TYPES[dtype]), loads_of(rows, rows, experts, empty=(1,) if experts > 2 else ())
    bias = normal(2, experts, n)
    for given, out, activation in ((None, TYPES[dtype], "none"), (bias, torch.float32, "gelu"), (bias, TYPES[dtype], "relu")):
        got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), bias=None if given is None else given.cuda(), activation=activation, out_dtype=out)
        want, size = product_in_64(x, w, loads, given, activation)
        assert_near(got, want, size, group, k, gelu=activation == "gelu")


# ------------------------------------------------------------------------------------------- the tiles
#: columns of the tiles; rows, in, out, experts, group
TILES = [(128, 1300, 264, 1300, 4, 32), (128, 1300, 264, 1300, 4, 64), (128, 600, 256, 2048, 4, 128), (256, 3000, 264, 1300, 4, 32),
         (256, 3000, 264, 1300, 4, 64), (256, 3000, 256, 2048, 4, 128)]


def test_the_tiles_below_are_reached():
    for columns, *shape in TILES:
        assert columns_of("bf16", *shape) == columns_of("f16", *shape, cells=shape[0]) == columns, shape


@pytest.mark.gpu
@pytest.mark.parametrize("columns,rows,k,n,experts,group", TILES)
def test_loads_that_do_not_fill_the_rows_of_tiles(columns, rows, k, n, experts, group):
    """Rows behind the last expert's are left as they were; loads below zero count as none; rows behind the last of x do not exist."""
    w, x = Weights(1, experts, n, k, group), normal(2, rows, k, dtype=torch.bfloat16)
    on = w.cuda()
    for given in ([3, 0, rows // 2, 5], [-7, 64, -1, 65], [0, 0, 0, 0], [rows - 5, 100, 7, 9], [0, 2000000000, 2000000000, 1], [rows] * 4, [-(1 << 31), rows - 63, 0, 62]):
        taken, left = [], rows
        for load in given:
            taken.append(max(0, min(load, left)))
            left -= taken[-1]
        out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
        got = grouped_linear_int4(x.cuda(), on, torch.tensor(given, dtype=torch.int32, device="cuda"), out=out)
        want, size = product_in_64(x, w, torch.tensor(taken))
        assert_near(got, want, size, group, k)
        assert bool((got[rows - left:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("columns,rows,k,n,experts,group", TILES)
def test_a_row_of_its_own_in_tiles(columns, rows, k, n, experts, group, dtype, zeros):
    """A row's result does not depend on what the others hold; one that holds NaN or an infinity gives NaN behind an activation too."""
    w, loads = Weights(1, experts, n, k, group, zeros=zeros), loads_of(2, rows, experts)
    on = w.cuda()
    x = normal(3, rows, k, dtype=TYPES[dtype])
    bad = x.clone()
    bad[0, 5], bad[70, k - 1], bad[rows - 1, 100], bad[131, 140] = float("nan"), float("inf"), float("-inf"), float("nan")
    sound = torch.isfinite(bad).all(1)
    for activation in ("none", "relu", "gelu"):
        alone, got = (grouped_linear_int4(t.cuda(), on, loads.cuda(), activation=activation).cpu() for t in (x, bad))
        assert torch.equal(got[sound], alone[sound]) and got[~sound].isnan().all()
        want, size = product_in_64(x, w, loads, activation=activation)
        assert_near(alone, want, size, group, k, gelu=activation == "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("columns,rows,k,n,experts,group", TILES)
def test_entries_that_name_no_cell_in_tiles(columns, rows, k, n, experts, group):
    w, loads, bias = Weights(1, experts, n, k, group, zeros=True).cuda(), loads_of(2, rows, experts).cuda(), normal(3, experts, n).cuda()
    cells = rows // 3
    x = normal(4, cells, k, dtype=torch.bfloat16).cuda()
    for per_cell in (1, 3):
        entries = torch.randint(1, cells * per_cell + 1, (rows,), generator=torch.Generator().manual_seed(5))
        entries[::11], entries[1::13], entries[2::17], entries[3::19], entries[4::23] = 0, -1, -(1 << 31), (1 << 31) - 1, cells * per_cell + 1
        there = (entries >= 1) & (entries <= cells * per_cell)
        packed = torch.where(there.cuda()[:, None], x[((entries - 1) // per_cell).clamp(0, cells - 1).cuda()], 0)
        want = grouped_linear_int4(packed, w, loads, bias=bias)
        got = grouped_linear_int4(x, w, loads, bias=bias, row_entries=entries.int().cuda(), entries_per_cell=per_cell)
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("columns,rows", [(128, 900), (256, 3100)])
def test_strides_and_addresses_in_tiles(columns, rows):
    k, n, experts, group = 256, 1300, 2, 128
    assert columns_of("bf16", rows, k, n, experts, group) == columns
    w, loads = Weights(1, experts, n, k, group, zeros=True), loads_of(2, rows, experts).cuda()
    base = normal(3, rows * 2, k + 8, dtype=torch.bfloat16).cuda()
    bias = normal(4, n, experts).t()
    packed = w.cuda()
    shifted = torch.empty(packed.values.numel() + 3, dtype=torch.uint8, device="cuda")[3:].view(packed.values.shape)
    shifted.copy_(packed.values)
    other = packed._replace(values=shifted, scales=packed.scales.transpose(0, 1).contiguous().transpose(0, 1), zeros=packed.zeros.clone())
    views = (base[::2, :k], base[:rows, 3:k + 3], base[:rows].reshape(-1)[1:1 + rows * k].view(rows, k), base[:1, :k].expand(rows, k))
    for dtype in (torch.bfloat16, torch.float32):
        for x in views:
            want = grouped_linear_int4(x.contiguous().clone(), packed, loads, bias=bias.contiguous().cuda(), out_dtype=dtype)
            assert torch.equal(grouped_linear_int4(x, other, loads, bias=bias.cuda(), out_dtype=dtype), want)
        room = torch.zeros(rows * n + 2, dtype=dtype, device="cuda")
        got = grouped_linear_int4(x, packed, loads, bias=bias.cuda(), out=room[1:-1].view(rows, n))  # (an odd address)
        assert torch.equal(got, want) and float(room[0]) == float(room[-1]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("columns,n", [(128, 1024), (256, 2048)])
def test_two_calls_of_tiles_at_once(columns, n):
    rows = 2000
    assert columns_of("bf16", rows, 512, n, 4, 64) == columns
    w = [Weights(i, 4, n, 512, 64, zeros=True).cuda() for i in range(2)]
    x = [normal(i, rows, 512, dtype=torch.bfloat16).cuda() for i in range(2)]
    loads = [loads_of(i, rows, 4).cuda() for i in range(2)]
    want = [grouped_linear_int4(x[i], w[i], loads[i]) for i in range(2)]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(grouped_linear_int4(x[i], w[i], loads[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(made, want[i]) for i in range(2) for made in got[i])


@pytest.mark.gpu
def test_a_layer_of_tiles_on_a_stream_and_replayed():
    """Gate, route and two products, of 256 and of 128 columns: each against 64 bits, on a stream of its own, captured and replayed for other inputs."""
    tokens, d, d_ff, paths, k = 3000, 256, 1024, 6, 2
    assert columns_of("bf16", tokens * k, d, d_ff, paths, 64, cells=tokens) == 256 and columns_of("bf16", tokens * k, d_ff, d, paths, 128) == 128
    w1, w2 = Weights(1, paths, d_ff, d, 64, zeros=True), Weights(2, paths, d, d_ff, 128)
    on1, on2 = w1.cuda(), w2.cuda()

    def layer(x, scores):
        ids, weights = c_router.gate_topk(scores, k, True)
        loads, _, seat_rows, entries = c_router.route_by_path(ids, paths)
        hidden = grouped_linear_int4(x, on1, loads, activation="gelu", row_entries=entries, entries_per_cell=k)
        y = grouped_linear_int4(hidden, on2, loads, out_dtype=torch.float32)
        return c_router.combine_by_rows(y, ids, seat_rows, weights, out_dtype=x.dtype), hidden, y, loads, entries

    def inputs(seed):
        return normal(seed, tokens, d, dtype=torch.bfloat16, scale=0.3).cuda(), normal(seed + 1, tokens, paths).cuda()

    first = inputs(1)
    _, hidden, y, loads, entries = (t.cpu() for t in layer(*first))
    assert int(loads.sum()) == tokens * k
    want, size = product_in_64(first[0].cpu()[(entries.long() - 1) // k], w1, loads, activation="gelu")
    assert_near(hidden, want, size, 64, d, gelu=True)
    want, size = product_in_64(hidden, w2, loads)
    assert_near(y, want, size, 128, d_ff)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = inputs(11)
        made = layer(*second)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(made, layer(*second)))
    x, scores = inputs(21)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer(x, scores)
    for seed in (31, 41, 51):
        new = inputs(seed)
        x.copy_(new[0]), scores.copy_(new[1])
        graph.replay()
        eager = layer(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("columns,n", [(128, 64), (256, 160)])
def test_rows_beyond_four_gib_in_tiles(columns, n):
    """The last rows of x lie past 2^32 bytes."""
    rows, k = 270000, 8192
    assert columns_of("bf16", rows, k, n, 2, 128) == columns
    w = Weights(1, 2, n, k, 128)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    tail = normal(2, 100, k, dtype=torch.bfloat16)
    x[-100:] = tail.cuda()
    got = grouped_linear_int4(x, w.cuda(), torch.tensor([rows - 100, 100], dtype=torch.int32, device="cuda"))
    want, size = product_in_64(tail, w, torch.tensor([0, 100]))
    assert not got[:-100].any()
    assert_near(got[-100:], want, size, 128, k)


@pytest.mark.gpu
def test_results_beyond_four_gib_in_tiles():
    """The last results lie past 2^32 bytes (and 2^31 elements)."""
    rows, k, n = 300000, 64, 8192
    assert columns_of("bf16", rows, k, n, 2, 64) == 256
    w, x = Weights(1, 2, n, k, 64), normal(2, rows, k, dtype=torch.bfloat16)
    loads = torch.tensor([rows - 100, 100], dtype=torch.int32)
    got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda())
    for some, given in ((slice(0, 100), [100, 0]), (slice(rows - 200, rows), [100, 100])):
        want, size = product_in_64(x[some], w, torch.tensor(given))
        assert_near(got[some], want, size, 64, k)


@pytest.mark.gpu
def test_weights_beyond_four_gib_in_tiles():
    """The last expert's weights lie past 2^32 bytes: the bits of the same weights at the beginning of an array."""
    experts, n, k, rows = 66, 8192, 16384, 2000
    assert columns_of("bf16", rows, k, n, experts, 128) == columns_of("bf16", rows, k, n, 1, 128) == 256
    values = torch.zeros(experts, n // 16, k // 128, 1024, dtype=torch.uint8, device="cuda")
    scales = torch.ones(experts, n // 16, k // 128, 16, dtype=torch.bfloat16, device="cuda")
    values[-1].copy_(torch.randint(0, 256, values.shape[1:], dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    assert (values.numel() // experts) * (experts - 1) > 1 << 32
    loads = torch.zeros(experts, dtype=torch.int32, device="cuda")
    loads[-1] = rows
    x = normal(1, rows, k, dtype=torch.bfloat16).cuda()
    got = grouped_linear_int4(x, Int4Weight(values, scales, None, k, n, 128), loads)
    want = grouped_linear_int4(x, Int4Weight(values[-1:].clone(), scales[-1:].clone(), None, k, n, 128), loads[-1:])
    assert torch.equal(got, want) and bool(want.any())


@pytest.mark.gpu
@pytest.mark.parametrize("columns,n", [(128, 700), (256, 1300)])
def test_cells_up_to_two_gib_in_tiles(columns, n):
    """Rows gathered from cells that end just below 2^31 bytes."""
    cells, rows, k = 131000, 3000, 8192
    assert columns_of("bf16", rows, k, n, 2, 64, cells=cells) == columns and columns_of("bf16", rows, k, n, 2, 64, cells=1 << 17) == 16
    w, loads = Weights(1, 2, n, k, 64).cuda(), torch.tensor([1000, 2000], dtype=torch.int32, device="cuda")
    x = torch.zeros(cells, k, dtype=torch.bfloat16, device="cuda")
    x[-rows:] = normal(2, rows, k, dtype=torch.bfloat16).cuda()
    entries = torch.arange(cells, cells - rows, -1, dtype=torch.int32, device="cuda")
    got = grouped_linear_int4(x, w, loads, row_entries=entries)
    want = grouped_linear_int4(x[-rows:].flip(0), w, loads)
    assert torch.equal(got, want) and bool(want.any(1).all())


def test_launches_of_too_many_threads_are_refused_without_a_gpu():
    lib, some = _lib.lib(), 16  # an address that is never read: every call ends before a launch

    def code(x_dtype, experts, rows, n, k):
        return lib.brt_hip_grouped_gemm_int4(some, x_dtype, None, 1, 0, some, some, 2, None, 128, some, None, 0, some, x_dtype, experts, rows, n, k, 0, None)

    for given in ((0, 8, 1 << 20, 1 << 14, 2048), (0, 1 << 22, 1 << 23, 1 << 8, 512), (2, 8, (1 << 24) - 1, 1 << 14, 2048), (1, 1 << 20, 1 << 22, 1 << 11, 1024)):
        assert code(*given) == -4 and b"too many tiles" in lib.brt_hip_last_error(), given

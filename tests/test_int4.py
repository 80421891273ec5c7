"""Products with 4-bit weights against the definition in 64 bits, the layout of the weights, and their refusals.

Products of a weight (0 .. 15) and an element are exact in fp32, and so are the three parts that an fp32 element is split into but for 2^-27 of
it.  A group's sum starts from -zero times its sum of x: of ``group`` terms each (three times as many of fp32 rows), every addition off by
at most a step of 2^-23 of the magnitudes added so far, zero * |x| and q * |x|.  The scale's multiply-add, the sum over blocks and wavefronts and
the bias add at most one rounding per group and 20 more: (6 * group + groups + 20) * 2^-23 of the sum of scale * (q + zero) * |x| in
all.  Those errors have both signs; the bound is not often approached.  GELU is within 4.3e-6 for 16-bit results and 4 steps of 2^-23 of its
operand for fp32 ones, and passes an error on at most 1.13-fold.  The last rounding is half a step (``eps / 2``) of the value.
"""
import pytest
import torch

import brt._C.router as c_router
from brainstorm_amd import _lib
from brt.jit import Int4Weight, grouped_linear_int4, pack_int4, quantize_int4

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def loads_of(seed, rows, experts, empty=()):
    gen = torch.Generator().manual_seed(seed)
    share = torch.rand(experts, generator=gen) ** 2
    for e in empty:
        share[e] = 0
    return torch.bincount(torch.multinomial(share, rows, True, generator=gen), minlength=experts).int() if rows else torch.zeros(experts, dtype=torch.int32)


class Weights:
    """Random values, scales and zeros, and what they stand for."""

    def __init__(self, seed, experts, n, k, group, zeros=False, scale_dtype=torch.bfloat16):
        gen = torch.Generator().manual_seed(seed)
        groups = -(-k // group)
        self.q = torch.randint(0, 16, (experts, n, k), generator=gen).to(torch.uint8)
        self.s = (torch.rand(experts, n, groups, generator=gen) * 0.01 + 0.001).to(scale_dtype)
        self.z = torch.randint(0, 16, (experts, n, groups), generator=gen).to(torch.uint8) if zeros else None
        self.group, self.k = group, k
        self.packed = pack_int4(self.q, self.s, self.z, group=group)

    def spread(self, t):
        return t.double().repeat_interleave(self.group, -1)[..., :self.k]

    def zero(self, e):
        return 8.0 if self.z is None else self.spread(self.z[e])

    def values(self, e):
        return (self.q[e].double() - self.zero(e)) * self.spread(self.s[e])

    def sizes(self, e):
        return (self.q[e].double() + self.zero(e)) * self.spread(self.s[e])

    def cuda(self):
        return Int4Weight(*(t.cuda() if torch.is_tensor(t) else t for t in self.packed))


def product_in_64(x, w, loads, bias=None, activation=None):
    """(result, magnitudes) of packed rows; rows behind the last expert's are NaN."""
    rows, n = x.shape[0], w.q.shape[1]
    want = torch.full((rows, n), float("nan"), dtype=torch.float64)
    size = torch.zeros(rows, n, dtype=torch.float64)
    first = 0
    for e, load in enumerate(loads.tolist()):
        here = slice(first, first + load)
        part = x[here].double()
        want[here], size[here] = part @ w.values(e).t(), part.abs() @ w.sizes(e).t()
        if bias is not None:
            want[here] += bias[e].double()
            size[here] += bias[e].double().abs()
        first += load
    if activation == "gelu":
        want = torch.nn.functional.gelu(want)
    elif activation == "relu":
        want = torch.where(want < 0, torch.zeros_like(want), want)
    return want, size


def assert_near(got, want, size, group, k, gelu=False):
    got, kept = got.cpu(), ~want.isnan()
    info = torch.finfo(got.dtype)
    off = (6 * group + -(-k // group) + 20) * 2.0 ** -23 * size
    if gelu:
        off = 1.13 * off + (4.0 * 2.0 ** -23 * (want.abs() + 1) if got.dtype == torch.float32 else 4.3e-6)
    bound = off + info.eps / 2 * (want.abs() + off) + info.tiny * info.eps
    far = ((got.double() - want).abs() / bound)[kept]
    assert not far.numel() or float(far.max()) <= 1.0, f"{float(far.max())} of the bound"
    if far.numel() >= 64 and float(want[kept].norm()) > 0:  # (both signs: the norm of the errors of the sum stays far below the bound)
        rel = float((got.double() - want)[kept].norm() / want[kept].norm())
        assert rel <= 0.6 * info.eps + 2e-6 + (4.3e-6 / float(want[kept].square().mean().sqrt()) if gelu and info.eps > 1e-6 else 0.0), rel


# ------------------------------------------------------------------------------------ the layout
@pytest.mark.parametrize("experts,n,k,group", [(1, 1, 1, 32), (2, 16, 128, 128), (3, 17, 136, 32), (2, 40, 264, 64), (1, 100, 96, 128)])
def test_layout_of_the_bytes(experts, n, k, group):
    w = Weights(1, experts, n, k, group, zeros=True, scale_dtype=torch.float32)
    values, scales, zeros = w.packed[:3]
    assert values.shape == (experts, -(-n // 16), -(-k // 128), 1024) and values.dtype == torch.uint8
    assert scales.shape == zeros.shape == (experts, -(-n // 16), -(-k // group), 16)
    for e in range(experts):
        for row in range(0, n, 3):
            for column in range(k):
                block, c = divmod(column, 128)
                g, i = c % 32 // 8, c % 8
                byte = int(values[e, row // 16, block, 16 * (16 * g + row % 16) + 4 * (c // 32) + i % 4])
                assert (byte >> (4 * (i // 4))) & 15 == int(w.q[e, row, column])
            for at in range(-(-k // group)):
                assert float(scales[e, row // 16, at, row % 16]) == float(w.s[e, row, at])
                assert int(zeros[e, row // 16, at, row % 16]) == int(w.z[e, row, at])
    assert (w.packed.in_features, w.packed.out_features, w.packed.group) == (k, n, group)


def unpacked(packed):
    """[experts, out_features, in_features] that an Int4Weight stands for."""
    values, scales, zeros, k, n, group = packed
    experts, tiles, blocks, _ = values.shape
    at = torch.arange(1024)
    g, r, j, m = at // 256, at // 16 % 16, at // 4 % 4, at % 4
    q = torch.zeros(experts, tiles, 16, blocks, 128, dtype=torch.float64)
    for half in (0, 1):
        q[:, :, r, :, 32 * j + 8 * g + m + 4 * half] = ((values >> (4 * half)) & 15).double().permute(3, 0, 1, 2)
    q = q.view(experts, tiles * 16, blocks * 128)[:, :n, :k]

    def spread(t):
        return t.double().transpose(2, 3).reshape(experts, tiles * 16, -1)[:, :n].repeat_interleave(group, 2)[:, :, :k]

    return (q - (8.0 if zeros is None else spread(zeros))) * spread(scales)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("experts,n,k,group", [(1, 5, 8, 32), (2, 33, 200, 64), (1, 64, 512, 128)])
def test_quantized_weights(experts, n, k, group, zeros, dtype):
    """Half a step of the scale at most; the scale's own rounding moves the largest weight of a group (7 or 15 steps of it) by up to that
    many half steps of its type more, which holding to 0 .. 15 may cut off."""
    weight = normal(1, experts, n, k, dtype=TYPES[dtype])
    weight[0, 0, :4] = 0
    weight[0, 1] = 0
    weight[0, 2] = 1.0
    packed = quantize_int4(weight, group, zeros=zeros)
    got = unpacked(packed)
    step = packed.scales.double().transpose(2, 3).reshape(experts, -1, packed.scales.shape[2])[:, :n].repeat_interleave(group, 2)[:, :, :k]
    slack = 0.5 + 15 * torch.finfo(TYPES[dtype]).eps + 1e-5 + (0.5 if zeros else 0.0)  # (the zero point is rounded too)
    assert bool(((got - weight.double()).abs() <= slack * step + 1e-12).all())
    assert not got[0, 1].any() and packed.scales.dtype == TYPES[dtype] and (packed.zeros is not None) == zeros
    again = quantize_int4(weight, group, zeros=zeros, scale_dtype=torch.float32)
    assert again.scales.dtype == torch.float32
    if not zeros:
        assert abs(float(unpacked(again)[0, 2, 0]) - 1.0) <= 1e-6


@pytest.mark.parametrize("zeros", [False, True])
def test_quantized_weights_whose_reciprocal_scale_overflows(zeros):
    """A scale below 2^-128 has no reciprocal in fp32; weights and scale are steps of 2^-149 there."""
    weight = torch.tensor([[[0.0, 1e-39, -3e-39, 7e-40, 0.0, 2e-39, -1e-39, 3e-39]]])
    packed = quantize_int4(weight, 32, zeros=zeros)
    step = float(packed.scales.max())
    assert 0 < step < 2.0 ** -128
    assert bool(((unpacked(packed) - weight.double()).abs() <= 1.01 * step).all())
    assert not unpacked(packed)[0, 0, [0, 4]].any()


def test_refusals_of_the_layout():
    q, s = torch.zeros(2, 16, 64, dtype=torch.uint8), torch.ones(2, 16, 1)
    for call, error, words in (
            (lambda: pack_int4(q, s, group=48), NotImplementedError, "48"),
            (lambda: pack_int4(q.int(), s, group=64), RuntimeError, "uint8"),
            (lambda: pack_int4(q[0], s, group=64), RuntimeError, "uint8"),
            (lambda: pack_int4(q, s.double(), group=64), NotImplementedError, "scales"),
            (lambda: pack_int4(q, s, group=32), RuntimeError, "groups"),
            (lambda: pack_int4(q, s, s.int(), group=64), RuntimeError, "zeros"),
            (lambda: pack_int4(q + 16, s, group=64), RuntimeError, "0 .. 15"),
            (lambda: quantize_int4(torch.ones(2, 16, 64), 100), NotImplementedError, "100"),
            (lambda: quantize_int4(torch.ones(16, 64)), RuntimeError, "weight"),
            (lambda: quantize_int4(torch.ones(2, 16, 64).double()), RuntimeError, "weight"),
            (lambda: quantize_int4(torch.ones(2, 16, 64), scale_dtype=torch.int32), NotImplementedError, "scales")):
        with pytest.raises(error, match=words):
            call()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_weights_and_scales_that_are_not_finite_are_refused(bad, zeros):
    """They would come out as scales that are not finite, or as weights of any value in their place."""
    for dtype in TYPES.values():
        weight = normal(1, 3, 5, 72, dtype=dtype)
        weight[2, 4, 71] = bad
        with pytest.raises(RuntimeError, match="expert 2 holds values that are not finite"):
            quantize_int4(weight, 32, zeros=zeros)
        scales = torch.ones(2, 16, 2, dtype=dtype)
        scales[1, 3, 1] = bad
        with pytest.raises(RuntimeError, match="scales must be finite"):
            pack_int4(torch.zeros(2, 16, 64, dtype=torch.uint8), scales, group=32)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantized_weights_do_not_depend_on_the_default_type(default, zeros):
    weight = normal(1, 2, 33, 200) * 3e4
    want = quantize_int4(weight, 64, zeros=zeros)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = quantize_int4(weight, 64, zeros=zeros)
        again = pack_int4(torch.zeros(2, 33, 200, dtype=torch.uint8), torch.ones(2, 33, 4, dtype=torch.float32), group=64)
    finally:
        torch.set_default_dtype(before)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got[:3], want[:3])) and got.scales.dtype == again.scales.dtype == torch.float32


@pytest.mark.parametrize("zeros", [False, True])
def test_scales_beyond_their_type_are_refused(zeros):
    weight = torch.zeros(2, 4, 64)
    weight[1, 2, 5] = 15 * 65504.0
    assert quantize_int4(weight, 32, zeros=zeros).scales.isfinite().all()
    at_the_border = weight / 15 * (15 if zeros else 7)
    assert float(quantize_int4(at_the_border, 32, zeros=zeros, scale_dtype=torch.float16).scales.max()) == 65504.0
    with pytest.raises(RuntimeError, match="expert 1 needs a scale beyond torch.float16"):
        quantize_int4(weight * 2, 32, zeros=zeros, scale_dtype=torch.float16)


# ---------------------------------------------------------------------------------- the products
SHAPES = [  # rows, in, out, experts, group
    (1, 8, 1, 1, 32), (1, 128, 16, 1, 128), (1, 2048, 512, 4, 128), (2, 136, 17, 3, 64), (5, 64, 40, 2, 32), (16, 256, 64, 1, 128), (17, 384, 33, 1, 32),
    (33, 776, 1001, 12, 32), (48, 1024, 256, 8, 64), (100, 40, 100, 5, 64), (130, 512, 96, 3, 128), (257, 264, 320, 4, 32), (300, 1024, 128, 64, 128),
    (64, 4096, 48, 2, 64), (700, 200, 72, 3, 128), (1500, 384, 264, 2, 64), (2049, 136, 130, 5, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,k,n,experts,group", SHAPES)
def test_products(rows, k, n, experts, group, zeros, dtype):
    dtype = TYPES[dtype]
    w = Weights(rows + k, experts, n, k, group, zeros, scale_dtype=torch.bfloat16 if zeros else torch.float16)
    x, loads = normal(1, rows, k, dtype=dtype), loads_of(rows, rows, experts, empty=(1,) if experts > 2 else ())
    got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda())
    want, size = product_in_64(x, w, loads)
    assert got.dtype == dtype and got.shape == (rows, n)
    assert_near(got, want, size, group, k)


KERNELS = [  # columns of the tiles that take these sizes; rows, in, out, experts, group
    (16, 200, 264, 48, 4, 64), (16, 400, 328, 1100, 4, 64), (16, 156, 136, 2100, 9, 64), (16, 200, 64, 100, 2, 128), (16, 586, 328, 1001, 5, 128),
    (16, 3615, 136, 100, 40, 32), (16, 5, 4104, 100, 2, 128), (16, 8, 1032, 1001, 8, 64), (16, 8, 520, 1001, 8, 32), (16, 40, 1096, 1300, 16, 128),
    (16, 40, 600, 1300, 16, 64), (16, 60, 904, 2100, 40, 32), (16, 100, 1096, 1300, 4, 128), (16, 100, 600, 1300, 4, 64),
    (128, 1420, 328, 1300, 9, 32), (128, 2043, 488, 1001, 20, 64), (128, 3485, 136, 600, 5, 128), (128, 4392, 488, 384, 128, 64),
    (256, 642, 136, 2100, 40, 128), (256, 3144, 72, 1001, 40, 32), (256, 3347, 264, 1300, 2, 64), (256, 3585, 328, 1300, 3, 32),
]


def test_which_kernel_takes_the_shapes_below():
    kernel = _lib.lib().brt_hip_grouped_gemm_int4_kernel
    for columns, rows, k, n, experts, group in KERNELS:
        assert kernel(2, -1, group, experts, rows, n, k) == kernel(1, rows, group, experts, rows, n, k) == columns, (columns, rows, k, n, experts, group)
        assert kernel(0, -1, group, experts, rows, n, k) == 16
    assert kernel(2, 0, 128, 8, 4096, 4096, 4096) == 16 and kernel(2, 1 << 20, 128, 8, 4096, 4096, 4096) == 16  # no cells; cells beyond 31 bits
    assert kernel(2, -1, 48, 8, 4096, 4096, 4096) == kernel(3, -1, 64, 8, 4096, 4096, 4096) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("zeros,scales", [(False, "bf16"), (True, "f16"), (True, "f32")])
@pytest.mark.parametrize("columns,rows,k,n,experts,group", KERNELS)
def test_products_of_every_kernel(columns, rows, k, n, experts, group, zeros, scales, dtype):
    """Ragged loads with empty experts, tails of K and N in every kernel, with and without row entries, 16-bit and fp32 results."""
    dtype = TYPES[dtype]
    w = Weights(rows + k, experts, n, k, group, zeros, scale_dtype=TYPES[scales])
    x, loads, bias = normal(1, rows, k, dtype=dtype), loads_of(rows, rows, experts, empty=(1,) if experts > 2 else ()), normal(2, experts, n)
    for out, activation in ((dtype, "gelu"), (torch.float32, "none")):
        got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), bias=bias.cuda(), activation=activation, out_dtype=out)
        want, size = product_in_64(x, w, loads, bias, activation)
        assert_near(got, want, size, group, k, gelu=activation == "gelu")
    cells = rows // 2 + 1
    entries = torch.randint(-1, 2 * cells + 2, (rows,), generator=torch.Generator().manual_seed(3)).int()
    there = (entries >= 1) & (entries <= 2 * cells)
    packed = torch.where(there[:, None], x[((entries.long() - 1) // 2).clamp(0, cells - 1)], 0)
    want = grouped_linear_int4(packed.cuda(), w.cuda(), loads.cuda(), bias=bias.cuda())
    got = grouped_linear_int4(x[:cells].cuda(), w.cuda(), loads.cuda(), bias=bias.cuda(), row_entries=entries.cuda(), entries_per_cell=2)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["none", "relu", "gelu"])
@pytest.mark.parametrize("dtype,out,scales", [("bf16", "bf16", "f32"), ("bf16", "f32", "bf16"), ("f16", "bf16", "f16"), ("f32", "f16", "f32"), ("f32", "f32", "bf16")])
@pytest.mark.parametrize("rows,k,n,experts,group", [(3, 256, 100, 2, 128), (60, 520, 65, 4, 32), (900, 256, 384, 3, 64)])
def test_bias_activation_and_types(rows, k, n, experts, group, dtype, out, scales, activation):
    w = Weights(rows, experts, n, k, group, zeros=True, scale_dtype=TYPES[scales])
    x, loads = normal(1, rows, k, dtype=TYPES[dtype], scale=0.3), loads_of(rows, rows, experts)
    for bias_type in (dtype, "f32"):
        bias = normal(3, experts, n, dtype=TYPES[bias_type])
        want, size = product_in_64(x, w, loads, bias, activation)
        got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), bias=bias.cuda(), activation=activation, out_dtype=TYPES[out])
        assert got.dtype == TYPES[out]
        assert_near(got, want, size, group, k, gelu=activation == "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 600, 5000])
def test_loads_that_do_not_fill_the_rows(rows):
    """Rows behind the last expert's are left as they were; loads below zero count as none; rows behind the last of x do not exist."""
    k, n, experts, group = 128, 80, 4, 64
    w, x = Weights(1, experts, n, k, group), normal(2, rows, k, dtype=torch.bfloat16)
    for given in ([3, 0, rows // 2, 5], [-7, 4, -1, 2], [0, 0, 0, 0], [rows - 5, 100, 7, 9], [0, 2000000000, 2000000000, 1]):
        taken, left = [], rows
        for load in given:
            taken.append(max(0, min(load, left)))
            left -= taken[-1]
        out = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
        got = grouped_linear_int4(x.cuda(), w.cuda(), torch.tensor(given, dtype=torch.int32, device="cuda"), out=out)
        assert got.data_ptr() == out.data_ptr()
        want, size = product_in_64(x, w, torch.tensor(taken))
        assert_near(got, want, size, group, k)
        assert bool((got[rows - left:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cells,k,paths,d,n,capacity", [(1, 1, 3, 64, 33, 4), (40, 2, 4, 136, 48, 12), (300, 2, 8, 256, 64, 200), (900, 1, 3, 128, 96, 250)])
def test_rows_named_by_their_entries(cells, k, paths, d, n, capacity, dtype):
    """The same bits as dispatch_by_rows and the product of its rows, padding rows and dropped cells among them."""
    dtype = TYPES[dtype]
    gen = torch.Generator().manual_seed(cells)
    ids = torch.rand(cells, paths, generator=gen).argsort(1)[:, :k].int().contiguous().cuda()
    x, w = normal(1, cells, d, dtype=dtype).cuda(), Weights(2, paths, n, d, 64, zeros=True)
    caps = torch.tensor([capacity], dtype=torch.int32, device="cuda")
    bias = normal(3, paths, n).cuda()
    for padding in (False, True):
        rows = paths * capacity if padding else cells * k
        loads, _, seat_rows, entries = c_router.route_by_path(ids, paths, caps, capacity_padding=padding, rows=rows)
        dispatched = c_router.dispatch_by_rows(x, entries, k)
        want = grouped_linear_int4(dispatched, w.cuda(), loads, bias=bias, out=torch.zeros(rows, n, dtype=dtype, device="cuda"))
        got = grouped_linear_int4(x, w.cuda(), loads, bias=bias, out=torch.zeros(rows, n, dtype=dtype, device="cuda"), row_entries=entries, entries_per_cell=k)
        assert torch.equal(got, want)
    strange = torch.tensor([0, -5, cells * k + 1, 1], dtype=torch.int32, device="cuda")  # none of the first three is a cell's
    got = grouped_linear_int4(x, w.cuda(), torch.tensor([4] + [0] * (paths - 1), dtype=torch.int32, device="cuda"), bias=bias, row_entries=strange, entries_per_cell=k)
    assert torch.equal(got[:3].float(), bias[:1].to(dtype).float().expand(3, n))
    none = grouped_linear_int4(x[:0], w.cuda(), torch.tensor([4] + [0] * (paths - 1), dtype=torch.int32, device="cuda"), bias=bias, row_entries=strange, entries_per_cell=k)
    assert torch.equal(none.float(), bias[:1].to(dtype).float().expand(4, n))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [20, 500, 3000])
def test_a_row_of_its_own(rows, dtype):
    """A row's result does not depend on what the others hold; one that holds NaN or an infinity gives NaN behind an activation too."""
    k, n, experts = 200, 48, 3
    w, loads = Weights(1, experts, n, k, 32, zeros=True).cuda(), loads_of(2, rows, experts).cuda()
    x = normal(3, rows, k, dtype=TYPES[dtype]).cuda()
    bad = x.clone()
    bad[0, 5], bad[7, k - 1], bad[rows - 1, 100] = float("nan"), float("inf"), float("-inf")
    for activation in ("none", "relu", "gelu"):
        want, got = (grouped_linear_int4(t, w, loads, activation=activation) for t in (x, bad))
        sound = torch.isfinite(bad).all(1)
        assert torch.equal(got[sound], want[sound]) and got[~sound].isnan().all()


@pytest.mark.gpu
def test_large_and_tiny_values():
    """Elements of every size that the types hold, none of them lost beside the others' products (fp32 rows are split exactly)."""
    k, n = 64, 16
    w = Weights(1, 1, n, k, 32, zeros=True, scale_dtype=torch.float32)
    loads = torch.tensor([6], dtype=torch.int32)
    for dtype in TYPES.values():
        info = torch.finfo(dtype)
        x = normal(2, 6, k, dtype=torch.float64)
        for r, size in enumerate((info.max / 2.0 ** 14, info.tiny * 2.0 ** 10, 1e3, 1e-3, 1.0, 0.0)):
            x[r] *= size / 8
        x = x.to(dtype)
        want, size = product_in_64(x, w, loads)
        got = grouped_linear_int4(x.cuda(), w.cuda(), loads.cuda(), out_dtype=torch.float32)
        # (parts of fp32 elements below 2^-126 and products below it are lost: an absolute 64 * 2^-126 * 15 of the scale)
        assert_near(got.double().float(), want, size + 64 * 15 * 2.0 ** -103, 32, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [9, 700])
def test_strides_and_addresses(rows):
    k, n, experts = 128, 50, 2
    w, loads = Weights(1, experts, n, k, 64, zeros=True), loads_of(2, rows, experts).cuda()
    base = normal(3, rows * 2, k + 8, dtype=torch.bfloat16).cuda()
    bias = normal(4, n, experts).t()
    packed = w.cuda()
    shifted = torch.empty(packed.values.numel() + 3, dtype=torch.uint8, device="cuda")[3:].view(packed.values.shape)
    shifted.copy_(packed.values)
    other = packed._replace(values=shifted, scales=packed.scales.transpose(0, 1).contiguous().transpose(0, 1), zeros=packed.zeros.clone())
    for x in (base[::2, :k], base[:rows, 3:k + 3], base[:rows].view(-1)[1:1 + rows * k].view(rows, k), base[:1, :k].expand(rows, k)):
        want = grouped_linear_int4(x.contiguous().clone(), packed, loads, bias=bias.contiguous().cuda())
        got = grouped_linear_int4(x, other, loads, bias=bias.cuda())
        assert torch.equal(got, want)
    room = torch.zeros(rows * n + 1, dtype=torch.bfloat16, device="cuda")
    got = grouped_linear_int4(x, packed, loads, bias=bias.cuda(), out=room[1:].view(rows, n))  # (an odd address)
    assert torch.equal(got, want) and float(room[0]) == 0.0


@pytest.mark.gpu
def test_no_rows_no_columns():
    w, loads = Weights(1, 2, 20, 64, 32).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    assert grouped_linear_int4(torch.zeros(0, 64, device="cuda"), w, loads).shape == (0, 20)
    assert grouped_linear_int4(torch.zeros(5, 64, device="cuda"), w, loads).shape == (5, 20)
    bare = Weights(1, 2, 0, 64, 32).cuda()
    assert grouped_linear_int4(torch.zeros(5, 64, device="cuda"), bare, loads).shape == (5, 0)


@pytest.mark.gpu
def test_weights_beyond_four_gib():
    """The last expert's weights lie past 2^32 bytes, its rows' results past 2^31 elements of x."""
    experts, n, k = 66, 8192, 16384
    values = torch.zeros(experts, n // 16, k // 128, 1024, dtype=torch.uint8, device="cuda")
    scales = torch.ones(experts, n // 16, k // 128, 16, dtype=torch.bfloat16, device="cuda")
    some = torch.randint(0, 256, values.shape[1:], dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    values[-1].copy_(some)
    loads = torch.zeros(experts, dtype=torch.int32, device="cuda")
    loads[-1] = 3
    x = normal(1, 3, k, dtype=torch.bfloat16).cuda()
    got = grouped_linear_int4(x, Int4Weight(values, scales, None, k, n, 128), loads)
    want = grouped_linear_int4(x, Int4Weight(values[-1:].clone(), scales[-1:].clone(), None, k, n, 128), loads[-1:])
    assert torch.equal(got, want) and bool(want.any())


@pytest.mark.gpu
def test_rows_beyond_four_gib():
    rows, k, n = 270000, 8192, 16
    w = Weights(1, 2, n, k, 128)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    tail = normal(2, 40, k, dtype=torch.bfloat16)
    x[-40:] = tail.cuda()
    loads = torch.tensor([rows - 40, 40], dtype=torch.int32)
    got = grouped_linear_int4(x, w.cuda(), loads.cuda())
    want, size = product_in_64(tail, w, torch.tensor([0, 40]))
    assert not got[:-40].any()
    assert_near(got[-40:], want, size, 128, k)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 24, 700])
def test_a_served_layer_on_a_stream_and_replayed(tokens):
    """Gate, route, two products and the combine: against plain torch in 64 bits, on a stream of its own, captured and replayed for other inputs."""
    d, d_ff, paths, k = 128, 256, 6, 2
    w1, w2 = Weights(1, paths, d_ff, d, 64, zeros=True), Weights(2, paths, d, d_ff, 128)
    on1, on2 = w1.cuda(), w2.cuda()

    def layer(x, scores):
        ids, weights = c_router.gate_topk(scores, k, True)
        loads, _, seat_rows, entries = c_router.route_by_path(ids, paths)
        hidden = grouped_linear_int4(x, on1, loads, activation="gelu", row_entries=entries, entries_per_cell=k)
        y = grouped_linear_int4(hidden, on2, loads, out_dtype=torch.float32)
        return c_router.combine_by_rows(y, ids, seat_rows, weights, out_dtype=x.dtype), ids, weights

    def inputs(seed):
        return normal(seed, tokens, d, dtype=torch.bfloat16, scale=0.3).cuda(), normal(seed + 1, tokens, paths).cuda()

    def check(made, x, scores):
        out, ids, weights = (t.cpu() for t in made)
        want, size = torch.zeros(tokens, d, dtype=torch.float64), torch.zeros(tokens, d, dtype=torch.float64)
        x = x.cpu().double()
        for t in range(tokens):
            for j in range(k):
                e = int(ids[t, j])
                hidden = torch.nn.functional.gelu(x[t] @ w1.values(e).t())
                want[t] += float(weights[t, j]) * (hidden @ w2.values(e).t())
                size[t] += float(weights[t, j]) * (hidden.abs() @ w2.values(e).abs().t())
        # the hidden rows are rounded to bf16 (2^-8 each, a little more at borders), the result once
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * (1.1 * size + want.abs()) + 1e-4).all())

    first = inputs(1)
    check(layer(*first), *first)
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
@pytest.mark.parametrize("rows", [20, 2000])
def test_two_calls_at_once(rows):
    w = [Weights(i, 4, 512, 512, 64, zeros=True).cuda() for i in range(2)]
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
@pytest.mark.parametrize("tokens,paths", [(40, 4), (3000, 16)])
def test_a_layer_is_trained_and_then_served_in_four_bits(tokens, paths):
    """A step with the losses (gradients of cells, scores and experts against torch in 64 bits), its experts in 4 bits then, for the same route."""
    d, d_ff, k = 64, 96, 2
    x, scores = normal(1, tokens, d, scale=0.5).cuda().requires_grad_(), normal(2, tokens, paths).cuda().requires_grad_()
    w1, w2 = normal(3, paths, d_ff, d, scale=d ** -0.5).cuda().requires_grad_(), normal(4, paths, d, d_ff, scale=d_ff ** -0.5).cuda().requires_grad_()
    grad, leaves = normal(5, tokens, d).cuda(), [x, scores, w1, w2]
    ids, weights = c_router.gate_topk(scores, k, softmax=True, differentiable=True)
    balance, z, counts = c_router.balance_loss(scores, ids)
    loads, _, seat_rows, entries = c_router.route_by_path(ids, paths)
    assert torch.equal(loads, counts)
    rows = c_router.dispatch_by_rows(x, entries, k, seat_rows=seat_rows)
    parts = [torch.nn.functional.gelu(part @ w1[e].t()) @ w2[e].t() for e, part in enumerate(rows.split(loads.tolist()))]
    out = c_router.combine_by_rows(torch.cat(parts), ids, seat_rows, weights, row_entries=entries)
    made = torch.autograd.grad([out, balance, z], leaves, [grad, torch.tensor(0.5, device="cuda"), torch.tensor(0.1, device="cuda")])

    x64, s64, w164, w264 = (t.detach().cpu().double().requires_grad_() for t in leaves)
    chosen, p = ids.cpu().long(), torch.softmax(s64, 1)
    want = torch.zeros(tokens, d, dtype=torch.float64)
    for e in range(paths):
        share = (p * torch.nn.functional.one_hot(chosen, paths).sum(1))[:, e:e + 1]
        want = want + share * (torch.nn.functional.gelu(x64 @ w164[e].t()) @ w264[e].t())
    balance64 = paths / (tokens * tokens * k) * (counts.cpu() * p.sum(0)).sum()
    z64 = torch.logsumexp(s64, 1).square().mean()
    wants = torch.autograd.grad((want * grad.cpu()).sum() + 0.5 * balance64 + 0.1 * z64, [x64, s64, w164, w264])
    # fp32 throughout: products of at most 3000 terms, each sum off by less than 1e-5 of its magnitudes
    for got, exact in zip([out.detach(), balance.detach(), z.detach(), *made], [want.detach(), balance64.detach(), z64.detach(), *wants]):
        assert float((got.cpu().double() - exact).norm()) <= 1e-5 * float(exact.norm())

    served1, served2 = quantize_int4(w1, 32, zeros=True), quantize_int4(w2, 32)
    with torch.no_grad():
        ids4, weights4 = c_router.gate_topk(scores, k, softmax=True)
        balance4, z4, counts4 = c_router.balance_loss(scores, ids4)
        loads4, _, seat_rows4, entries4 = c_router.route_by_path(ids4, paths)
        hidden = grouped_linear_int4(x, served1, loads4, activation="gelu", row_entries=entries4, entries_per_cell=k)
        got = c_router.combine_by_rows(grouped_linear_int4(hidden, served2, loads4), ids4, seat_rows4, weights4)
    assert torch.equal(ids4, ids) and torch.equal(counts4, counts) and torch.equal(balance4, balance) and torch.equal(z4, z)
    v1, v2 = unpacked(Int4Weight(*(t.cpu() if torch.is_tensor(t) else t for t in served1))), unpacked(Int4Weight(*(t.cpu() if torch.is_tensor(t) else t for t in served2)))
    want4 = torch.zeros(tokens, d, dtype=torch.float64)
    for e in range(paths):
        share = (p.detach() * torch.nn.functional.one_hot(chosen, paths).sum(1))[:, e:e + 1]
        want4 += share * (torch.nn.functional.gelu(x64.detach() @ v1[e].t()) @ v2[e].t())
    assert float((got.cpu().double() - want4).norm()) <= 1e-5 * float(want4.norm())
    # what 4 bits are worth: a step of 2/15 to 2/7 of a group's range, half of it off at most
    assert float((want4 - want.detach()).norm()) <= 0.25 * float(want.detach().norm())


@pytest.mark.gpu
def test_refusals():
    w, loads = Weights(1, 2, 20, 64, 32, zeros=True).cuda(), torch.tensor([2, 3], dtype=torch.int32, device="cuda")
    x, bias = normal(2, 5, 64, dtype=torch.bfloat16).cuda(), normal(3, 2, 20).cuda()
    entries = torch.arange(1, 6, dtype=torch.int32, device="cuda")
    room = torch.zeros(5, 20, dtype=torch.bfloat16, device="cuda")
    narrow = Weights(1, 2, 20, 60, 32).cuda()
    for call, error, words in (
            (lambda: grouped_linear_int4(x.cpu(), w, loads), RuntimeError, "CUDA tensor"),
            (lambda: grouped_linear_int4(x, w._replace(values=w.values.cpu()), loads), RuntimeError, "CUDA tensor"),
            (lambda: grouped_linear_int4(x, w._replace(zeros=w.zeros.cpu()), loads), RuntimeError, "another device"),
            (lambda: grouped_linear_int4(x[:, :56], w, loads), RuntimeError, "in_features"),
            (lambda: grouped_linear_int4(x[0], w, loads), RuntimeError, "in_features"),
            (lambda: grouped_linear_int4(normal(1, 5, 60).cuda(), narrow, loads), NotImplementedError, "units of 8"),
            (lambda: grouped_linear_int4(x.double(), w, loads), NotImplementedError, "x data type"),
            (lambda: grouped_linear_int4(x, w, loads, out_dtype=torch.float64), NotImplementedError, "output data type"),
            (lambda: grouped_linear_int4(x, w._replace(group=48), loads), NotImplementedError, "groups"),
            (lambda: grouped_linear_int4(x, w._replace(group=64), loads), RuntimeError, "scales"),
            (lambda: grouped_linear_int4(x, w._replace(out_features=40), loads), RuntimeError, "values"),
            (lambda: grouped_linear_int4(x, w._replace(values=w.values.int()), loads), RuntimeError, "values"),
            (lambda: grouped_linear_int4(x, w._replace(scales=w.scales.double()), loads), NotImplementedError, "scale data type"),
            (lambda: grouped_linear_int4(x, w._replace(zeros=w.zeros.int()), loads), RuntimeError, "zeros"),
            (lambda: grouped_linear_int4(x, w, loads.long()), RuntimeError, "int32"),
            (lambda: grouped_linear_int4(x, w, loads[:1]), RuntimeError, "one load per expert"),
            (lambda: grouped_linear_int4(x, w, loads, bias=bias[:, :4]), RuntimeError, "bias"),
            (lambda: grouped_linear_int4(x, w, loads, row_entries=entries.long()), RuntimeError, "int32"),
            (lambda: grouped_linear_int4(x, w, loads, row_entries=entries[None]), RuntimeError, "vector"),
            (lambda: grouped_linear_int4(x, w, loads, row_entries=entries, entries_per_cell=0), RuntimeError, "at least one"),
            (lambda: grouped_linear_int4(x, w, loads, out=room[:4]), RuntimeError, "contiguous"),
            (lambda: grouped_linear_int4(x, w, loads, out=room, out_dtype=torch.float32), RuntimeError, "says its type"),
            (lambda: grouped_linear_int4(x, w, loads, out=x.view(-1)[:100].view(5, 20)), RuntimeError, "shares memory"),
            (lambda: grouped_linear_int4(x, w, loads, out=room.clone().requires_grad_()), RuntimeError, "carries gradients")):
        with pytest.raises(error, match=words):
            call()
    leaf = torch.ones_like(room, requires_grad=True)
    product = leaf * room
    grouped_linear_int4(x, w, loads, out=room)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        made = torch.zeros_like(room)
        assert torch.equal(grouped_linear_int4(x, w, loads, out=made), room)


def test_argument_errors_of_the_library_need_no_gpu():
    call = _lib.lib().brt_hip_grouped_gemm_int4
    some = 16  # an address that is never read: every call ends before a launch
    good = dict(x=some, x_dtype=2, entries=None, per_cell=1, T=4, w=some, scales=some, s_dtype=2, zeros=None, group=128, loads=some, bias=None, bias_dtype=0,
                out=some, out_dtype=2, E=2, P=4, N=16, K=64, act=0, stream=None)

    def code(**change):
        return call(*{**good, **change}.values())

    assert code(P=0) == 0 and code(N=0) == 0
    for change in ({"E": 0}, {"P": -1}, {"N": -1}, {"K": -8}, {"x": None}, {"w": None}, {"scales": None}, {"loads": None}, {"out": None},
                   {"entries": some, "per_cell": 0}, {"entries": some, "T": -1}):
        assert code(**change) == -1, change
    for change in ({"group": 16}, {"x_dtype": 3}, {"out_dtype": 5}, {"s_dtype": -1}, {"bias": some, "bias_dtype": 9}, {"act": 4}, {"K": 0}, {"K": 60}, {"x": 24},
                   {"w": 24}, {"scales": 24}, {"zeros": 18}, {"P": 1 << 24}, {"N": (1 << 28) + 1}, {"K": (1 << 28) + 8}, {"E": (1 << 28) + 1},
                   {"P": (1 << 24) - 1, "N": 1 << 28, "E": 1 << 28}, {"P": (1 << 24) - 1, "N": 1 << 20}, {"x_dtype": 0, "P": (1 << 24) - 1, "N": 2048}):
        assert code(**change) == -4, change

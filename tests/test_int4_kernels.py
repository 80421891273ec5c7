"""Every kernel of the products with 4-bit weights at the values, loads and layouts where it can go wrong, against the definition in 64 bits.

Bounds as in ``test_int4`` (``assert_near``), and what is left of them where numbers are tiny: the third part of an fp32 element is a multiple of
2^-133, so the element is off by at most 2^-134; sums and their products with scales are held in units of 2^-15 with the fp32 grid's 2^-149, so an
addition to a result is off by at most 2^-135 beside its relative error.
"""
import pytest
import torch

from brainstorm_amd import _lib
from brt.jit import grouped_linear_int4, pack_int4
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

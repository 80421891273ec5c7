"""Products in 8-bit floating point with block scales, against the definition in 64 bits, and their refusals.

Quantization is exact arithmetic with named roundings: bits are compared.  A product's terms are exact in fp32; for an fp32
result a block's sum is within 128 * 2^-23 of the sum of the terms' magnitudes (128 additions, each off by at most a step), its
scale adds two roundings (sx * sw, and the multiply-add), the sum over KB blocks KB more, the bias one: (128 + KB + 3) * 2^-23 of
the magnitudes in all.  For 16-bit results the matrix instruction keeps 13 bits below the largest of (at most) 16 products that it
adds at once: a term is off by less than 2^-13 of that largest one, 16 of them by 2^-9 of it, so a sum by 2^-9 of the magnitudes;
and as these errors have both signs, the norm of all of them stays under 2^-14 of the result's (1.3e-5 measured), which is
asked for beside half a step of the type (0.6 of it in the mean square).  GELU is within 4.3e-6 and passes an error on at most
1.13-fold.  The last rounding is half a step (``eps / 2``) of the value.
"""
import pytest
import torch

from brt.jit import grouped_linear_fp8, quantize_rows

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def quantized_here(x):
    """The definition on the host: (q, scales), every operation rounded in fp32."""
    rows, d = x.shape
    padded = torch.zeros(rows, -(-d // 128) * 128)
    padded[:, :d] = x.float()
    blocks = padded.view(rows, -1, 128)
    top = blocks.abs().amax(2)
    top = torch.where(top < 2.0 ** -100, torch.tensor(2.0 ** -100), top)
    q = (blocks * (top.reciprocal() * 448.0)[:, :, None]).to(F8).view(torch.uint8).view(rows, -1)[:, :d]
    return q.contiguous().view(F8), top / 448.0


def weights(seed, experts, n, k):
    nb, kb = -(-n // 128), -(-k // 128)
    gen = torch.Generator().manual_seed(seed)
    q = normal(seed, experts, n, k, scale=60.0).clamp(-448, 448).to(F8)
    return q, torch.rand(experts, nb, kb, generator=gen) * 1e-3 + 1e-4


def spread(scales, n, k):
    return scales.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def loads_of(seed, rows, experts, empty=()):
    gen = torch.Generator().manual_seed(seed)
    share = torch.rand(experts, generator=gen) ** 2
    for e in empty:
        share[e] = 0
    return torch.bincount(torch.multinomial(share, rows, True, generator=gen), minlength=experts).int() if rows else torch.zeros(experts, dtype=torch.int32)


def product_in_64(xq, xs, w, ws, loads, bias=None, activation=None):
    """(result, magnitudes of the terms) of packed rows; rows behind the last expert's are NaN."""
    rows, k = xq.shape
    n = w.shape[1]
    x = xq.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    want = torch.full((rows, n), float("nan"), dtype=torch.float64)
    size = torch.zeros(rows, n, dtype=torch.float64)
    first = 0
    for e, load in enumerate(loads.tolist()):
        here = slice(first, first + load)
        values = w[e].double() * spread(ws[e], n, k)
        want[here], size[here] = x[here] @ values.t(), x[here].abs() @ values.abs().t()
        if bias is not None:
            want[here] += bias[e].double()
            size[here] += bias[e].double().abs()
        first += load
    if activation == "gelu":
        want = torch.nn.functional.gelu(want)
    elif activation == "relu":
        want = torch.where(want < 0, torch.zeros_like(want), want)
    return want, size


def assert_near(got, want, size, kb, gelu=False, exact=None):
    got, kept = got.cpu(), ~want.isnan()
    info = torch.finfo(got.dtype)
    exact = got.dtype == torch.float32 if exact is None else exact
    off = ((128 + kb + 3) * 2.0 ** -23 + (0.0 if exact else 2.0 ** -9)) * size * (1.13 if gelu else 1.0) + (4.3e-6 if gelu else 0.0)
    bound = off + info.eps / 2 * (want.abs() + off) + info.tiny * info.eps
    far = ((got.double() - want).abs() / bound)[kept]
    assert not far.numel() or float(far.max()) <= 1.0, f"{float(far.max())} of the bound"
    if not exact and far.numel() >= 64:
        rel = float((got.double() - want)[kept].norm() / want[kept].norm())
        assert rel <= 0.6 * info.eps + 2.0 ** -14 + (4.3e-6 / float(want[kept].square().mean().sqrt()) if gelu else 0.0), rel


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,d", [(1, 16), (1, 128), (3, 144), (8, 256), (9, 2048), (65, 1008), (300, 4096), (1000, 128)])
def test_quantized_rows(rows, d, dtype):
    x = normal(rows + d, rows, d, dtype=TYPES[dtype])
    x[0] = 0
    if rows > 2:
        x[1, : d // 2] *= 1e-4
        x[2] = torch.linspace(-1, 1, d)
    q, scales = quantize_rows(x.cuda())
    want_q, want_scales = quantized_here(x)
    assert q.dtype == F8 and q.shape == x.shape and scales.shape == want_scales.shape
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(q.contiguous().view(torch.uint8).cpu(), want_q.view(torch.uint8))


@pytest.mark.gpu
def test_every_16_bit_value_is_rounded_as_torch_rounds_it():
    for dtype in (torch.bfloat16, torch.float16):
        bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.uint16).view(torch.int16)
        x = bits.view(dtype).view(-1, 16).repeat(1, 8).contiguous()
        x = x[torch.isfinite(x.float()).all(1)]
        q, scales = quantize_rows(x.cuda())
        want_q, want_scales = quantized_here(x)
        assert torch.equal(scales.cpu(), want_scales) and torch.equal(q.view(torch.uint8).cpu(), want_q.view(torch.uint8))


@pytest.mark.gpu
def test_blocks_with_nan_and_infinity_and_tiny_values():
    x = normal(1, 6, 256)
    x[0, 3], x[1, 200], x[2, :128] = float("nan"), float("inf"), 1e-40
    x[3, 128:] = -0.0
    q, scales = quantize_rows(x.cuda())
    q, scales = q.float().cpu(), scales.cpu()
    assert scales[0, 0].isnan() and q[0, :128].isnan().all() and torch.isfinite(q[0, 128:]).all()
    assert scales[1, 1] == float("inf") and q[1, 200].isnan()
    assert scales[2, 0] == 2.0 ** -100 / 448 and torch.isfinite(q).logical_or(torch.zeros_like(q) + (torch.arange(6)[:, None] < 2)).all()
    assert not q[3, 128:].any()
    w, ws = weights(2, 1, 64, 256)
    out = grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), torch.tensor([6], dtype=torch.int32, device="cuda"))
    assert out[0].isnan().all() and out[1].isnan().all() and torch.isfinite(out[2:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,n,experts", [(6, 256, 64, 1), (40, 256, 72, 3), (200, 256, 384, 2), (1000, 384, 144, 1), (3000, 272, 3008, 60),
                                              (3100, 128, 4112, 3), (2200, 256, 16400, 2)])
def test_activations_hand_nan_on(rows, k, n, experts, dtype, activation):
    """Rows that hold NaN or an infinity are NaN in every kind of kernel, also as blocks; the rows beside them keep their bits."""
    w, ws = (t.cuda() for t in weights(2, experts, n, k))
    loads, bias = loads_of(3, rows, experts).cuda(), normal(4, experts, n).cuda()
    good = normal(1, rows, k, dtype=TYPES[dtype]).cuda()
    x = good.clone()
    bad = torch.tensor([0, rows // 2, rows - 1], device="cuda")
    x[bad[0], 3], x[bad[1], k - 1], x[bad[2], k // 2] = float("nan"), float("inf"), float("-inf")
    kept = torch.ones(rows, dtype=torch.bool, device="cuda").index_fill(0, bad, False)
    out = grouped_linear_fp8(x, w, ws, loads, bias=bias, activation=activation)
    assert out[bad].isnan().all()
    assert torch.equal(out[kept], grouped_linear_fp8(good, w, ws, loads, bias=bias, activation=activation)[kept])
    if n % 16 == 0:
        q, scales = grouped_linear_fp8(x, w, ws, loads, bias=bias, activation=activation, out_blocks=True)
        assert scales[bad].isnan().all() and q[bad].float().isnan().all()
        want, want_scales = grouped_linear_fp8(good, w, ws, loads, bias=bias, activation=activation, out_blocks=True)
        assert torch.equal(scales[kept], want_scales[kept]) and torch.equal(q[kept].view(torch.uint8), want[kept].view(torch.uint8))


CASES = [  # rows, in, out, experts
    (1, 16, 1, 1), (1, 128, 64, 1), (1, 2048, 520, 4), (2, 1040, 129, 3), (5, 272, 136, 8), (17, 144, 72, 2), (48, 1024, 512, 8),
    (33, 512, 4, 1), (64, 640, 260, 1), (100, 384, 256, 130), (129, 256, 136, 1), (300, 2064, 200, 2), (700, 128, 384, 4),
    (513, 528, 264, 1), (777, 1152, 520, 2), (1500, 400, 300, 3),
    # every kind of tile, with lists that workgroups walk in several tiles: see launch_any_tiles
    (200, 256, 8200, 8), (2600, 144, 1030, 2), (3000, 272, 3000, 60), (3100, 128, 4104, 3), (2200, 256, 16400, 2), (900, 384, 2056, 120),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", ["plain", "gelu_bias", "relu", "rows_behind"])
@pytest.mark.parametrize("rows,k,n,experts", CASES)
def test_products(rows, k, n, experts, form, dtype):
    dtype = TYPES[dtype]
    x = normal(rows, rows, k, dtype=dtype)
    w, ws = weights(k, experts, n, k)
    loads = loads_of(n, rows - rows // 3 if form == "rows_behind" else rows, experts, empty=(0,) if experts > 2 else ())
    bias = normal(4, experts, n, dtype=dtype) if form == "gelu_bias" else None
    activation = {"gelu_bias": "gelu", "relu": "relu"}.get(form)
    xq, xs = quantized_here(x)
    want, size = product_in_64(xq, xs, w, ws, loads, bias, activation)
    out = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    bias = None if bias is None else bias.cuda()
    got = grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda(), bias=bias, activation=activation, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert_near(got, want, size, -(-k // 128), activation == "gelu")
    behind = int(loads.sum())
    assert bool((got[behind:] == 7.0).all())  # rows behind the last expert's: as they were
    # the rows quantized beforehand give the same bits
    again = grouped_linear_fp8(*([xq.cuda()] + [w.cuda(), ws.cuda(), loads.cuda()]), bias=bias, activation=activation,
                               x_scales=xs.cuda(), out_dtype=dtype)
    assert torch.equal(again[:behind], got[:behind])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("activation", ["gelu", "relu", None])
@pytest.mark.parametrize("rows,k,n,experts", [(3, 256, 512, 2), (200, 256, 384, 2), (900, 512, 512, 2), (1000, 384, 144, 1), (3000, 272, 3008, 60),
                                              (2600, 144, 1040, 2), (3100, 128, 4112, 3), (2200, 256, 16400, 2)])
def test_result_in_blocks_is_the_quantized_result(rows, k, n, experts, activation, dtype):
    x, (w, ws) = normal(1, rows, k, dtype=TYPES[dtype]).cuda(), (t.cuda() for t in weights(2, experts, n, k))
    loads, bias = loads_of(3, rows, experts).cuda(), normal(4, experts, n).cuda()
    out = grouped_linear_fp8(x, w, ws, loads, bias=bias, activation=activation)
    q, scales = grouped_linear_fp8(x, w, ws, loads, bias=bias, activation=activation, out_blocks=True)
    want_q, want_scales = quantize_rows(out)
    assert q.shape == out.shape and torch.equal(scales, want_scales)
    assert torch.equal(q.contiguous().view(torch.uint8), want_q.contiguous().view(torch.uint8))
    # columns behind the last one are zeros: the next product reads whole blocks
    padded = torch.as_strided(q.view(torch.uint8), (rows, q.stride(0)), (q.stride(0), 1))
    assert not padded[:, n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n,experts", [(5, 1024, 520, 2), (200, 512, 256, 2), (1500, 384, 300, 3), (3000, 272, 3000, 60), (3100, 128, 4104, 3)])
def test_fp32_results_of_the_8_bit_instruction(rows, k, n, experts):
    x, (w, ws) = normal(1, rows, k, dtype=torch.bfloat16), weights(2, experts, n, k)
    loads = loads_of(3, rows, experts)
    xq, xs = quantized_here(x)
    want, size = product_in_64(xq, xs, w, ws, loads)
    got = grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda(), out_dtype=torch.float32, exact=False)
    assert_near(got, want, size, -(-k // 128), exact=False)
    # rounded to 16 bits it is the 16-bit result
    assert torch.equal(got.bfloat16(), grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda()))
    with pytest.raises(NotImplementedError, match="exact products"):
        grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda(), exact=True)


@pytest.mark.gpu
def test_bits_of_a_row_do_not_depend_on_the_rows_beside_it():
    """Kernels differ by the rows an expert has; the sums and their order are the same."""
    k, n = 1024, 640
    w, ws = (t.cuda() for t in weights(1, 1, n, k))
    x = normal(2, 2000, k, dtype=torch.bfloat16).cuda()
    whole = grouped_linear_fp8(x, w, ws, torch.tensor([2000], dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    for rows in (1, 16, 17, 64, 100, 300):
        part = grouped_linear_fp8(x[:rows], w, ws, torch.tensor([rows], dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
        torch.testing.assert_close(part, whole[:rows], rtol=1e-5, atol=1e-5 * float(whole.abs().max()))


@pytest.mark.gpu
def test_strides_types_and_loads_that_do_not_fit():
    k, n = 256, 128
    w, ws = (t.cuda() for t in weights(1, 2, n, k))
    x = normal(2, 40, k, dtype=torch.bfloat16).cuda()
    loads = torch.tensor([25, 15], dtype=torch.int32, device="cuda")
    want = grouped_linear_fp8(x, w, ws, loads)
    wide = torch.zeros(40, 2 * k, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(grouped_linear_fp8(wide[:, ::2], w, ws, loads), want)
    flat = torch.empty(40 * k + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.equal(grouped_linear_fp8(flat[1:].view(40, k), w, ws, loads), want)
    q, scales = quantize_rows(x)
    rows = torch.zeros(40, k + 48, dtype=torch.uint8, device="cuda").view(F8)
    rows[:, :k] = q
    assert torch.equal(grouped_linear_fp8(rows[:, :k], w, ws, loads, x_scales=scales.contiguous()), want)
    out = torch.empty(40, n, dtype=torch.float16, device="cuda")
    grouped_linear_fp8(x, w, ws, loads, out=out)
    assert torch.equal(out, grouped_linear_fp8(x, w, ws, loads, out_dtype=torch.float16))
    # loads beyond the rows that there are, and below zero: rows are bounded by what x holds
    odd = torch.tensor([-3, 1000], dtype=torch.int32, device="cuda")
    alone = grouped_linear_fp8(x, w[1:], ws[1:], torch.tensor([40], dtype=torch.int32, device="cuda"))
    assert torch.equal(grouped_linear_fp8(x, w, ws, odd), alone)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [7, 300, 3000])
def test_loads_that_name_more_rows_than_there_are(rows):
    """Rows behind the last one do not exist, whatever the loads say: results of the first rows are those of loads that fit."""
    k, n, experts = 128, 1040, 5
    w, ws = (t.cuda() for t in weights(1, experts, n, k))
    x = normal(2, rows, k, dtype=torch.bfloat16).cuda()
    first = rows // 3
    fits = torch.tensor([first, 0, rows - first, 0, 0], dtype=torch.int32, device="cuda")
    want = grouped_linear_fp8(x, w, ws, fits)
    most = 2 ** 31 - 1
    for odd in ([first, -5, most, most, most], [first, 0, rows, rows, 1], [first, -most - 1, rows - first, 7, -1]):
        got = grouped_linear_fp8(x, w, ws, torch.tensor(odd, dtype=torch.int32, device="cuda"))
        assert torch.equal(got, want)
    # ... and where the loads are added up in several passes
    w, ws = w[:1].expand(130, -1, -1).contiguous(), ws[:1].expand(130, -1, -1).contiguous()
    want = grouped_linear_fp8(x, w[:1], ws[:1], torch.tensor([rows], dtype=torch.int32, device="cuda"))
    for load in (rows, most):
        assert torch.equal(grouped_linear_fp8(x, w, ws, torch.full((130,), load, dtype=torch.int32, device="cuda")), want)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [144, 1024])
@pytest.mark.parametrize("loads", [[4600, 0], [4290, 310], [256 * 17, 248], [4000, 129], [2100, 128, 2200, 172], [1, 4599]])
def test_a_last_round_of_few_tiles(loads, k):
    """288 to 320 tiles of 256 x 256, or 576 to 624 of 128 x 256: the last round's are dealt out by halves, of which the second may be empty."""
    n, rows = 4096, 4600
    w, ws = weights(1, len(loads), n, k)
    loads = torch.tensor(loads, dtype=torch.int32)
    x = normal(2, rows, k, dtype=torch.bfloat16)
    xq, xs = quantized_here(x)
    want, size = product_in_64(xq, xs, w, ws, loads)
    for dtype in (torch.bfloat16, torch.float16):
        out = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
        assert_near(grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda(), out=out), want, size, -(-k // 128))
        assert bool((out[int(loads.sum()):] == 7.0).all())
    q, scales = grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda(), out_blocks=True)
    last = int(loads.sum())
    plain = quantize_rows(grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda())[:last])
    assert torch.equal(scales[:last], plain[1])  # (both kinds of tiles add up the blocks from the first on)
    assert torch.equal(q[:last].view(torch.uint8), plain[0].view(torch.uint8))


@pytest.mark.gpu
def test_many_experts():
    """More than the list in LDS holds: the kernel for few rows takes them, with any number of rows."""
    k, n, experts = 144, 72, 600
    w, ws = weights(1, experts, n, k)
    for rows in (5, 40000):
        x, loads = normal(2, rows, k, dtype=torch.bfloat16), loads_of(3, rows, experts)
        xq, xs = quantized_here(x)
        want, size = product_in_64(xq, xs, w, ws, loads)
        assert_near(grouped_linear_fp8(x.cuda(), w.cuda(), ws.cuda(), loads.cuda()), want, size, 2)


@pytest.mark.gpu
def test_two_calls_at_once_and_scales_beyond_the_ordinary():
    """Two streams at the same time; scales of e4m3 weights up to the largest fp32 can be multiplied with, and zero."""
    k, n = 512, 512
    w, ws = (t.cuda() for t in weights(1, 2, n, k))
    ws[0, 1], ws[1, 0] = 0.0, 3e30
    xs = [normal(s, 900, k, dtype=torch.bfloat16).cuda() for s in (2, 3)]
    loads = torch.tensor([400, 500], dtype=torch.int32, device="cuda")
    want = [grouped_linear_fp8(x, w, ws, loads) for x in xs]
    assert not want[0][:400, 128:256].any() and torch.isfinite(want[0].float()).all()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(grouped_linear_fp8(xs[i], w, ws, loads))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.gpu
def test_no_rows():
    w, ws = (t.cuda() for t in weights(1, 2, 64, 128))
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda")
    assert grouped_linear_fp8(x, w, ws, none).shape == (0, 64)
    q, scales = grouped_linear_fp8(x, w, ws, none, out_blocks=True)
    assert q.shape == (0, 64) and scales.shape == (0, 1)
    assert quantize_rows(x)[0].shape == (0, 128)


@pytest.mark.gpu
def test_on_a_stream_and_replayed():
    k, n, experts = 512, 384, 4
    w, ws = (t.cuda() for t in weights(1, experts, n, k))
    for rows in (6, 200, 1200):
        x, loads = normal(2, rows, k, dtype=torch.bfloat16).cuda(), loads_of(3, rows, experts).cuda()
        want = grouped_linear_fp8(x, w, ws, loads, activation="gelu")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = grouped_linear_fp8(x, w, ws, loads, activation="gelu")
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = grouped_linear_fp8(x, w, ws, loads, activation="gelu")
        for seed in (5, 6, 7):
            x.copy_(normal(seed, rows, k, dtype=torch.bfloat16))
            loads.copy_(loads_of(seed, rows, experts))
            graph.replay()
            eager = grouped_linear_fp8(x, w, ws, loads, activation="gelu")
            torch.cuda.synchronize()
            assert torch.equal(held, eager)


@pytest.mark.gpu
def test_refusals():
    k, n = 256, 128
    w, ws = (t.cuda() for t in weights(1, 2, n, k))
    x, loads = normal(2, 8, k, dtype=torch.bfloat16).cuda(), torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    ok = lambda **more: grouped_linear_fp8(more.pop("x", x), more.pop("w", w), more.pop("ws", ws), more.pop("loads", loads), **more)  # noqa: E731
    with pytest.raises(NotImplementedError, match="float8_e4m3fn"):
        ok(w=w.to(torch.bfloat16))
    with pytest.raises(RuntimeError, match="weight must be|x must be"):
        ok(x=x[:, :128])
    with pytest.raises(RuntimeError, match="weight_scales"):
        ok(ws=ws[:, :, :1])
    with pytest.raises(RuntimeError, match="weight_scales"):
        ok(ws=ws.double())
    with pytest.raises(RuntimeError, match="one load per expert"):
        ok(loads=loads[:1])
    with pytest.raises(RuntimeError, match="int32"):
        ok(loads=loads.long())
    with pytest.raises(RuntimeError, match="bias must be"):
        ok(bias=torch.zeros(n, device="cuda"))
    with pytest.raises(RuntimeError, match="x_scales belong"):
        ok(x_scales=torch.ones(8, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="x_scales belong"):
        ok(x=quantize_rows(x)[0])
    with pytest.raises(RuntimeError, match="x_scales must be"):
        ok(x=quantize_rows(x)[0], x_scales=torch.ones(8, 1, device="cuda"))
    with pytest.raises(RuntimeError, match="contiguous"):
        ok(out=torch.zeros(n, 8, device="cuda").t())
    with pytest.raises(RuntimeError, match="out is given"):
        ok(out=torch.zeros(8, n, device="cuda"), out_blocks=True)
    both = torch.zeros(16, n, device="cuda")
    with pytest.raises(RuntimeError, match="shares memory"):
        ok(w=w[:, :, :n].contiguous(), ws=ws[:, :, :1], x=both[4:12], out=both[:8])
    assert torch.equal(ok(w=w[:, :, :n].contiguous(), ws=ws[:, :, :1], x=both[8:], out=both[:8]), torch.zeros(8, n, device="cuda"))
    with pytest.raises(RuntimeError, match="shares memory"):
        table = torch.zeros(2, n, device="cuda")
        ok(x=x[:2], bias=table, out=table)
    with pytest.raises(NotImplementedError):
        ok(out_dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        ok(x=x.double())
    with pytest.raises(KeyError):
        ok(activation="tanh")
    with pytest.raises(NotImplementedError, match="multiple of 16 columns"):
        ok(w=w[:, :100].contiguous(), ws=ws, out_blocks=True)
    with pytest.raises(NotImplementedError, match="units of 16"):
        quantize_rows(torch.zeros(4, 40, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ok(x=x.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ok(loads=loads.cpu())


def test_arguments_are_checked_before_anything_runs():
    from brainstorm_amd import _lib

    lib = _lib.lib()
    assert lib.brt_hip_quantize_rows(None, 4, 128, 0, None, 64, None, None) == -1 and b"pitch" in lib.brt_hip_last_error()
    assert lib.brt_hip_quantize_rows(None, 4, 128, 9, None, 128, None, None) == -4
    assert lib.brt_hip_quantize_rows(None, 4, 128, 0, None, 128, None, None) == -1
    assert lib.brt_hip_quantize_rows(None, 0, 128, 0, None, 128, None, None) == 0
    call = lambda E=2, P=4, N=64, K=128, pitch=128, act=0, out=0: lib.brt_hip_grouped_gemm_fp8(  # noqa: E731
        None, 0, pitch, None, None, None, None, None, 0, None, out, None, E, P, N, K, act, 0, None)
    assert call() == -1 and call(E=0) == -1 and call(pitch=64) == -1 and call(act=5) == -4 and call(out=7) == -4
    assert lib.brt_hip_grouped_gemm_fp8(16, 0, 1 << 21, 16, 16, 16, 16, None, 0, 16, 0, None, 2, 4, 64, 1 << 21, 0, 0, None) == -4
    assert lib.brt_hip_grouped_gemm_fp8(16, 0, 128, 16, 16, 16, 16, None, 0, 16, 0, None, 2, 1 << 24, 64, 128, 0, 0, None) == -4
    assert lib.brt_hip_grouped_gemm_fp8(16, 0, 128, 16, 16, 16, 16, None, 0, 16, 0, 16, 2, 4, 64, 128, 0, 0, None) == -4
    assert lib.brt_hip_grouped_gemm_fp8(16, 0, 128, 16, 16, 16, 16, None, 0, 16, 2, None, 2, 4, 64, 128, 0, 1, None) == -4
    assert lib.brt_hip_grouped_gemm_fp8(16, 2, 128, None, 16, 16, 16, None, 0, 16, 2, None, 2, 4000, 640, 128, 0, 0, None) == -4
    assert lib.brt_hip_grouped_gemm_fp8(8, 0, 128, 16, 16, 16, 16, None, 0, 16, 0, None, 2, 4, 64, 128, 0, 0, None) == -4
    assert call(P=0) == 0 and call(N=0) == 0 and call(K=0, pitch=0) == -4
    assert lib.brt_hip_gate_topk_grad(None, None, None, None, None, 4, 4, 5, 0, 1, None) == -1
    assert lib.brt_hip_gate_topk_grad(None, None, None, None, None, 4, 2000, 1, 0, 1, None) == -4
    assert lib.brt_hip_gate_topk_grad(None, None, None, None, None, 4, 8, 1, 0, 1, None) == -1
    assert lib.brt_hip_gate_topk_grad(None, None, None, None, None, 1 << 30, 8, 1, 0, 1, None) == -4
    grads = lib.brt_hip_dispatch_by_rows_grad
    assert grads(None, None, None, None, None, None, 4, 0, 8, 4, 0, None) == -1
    assert grads(None, None, None, None, None, None, 4, 9, 8, 4, 0, None) == -4
    assert grads(None, None, None, None, None, None, 4, 1, 7, 4, 0, None) == -4
    assert grads(None, None, None, None, 16, None, 4, 1, 8, 4, 0, None) == -1
    assert grads(None, None, None, None, 16, None, 1 << 30, 4, 8, 4, 0, None) == -4
    back = lib.brt_hip_combine_by_rows_grad
    assert back(None, None, None, None, None, None, None, None, 4, 1, 8, 4, 1, 2, None) == -4
    assert back(None, None, None, None, None, None, 16, None, 4, 1, 8, 4, 0, 0, None) == -1


def test_dimensions_that_do_not_fit_in_32_bits_once_rounded_up():
    from brainstorm_amd import _lib

    lib = _lib.lib()
    last = 2 ** 31 - 16
    assert lib.brt_hip_quantize_rows(None, 1, last, 0, None, last, None, None) == -1 and b"pitch" in lib.brt_hip_last_error()
    call = lambda E, N: lib.brt_hip_grouped_gemm_fp8(  # noqa: E731
        16, 0, 128, 16, 16, 16, 16, None, 0, 16, 0, None, E, 4, N, 128, 0, 0, None)
    assert call(2, 2 ** 31 - 1) == -4 and b"columns" in lib.brt_hip_last_error()
    assert call(2 ** 31 - 1, 128) == -4 and b"columns" in lib.brt_hip_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cells", [1, 17, 300, 3000])
def test_a_served_layer_of_all_operators(cells):
    """Gate, route, dispatch, an expert FFN of two such products and the combine, against the same steps in 64 bits with the hidden
    rows rounded to bf16 as the layer holds them (a value near a border of e4m3 may be rounded to the other side: 1.4e-2 of the
    norm is half of what rounding to e4m3 itself costs)."""
    import brt._C.router as c_router

    experts, d, d_ff, k = 4, 256, 400, 2
    w1, s1 = weights(1, experts, d_ff, d)
    w2, s2 = weights(2, experts, d, d_ff)
    x, scores = normal(3, cells, d, dtype=torch.bfloat16), normal(4, cells, experts)
    dev = [t.cuda() for t in (w1, s1, w2, s2)]
    ids, weight = c_router.gate_topk(scores.cuda(), k, softmax=True)
    loads, _, seat_rows, row_entries = c_router.route_by_path(ids, experts)
    rows = c_router.dispatch_by_rows(x.cuda(), row_entries, k)
    hidden, scales = grouped_linear_fp8(rows, dev[0], dev[1], loads, activation="gelu", out_blocks=True)
    y = grouped_linear_fp8(hidden, dev[2], dev[3], loads, x_scales=scales)
    out = c_router.combine_by_rows(y, ids, seat_rows, weight)

    loads = loads.cpu()
    xq, xs = quantized_here(rows.cpu())
    h, _ = product_in_64(xq, xs, w1, s1, loads, activation="gelu")
    hq, hs = quantized_here(h.to(torch.bfloat16))
    want, _ = product_in_64(hq, hs, w2, s2, loads)
    want = (want[seat_rows.cpu().long() - 1] * weight.cpu().double()[:, :, None]).sum(1)
    assert float((out.cpu().double() - want).norm() / want.norm()) <= 1.4e-2

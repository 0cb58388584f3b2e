"""8-bit floats with a scale for each block of 128: rounding to them and back, the norm that ends in them, products of them.

Tolerances, from the formulas.  Rounding to e4m3 is compared bit for bit with the definition in float32.  Where the input of the rounding
is itself computed, a value v of a block with the scale s lands within half a step of it: 2^-4 |v|, or 2^-10 s where e4m3 is subnormal,
and the error of v comes on top.  The norm's factor is off by a float32 sum of squares in at most 110 additions a term (110 * 2^-24 of
the sum, half of it in the root) and six single roundings, below 2^-17 of a value.

A product's sum over a block of 128 has exact products (4 bits times 4), which the tensor core adds in float32; an addition, whatever
its order, rounds or cuts off at most 2^-23 of the block's sum of magnitudes, so 128 of them at most 2^-16 of it.  Each block's sum is
multiplied by its factor (rounded once) and added once, at most 2^-23 of the magnitudes so far, and the slices and the bias come to at
most 10 additions more.  With A the sum of all magnitudes, scaled, and B blocks: |error| <= (2^-16 + (B + 12) 2^-23) A, and half a unit
of the output's last place.  (What a wrong block would do: A / B of the magnitudes, at least 2^-8 A for the sizes below.)

The gated unit g * sigmoid(g) * u has slopes of at most 1.1 |u| and |g sigmoid(g)| in the errors of g and u; its exponential and division
are off by a few 2^-22 in the approximate form that bfloat16 outputs take, and by a few 2^-24 in float32."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def ops():
    from slipstream_b200 import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def fp8_values(g, n, k, extra=0):
    """Random e4m3 with a stride of 16s and ``extra`` bytes more, NaN between the rows."""
    stride = -(-k // 16) * 16 + extra
    store = torch.full((n, stride), 127, device=DEV, dtype=torch.uint8).view(E4M3)
    store[:, :k] = (normal(g, n, k) * 150).clamp_(-448, 448).to(E4M3)
    return store[:, :k]


def blocks_of(n):
    return -(-n // 128)


def fp8_rows(g, n, k, extra=0, turned=False):
    scales = torch.rand(n, blocks_of(k), generator=g, device=DEV) * 0.01 + 1e-4
    return ops().Fp8Rows(fp8_values(g, n, k, extra), scales.t().contiguous().t() if turned else scales)


def fp8_blocks(g, f, k, extra=0):
    return ops().Fp8Blocks(fp8_values(g, f, k, extra), torch.rand(blocks_of(f), blocks_of(k), generator=g, device=DEV) * 0.01 + 1e-4)


def spread(scales, shape, rows):
    """Scales of blocks as a matrix of the values' shape."""
    full = scales.repeat_interleave(128, dim=1)[:, : shape[1]]
    return full if rows == 1 else full.repeat_interleave(128, dim=0)[: shape[0]]


def values_of(x, dtype=F64):
    return x.values.to(dtype) * spread(x.scales.to(dtype), x.shape, 1 if isinstance(x, ops().Fp8Rows) else 128)


def tops_of(v, rows):
    n, k = v.shape
    padded = v.new_zeros(-(-n // rows) * rows, blocks_of(k) * 128)
    padded[:n, :k] = v
    return padded.reshape(-1, rows, blocks_of(k), 128).abs().amax(dim=(1, 3))


def check_definition(got, x, rows):
    """Bit for bit: scale = a / 448, q = e4m3(x * (448 / a)) in float32."""
    v = x.float()
    top = tops_of(v, rows)
    assert torch.equal(got.scales, top / torch.full_like(top, 448.0))
    inverse = torch.where(top > 0, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    assert got.values.dtype == E4M3 and got.values.shape == x.shape and got.values.stride(0) % 16 == 0
    assert torch.equal(got.values.view(torch.uint8), (v * spread(inverse, v.shape, rows)).to(E4M3).view(torch.uint8))


def check_near(got, v, slack):
    """Rows whose input is known to ``slack`` (a tensor like v, absolute)."""
    q, s = got.values.to(F64), spread(got.scales.to(F64), v.shape, 1)
    assert torch.all((q * s - v).abs() <= v.abs() * (2.0 ** -4 + 2.0 ** -16) + s * (2.0 ** -10 + 2.0 ** -16) + slack * 1.1)
    top, off = tops_of(v, 1), tops_of(slack, 1)
    assert torch.all((got.scales.to(F64) - top / 448).abs() <= (top * 2.0 ** -22 + off) / 448 + 1e-40)


WIDTHS = [1, 3, 16, 17, 127, 128, 129, 255, 896, 1001, 2051, 3584, 8193, 18944]


# --------------------------------------------------------------------------- rounding

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_rows(dtype, width):
    for rows, pad, shift in [(1, 0, 0), (5, 0, 0), (7, 8, 8), (6, 5, 1), (700 if width < 4000 else 301, 16, 0)]:
        x = normal(gen(width + rows), rows, width + pad, dtype=dtype)[:, shift:shift + width]
        for activations in (False, True):
            got = ops().quantize_rows_fp8(x, activations=activations)
            assert isinstance(got, ops().Fp8Rows) and got.scales.shape == (rows, blocks_of(width))
            check_definition(got, x, 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width", [(1, 1), (1, 3584), (127, 128), (128, 129), (129, 17), (300, 1001), (513, 896), (640, 4100)])
def test_quantize_blocks(dtype, rows, width):
    for pad, shift in [(0, 0), (8, 8), (5, 1)]:
        x = normal(gen(width + rows), rows, width + pad, dtype=dtype)[:, shift:shift + width]
        got = ops().quantize_blocks_fp8(x)
        assert isinstance(got, ops().Fp8Blocks) and got.scales.shape == (blocks_of(rows), blocks_of(width))
        check_definition(got, x, 128)


@pytest.mark.parametrize("blocks", [False, True])
def test_quantize_special_values(blocks):
    o = ops()
    x = normal(gen(3), 256, 384)
    x[0], x[2] = 0, 0
    x[3] *= 1e-37
    x[4] *= 1e37
    x[5, 128:256] = 0
    for r, v in ((6, float("inf")), (7, -float("inf")), (8, float("nan"))):
        x[r, 200] = v
    x[9] = 1e-45
    call = o.quantize_blocks_fp8 if blocks else o.quantize_rows_fp8
    if blocks:  # the same by whole blocks
        x[:128], x[128:256] = x[3].clone(), 0
        x[130, 300] = float("nan")
    got = call(x)
    bad = ~torch.isfinite(tops_of(x, 128 if blocks else 1))
    assert bad.any() and torch.equal(torch.isnan(got.scales), bad)
    q, s = got.values.float(), spread(got.scales, x.shape, 128 if blocks else 1)
    assert torch.isfinite(q).all() and (q[torch.isnan(s)] == 0).all()
    fine = ~torch.isnan(s)
    assert torch.all((q * s - x).abs()[fine] <= (x.abs() * (2.0 ** -4 + 2.0 ** -20) + s * 2.0 ** -9)[fine] + 448 * 2.0 ** -149)
    assert (got.scales[tops_of(x, 128 if blocks else 1) == 0] == 0).all()
    back = got.dequantize(F32)
    assert torch.equal(torch.isnan(back), torch.isnan(s))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width", [(1, 1), (3, 17), (5, 128), (130, 1000), (257, 3584), (33, 18944)])
def test_dequantize(dtype, rows, width):
    o, g = ops(), gen(rows + width)
    for x in (fp8_rows(g, rows, width), fp8_rows(g, rows, width, 48, True), fp8_blocks(g, rows, width, 16)):
        for activations in (False, True):
            got = o.dequantize_fp8(x, dtype, activations=activations)
            assert torch.equal(got, values_of(x, F32).to(dtype))
    every = torch.arange(256, device=DEV).to(torch.uint8).view(E4M3).reshape(2, 128)  # every e4m3, both NaN among them
    got = o.Fp8Rows(every, torch.ones(2, 1, device=DEV)).dequantize(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(every.float())) and torch.equal(got.nan_to_num(), every.to(dtype).nan_to_num())


def test_rows_after_the_last_are_left():
    """What lies behind the last row, and between rows, stays as it was: the memory is marked before."""
    o = ops()
    for width in (100, 129, 1000):
        x = normal(gen(width), 37, width)
        stride = -(-width // 16) * 16
        size = 37 * stride + 4 * 37 * blocks_of(width)
        marked = torch.full((size,), 0x5a, dtype=torch.uint8, device=DEV)
        where = marked.data_ptr()
        del marked
        got = o.quantize_rows_fp8(x)
        if got.values.data_ptr() != where:  # (the allocator gave other memory)
            continue
        whole = torch.as_strided(got.values.view(torch.uint8), (37, stride), (stride, 1))
        assert (whole[:, width:] == 0x5a).all()


# --------------------------------------------------------------------------- the norm

def normed(stream, weight, eps):
    s = stream.to(F64)
    return s / (s.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.to(F64)


@pytest.mark.parametrize("delta", [None, F32, BF16])
@pytest.mark.parametrize("width", [1, 3, 64, 128, 131, 896, 1001, 2051, 3584, 5120, 8192, 8200, 18944])
def test_add_rmsnorm(width, delta):
    o = ops()
    for rows, w_dtype, elsewhere in [(1, F32, False), (5, BF16, True), (9, F32, False), (700, BF16, False), (2400 if width <= 8192 else 301, F32, True)]:
        g = gen(width + rows)
        residual, weight = normal(g, rows, width) * 3, (1 + 0.1 * normal(g, width)).to(w_dtype)
        d = None if delta is None else normal(g, rows, width, dtype=delta)
        before = residual.clone()
        stream = residual if d is None else residual + d.float()
        out = torch.full_like(residual, 7.0) if elsewhere else None
        got = o.add_rmsnorm_fp8(residual, d, weight, 1e-6, residual_out=out)
        assert torch.equal(residual, before if elsewhere else stream) and (not elsewhere or torch.equal(out, stream))
        v = normed(stream, weight, 1e-6)
        check_near(got, v, v.abs() * 2.0 ** -17)


def test_norm_rows_stand_alone():
    """A row's bits do not depend on how many rows there are."""
    o = ops()
    for width in (512, 3584, 1537, 8192):
        residual, weight = normal(gen(width), 2600, width), normal(gen(1), width)
        whole = o.add_rmsnorm_fp8(residual, None, weight, 1e-6)
        for n in (1, 3, 299, 700):
            part = o.add_rmsnorm_fp8(residual[:n].contiguous(), None, weight, 1e-6)
            assert torch.equal(part.values.view(torch.uint8), whole.values[:n].view(torch.uint8)) and torch.equal(part.scales, whole.scales[:n])


def test_norm_special_rows():
    o = ops()
    x = normal(gen(5), 6, 300)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 299] = float("inf")
    got = o.add_rmsnorm_fp8(x, None, torch.ones(300, device=DEV), 1e-6)
    back = got.dequantize(F32)
    assert (back[1] == 0).all() and torch.isnan(back[2]).any() and torch.isnan(got.scales[3, 2])
    assert torch.isfinite(back[[0, 1, 4, 5]]).all()


# --------------------------------------------------------------------------- products

def plans(tokens, k, gated):
    """Forms that take such a call: both kernels, every tile, slices of K, blocks an SM.  (The sums of the widest tiles leave no room for
    two stages where K is cut.)"""
    out = []
    for tile in (16, 32, 48, 64, 96, 128, 160, 208, 256):
        if tile > (128 if gated else 256):
            continue
        for slices in (1, 2, 3, 8) if tile <= (96 if gated else 208) else (1,):
            for per in (1, 2) if tile <= (32 if gated else 64) else (1,):
                if slices <= blocks_of(k):
                    out.append((0, tile, slices, per))
    if not gated:
        out += [(1, tile, slices, 1) for tile in (128, 256) for slices in (2, 3, 8)]
    return out + [(1, tile, 1, 1) for tile in ((256,) if gated else (64, 128, 256))]


def products_of(x, w, bias):
    """The product in 64 bits, and the bound of its error before the last rounding."""
    xv, wv = values_of(x), values_of(w)
    y, a = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias is not None:
        y, a = y + bias.to(F64), a + bias.to(F64).abs()
    return y, a * (2.0 ** -16 + (blocks_of(x.shape[1]) + 12) * 2.0 ** -23)


def linear_close(got, ref):
    y, off = ref
    assert torch.all((got.to(F64) - y).abs() <= off + HALF[got.dtype] * (y.abs() + off) + 1e-37)


SIZES = [(1, 896, 1152), (1, 17, 5), (2, 1, 1), (15, 127, 127), (16, 128, 128), (17, 129, 129), (33, 300, 300), (64, 1000, 640), (65, 2100, 130),
         (128, 512, 384), (129, 3584, 200), (200, 1100, 1025), (257, 384, 257), (300, 640, 3000), (513, 1280, 640), (1000, 256, 1111), (2049, 512, 520)]


@pytest.mark.parametrize("tokens, k, features", SIZES)
def test_linear(tokens, k, features):
    o, g = ops(), gen(tokens + k)
    x, w = fp8_rows(g, tokens, k, 32 * (tokens % 2), turned=tokens % 3 > 0), fp8_blocks(g, features, k, 16 * (k % 2))
    for bias in (None, normal(g, features, dtype=BF16), normal(g, features)):
        ref = products_of(x, w, bias)
        for dtype in (F32, BF16):
            got = o.linear_fp8(x, w, bias, dtype)
            assert got.shape == (tokens, features) and got.dtype == dtype
            linear_close(got, ref)
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("tokens, k, features", [(1, 1500, 300), (24, 1500, 300), (150, 1100, 260), (515, 1500, 452), (700, 2100, 777)])
def test_linear_in_every_form(tokens, k, features):
    o, g = ops(), gen(tokens)
    x, w, bias = fp8_rows(g, tokens, k, turned=True), fp8_blocks(g, features, k), normal(g, features)
    ref = products_of(x, w, bias)
    for plan in plans(tokens, k, False):
        for dtype in (F32, BF16):
            linear_close(o.linear_fp8(x, w, bias, dtype, plan=plan), ref)
    o.check_errors(torch.device(DEV))


def test_linear_twice_gives_the_same_bits():
    o, g = ops(), gen(77)
    for tokens, k in ((9, 18944), (200, 8192), (1500, 2048)):
        x, w = fp8_rows(g, tokens, k), fp8_blocks(g, 640, k)
        first = o.linear_fp8(x, w, None, F32)
        for _ in range(5):
            assert torch.equal(o.linear_fp8(x, w, None, F32), first)


def test_products_in_slices_in_graphs_and_on_two_streams():
    """The parts of K stand in memory of the call's own: two calls at once, and a graph's replays beside calls outside of it, keep to theirs."""
    o, g = ops(), gen(31)
    plan = (1, 128, 4, 1)
    calls = [(fp8_rows(g, 200 + 56 * i, 2000, turned=True), fp8_blocks(g, 900, 2000), normal(g, 900)) for i in range(3)]
    expected = [o.linear_fp8(x, w, b, BF16, plan=plan) for x, w, b in calls]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [o.linear_fp8(x, w, b, BF16, plan=plan) for x, w, b in calls]
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for stream, (graph, outs) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
                again = [o.linear_fp8(x, w, b, BF16, plan=plan) for x, w, b in calls]
                for out, other in zip(outs, again):
                    out.copy_(torch.where(out == other, out, torch.nan))
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, expected))
    o.check_errors(torch.device(DEV))


def test_linear_blocks_meet_their_scales():
    """Powers of two as scales, one block at a time: sums of ones come out exactly, so each block of K and of features meets its own scale."""
    o = ops()
    for tokens, k, features in ((3, 500, 300), (300, 500, 300)):
        x = o.Fp8Rows(torch.zeros(tokens, 512, device=DEV).to(E4M3)[:, :k], torch.ones(tokens, 4, device=DEV))
        w = o.Fp8Blocks(torch.zeros(features, 512, device=DEV).to(E4M3)[:, :k], torch.ones(3, 4, device=DEV))
        x.values.fill_(1.0)
        w.values.fill_(1.0)
        x.scales.copy_(torch.exp2((torch.arange(tokens, device=DEV)[:, None] * 3 + torch.arange(4, device=DEV)) % 7 - 3.0))
        w.scales.copy_(torch.exp2((torch.arange(3, device=DEV)[:, None] * 2 + torch.arange(4, device=DEV) * 5) % 9 - 4.0))
        ref = values_of(x) @ values_of(w).t()
        for plan in plans(tokens, k, False):
            assert torch.equal(o.linear_fp8(x, w, None, F32, plan=plan).to(F64), ref), plan


def test_linear_scales_of_any_strides():
    o, g = ops(), gen(8)
    for tokens in (5, 400):
        x, w = fp8_rows(g, tokens, 1000), fp8_blocks(g, 300, 1000)
        store = torch.full((tokens, 3 * x.scales.shape[1]), float("nan"), device=DEV)
        store[:, ::3] = x.scales
        whole = torch.full((w.scales.shape[1], 2 * w.scales.shape[0]), float("nan"), device=DEV)
        whole[:, ::2] = w.scales.t()
        expected = o.linear_fp8(x, w, None, F32)
        assert torch.equal(o.linear_fp8(o.Fp8Rows(x.values, store[:, ::3]), o.Fp8Blocks(w.values, whole[:, ::2].t()), None, F32), expected)
        one = torch.full((1, 1), 0.5, device=DEV)
        x1, w1 = o.Fp8Rows(x.values, one.expand(tokens, 8)), o.Fp8Blocks(w.values, one.expand(3, 8))
        linear_close(o.linear_fp8(x1, w1, None, F32), products_of(x1, w1, None))


def test_linear_scales_that_are_not_numbers():
    o, g = ops(), gen(11)
    for tokens in (4, 300):
        x, w = fp8_rows(g, tokens, 256), fp8_blocks(g, 256, 256)
        x.scales[1, 1] = float("nan")
        x.scales[2] = 0
        w.scales[1, 0] = float("nan")
        got, ref = o.linear_fp8(x, w, None, F32), values_of(x) @ values_of(w).t()
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and (got[2, :128] == 0).all()


def test_linear_long_k_and_many_features():
    o, g = ops(), gen(12)
    for tokens in (3, 300):
        x, w = fp8_rows(g, tokens, 200000), fp8_blocks(g, 130, 200000)
        linear_close(o.linear_fp8(x, w, None, F32), products_of(x, w, None))
    features = 65536 * 128
    x, w = fp8_rows(g, 3, 16), fp8_blocks(g, features, 16)
    for n in (features - 127, features):
        part = o.Fp8Blocks(w.values[:n], w.scales)
        linear_close(o.linear_fp8(x, part, None, F32), products_of(x, part, None))
    o.check_errors(torch.device(DEV))


def units_of(x, w, bias, features):
    """The gated unit in 64 bits and the bound of its error before the last rounding."""
    y, off = products_of(x, w, bias)
    part = lambda t, i: t.reshape(t.shape[0], -1, 2, 128)[:, :, i].reshape(t.shape[0], -1)[:, :features]
    gate, up, dg, du = part(y, 0), part(y, 1), part(off, 0), part(off, 1)
    half = gate * torch.sigmoid(gate)
    return half * up, 1.1 * dg * (up.abs() + du) + half.abs() * du + (half * up).abs() * 2.0 ** -19


GATED = [(1, 896, 4864), (1, 33, 5), (8, 3584, 640), (16, 100, 128), (40, 1001, 1000), (130, 512, 130), (256, 768, 257), (300, 640, 1024), (777, 333, 333), (2049, 512, 1536)]


def gated_inputs(tokens, k, features, seed):
    g = gen(seed)
    x, w = fp8_rows(g, tokens, k, turned=True), fp8_blocks(g, 256 * blocks_of(features), k)
    x.scales.mul_(8.0 / k ** 0.5)
    return g, x, w


def unit_close(got, ref):
    y, off = ref
    if not isinstance(got, torch.Tensor):
        check_near(got, y, off)
    else:
        assert torch.all((got.to(F64) - y).abs() <= off + HALF[got.dtype] * (y.abs() + off) + 1e-30)


@pytest.mark.parametrize("tokens, k, features", GATED)
def test_gate_up_swiglu(tokens, k, features):
    o = ops()
    g, x, w = gated_inputs(tokens, k, features, tokens + k)
    for bias in (None, normal(g, w.shape[0], dtype=BF16), normal(g, w.shape[0])):
        ref = units_of(x, w, bias, features)
        for dtype in (F32, BF16, E4M3):
            got = o.gate_up_swiglu_fp8(x, w, bias, dtype, features=features)
            assert got.shape == (tokens, features) and (got.dtype == dtype if dtype != E4M3 else got.scales.shape == (tokens, blocks_of(features)))
            unit_close(got, ref)
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("tokens", [1, 24, 150, 515])
def test_gate_up_swiglu_in_every_form(tokens):
    o = ops()
    g, x, w = gated_inputs(tokens, 1500, 500, tokens)
    bias = normal(g, w.shape[0])
    ref = units_of(x, w, bias, 500)
    for plan in plans(tokens, 1500, True):
        for dtype in (F32, BF16, E4M3):
            unit_close(o.gate_up_swiglu_fp8(x, w, bias, dtype, features=500, plan=plan), ref)


def test_gated_unit_in_fp8_beside_the_float32_unit():
    """fp8 outputs are the float32 outputs of the same plan, rounded, but for the approximate exponential and division (2^-19 of a value
    at most); fewer features than the weight has, too."""
    o = ops()
    for tokens in (1, 9, 300):
        g, x, w = gated_inputs(tokens, 700, 640, tokens)
        for features in (640, 600, 129, 128, 3):
            for plan in ((0, 16, 1, 1), (0, 16, 3, 2), (0, 96, 2, 1), (0, 128, 1, 1), (1, 256, 1, 1)):
                unit = o.gate_up_swiglu_fp8(x, w, None, F32, features=features, plan=plan).to(F64)
                got = o.gate_up_swiglu_fp8(x, w, None, E4M3, features=features, plan=plan)
                assert got.shape == (tokens, features) and got.scales.shape == (tokens, blocks_of(features))
                check_near(got, unit, unit.abs() * 2.0 ** -19)


def test_gate_far_out():
    """Gates whose exponential overflows or vanishes."""
    o = ops()
    for tokens in (2, 300):
        values = torch.zeros(tokens, 16, device=DEV)
        values[:, 0] = 1
        weights = torch.zeros(256, 16, device=DEV)
        weights[:128, 0] = torch.arange(-64, 64, device=DEV)
        weights[128:, 0] = 100
        x = o.Fp8Rows(values.to(E4M3), torch.ones(tokens, 1, device=DEV))
        w = o.Fp8Blocks(weights.to(E4M3), torch.full((2, 1), 3.0, device=DEV))
        ref = units_of(x, w, None, 128)
        for dtype in (F32, BF16):
            got = o.gate_up_swiglu_fp8(x, w, None, dtype)
            assert torch.isfinite(got).all()
            unit_close(got, ref)


def test_stack_gate_up():
    o, g = ops(), gen(2)
    gate, up = normal(g, 200, 48), normal(g, 200, 48)
    stacked = o.stack_gate_up_fp8(gate, up)
    assert stacked.shape == (512, 48)
    x = o.quantize_rows_fp8(normal(g, 5, 48))
    got = o.gate_up_swiglu_fp8(x, o.quantize_blocks_fp8(stacked), None, F32, features=200)
    a, b = (values_of(x) @ values_of(o.quantize_blocks_fp8(t)).t() for t in (gate, up))
    off = values_of(x).abs() @ values_of(o.quantize_blocks_fp8(gate)).abs().t()
    ref = a * torch.sigmoid(a) * b
    assert got.shape == (5, 200) and torch.all((got.to(F64) - ref).abs() <= 2.0 ** -14 * (off * (a.abs() + b.abs() + off) + ref.abs()))


# --------------------------------------------------------------------------- as a program calls them

def test_weights_rounded_right_in_front_of_their_product():
    """A product may read its weights early: not before the kernel that rounds them is through, with one that lets go early between."""
    o = ops()
    for tokens in (3, 300):
        for seed in range(10):
            g = gen(seed)
            matrix, stream = normal(g, 512, 4096, dtype=BF16), normal(g, tokens, 4096)
            torch.cuda.synchronize()
            w = o.quantize_blocks_fp8(matrix)
            x = o.add_rmsnorm_fp8(stream, None, torch.ones(4096, device=DEV), 1e-6)
            got = o.linear_fp8(x, w, None, F32)
            linear_close(got, products_of(x, w, None))
            w.values.zero_()
            w.scales.fill_(float("nan"))
            del w  # (the next one may take its memory)


def layer_inputs(rows, hidden, inter, seed):
    g = gen(seed)
    o = ops()
    return dict(norm_w=1 + 0.1 * normal(g, hidden), w1=o.quantize_blocks_fp8(o.stack_gate_up_fp8(normal(g, inter, hidden), normal(g, inter, hidden)) / hidden ** 0.5),
                w2=o.quantize_blocks_fp8(normal(g, hidden, inter) / inter ** 0.5), residual=normal(g, rows, hidden), delta=normal(g, rows, hidden, dtype=BF16))


def layer(p, stream_out, inter):
    o = ops()
    x = o.add_rmsnorm_fp8(p["residual"], p["delta"], p["norm_w"], 1e-6, residual_out=stream_out)
    return o.linear_fp8(o.gate_up_swiglu_fp8(x, p["w1"], None, E4M3, features=inter), p["w2"])


@pytest.mark.parametrize("rows", [9, 300])
def test_layer_on_another_stream_and_in_a_graph(rows):
    """Norm, gated product, product: on a stream of its own, and captured and replayed with other inputs; two graphs side by side."""
    o = ops()
    inter = 600
    p = layer_inputs(rows, 512, inter, 21)
    stream_out = torch.empty_like(p["residual"])
    torch.cuda.synchronize()
    expected = layer(p, stream_out, inter)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = layer(p, torch.empty_like(stream_out), inter)
    side.synchronize()
    assert torch.equal(there, expected)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(p, stream_out, inter)
        graphs.append((graph, out))
    for seed in (1, 2):
        p["residual"].copy_(normal(gen(seed), rows, 512))
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        replayed = [out.clone() for _, out in graphs]
        now = layer(p, stream_out, inter)
        assert all(torch.equal(r, now) for r in replayed)
    o.check_errors(torch.device(DEV))


def test_layer_against_64_bits():
    """The run of a layer's operators against the same layer in 64 bits with the same weights: every rounding to e4m3 is off by at most
    2^-4 of a value (2^-10 of its block's scale more), which the products average; the bound takes them at their worst."""
    o, rows, hidden, inter = ops(), 33, 384, 500
    p = layer_inputs(rows, hidden, inter, 4)
    got = layer(p, torch.empty_like(p["residual"]), inter).to(F64)
    w1, w2 = values_of(p["w1"]).reshape(-1, 2, 128, hidden), values_of(p["w2"])
    gate_w, up_w = (w1[:, i].reshape(-1, hidden)[:inter] for i in (0, 1))
    v = normed(p["residual"] + p["delta"].float(), p["norm_w"], 1e-6)
    dv = v.abs() * 2.0 ** -4 + spread(tops_of(v, 1) / 448, v.shape, 1) * 2.0 ** -10 + v.abs() * 2.0 ** -16
    gate, up = v @ gate_w.t(), v @ up_w.t()
    dg, du = dv @ gate_w.abs().t(), dv @ up_w.abs().t()
    unit = gate * torch.sigmoid(gate) * up
    d = 1.1 * dg * (up.abs() + du) + (gate * torch.sigmoid(gate)).abs() * du
    d = d + (unit.abs() + d) * 2.0 ** -4 + spread(tops_of(unit.abs() + d, 1) / 448, unit.shape, 1) * 2.0 ** -10
    y, dy = unit @ w2.t(), (d + unit.abs() * 2.0 ** -14) @ w2.abs().t()
    assert torch.all((got - y).abs() <= dy + 2.0 ** -8 * (y.abs() + dy))


def test_two_blocks_share_an_sm_where_the_plan_says_so():
    from slipstream_b200.ops import fp8

    one, two = fp8._resident(0)
    sms = ops().sm_count(0)
    assert one[0] == sms and two[0] == 2 * sms and all(b > a for a, b in zip(one, two))


@pytest.mark.parametrize("plan", [[0, 16, 1, 1], (0, 16, 1), (0, 16, 1, 1, 1), (0, 16.0, 1, 1), (0, 2 ** 32 + 16, 1, 1), (0, 16, 2 ** 70, 1), (0, -16, 1, 1),
                                  (-1, 64, 1, 1), 16, "0111", (0, 24, 1, 1), (0, 16, 9, 1), (0, 16, 0, 1), (0, 16, 1, 3), (0, 272, 1, 1), (0, 80, 1, 2), (1, 64, 2, 1), (1, 128, 0, 1), (1, 256, 9, 1), (1, 32, 1, 1), (1, 192, 1, 1), (1, 320, 1, 1)])
def test_plans_that_are_none(plan):
    o = ops()
    rows, w = o.quantize_rows_fp8(torch.ones(4, 64, device=DEV)), o.quantize_blocks_fp8(torch.ones(256, 64, device=DEV))
    with pytest.raises(o.KernelError):
        o.linear_fp8(rows, w, plan=plan)
    with pytest.raises(o.KernelError):
        o.gate_up_swiglu_fp8(rows, w, plan=plan)


def test_launches_are_counted_where_there_are_any():
    o = ops()
    x, weight = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    rows, w = o.quantize_rows_fp8(x), o.quantize_blocks_fp8(torch.ones(256, 64, device=DEV))
    none = o.quantize_rows_fp8(x[:0])

    def counted(call):
        before = o.launch_count()
        try:
            call()
        except o.KernelError:
            pass
        return o.launch_count() - before

    for call in (lambda: o.quantize_rows_fp8(x), lambda: o.quantize_blocks_fp8(x), lambda: rows.dequantize(F32), lambda: o.add_rmsnorm_fp8(x, None, weight, 1e-6),
                 lambda: o.linear_fp8(rows, w), lambda: o.gate_up_swiglu_fp8(rows, w), lambda: o.gate_up_swiglu_fp8(rows, w, None, E4M3)):
        assert counted(call) == 1
    for call in (lambda: o.quantize_rows_fp8(x[:0]), lambda: o.quantize_blocks_fp8(x[:0]), lambda: none.dequantize(F32), lambda: o.add_rmsnorm_fp8(x[:0], None, weight, 1e-6),
                 lambda: o.linear_fp8(none, w), lambda: o.gate_up_swiglu_fp8(none, w), lambda: o.gate_up_swiglu_fp8(rows, w, None, E4M3, features=0)):
        assert counted(call) == 0
    for call in (lambda: o.quantize_rows_fp8(x.half()), lambda: rows.dequantize(torch.float16), lambda: o.add_rmsnorm_fp8(x, None, weight[:5], 1e-6),
                 lambda: o.linear_fp8(rows, w, weight), lambda: o.linear_fp8(rows, w, plan=(0, 24, 1, 1)), lambda: o.gate_up_swiglu_fp8(rows, rows)):
        assert counted(call) == 0


def test_refusals():
    o = ops()
    err = o.KernelError
    x = torch.zeros(4, 64, device=DEV)
    good, w = o.quantize_rows_fp8(x), o.quantize_blocks_fp8(torch.ones(256, 64, device=DEV))
    for call in (o.quantize_rows_fp8, o.quantize_blocks_fp8):
        for bad in (x.half(), x.cpu(), x.t(), x[:, :0], x[0], x.to(E4M3)):
            with pytest.raises(err):
                call(bad)
    for call in (lambda: o.dequantize_fp8(good, torch.float16), lambda: o.dequantize_fp8(x, F32), lambda: o.dequantize_fp8(good, E4M3)):
        with pytest.raises(err):
            call()
    for bad in (x.double(), x.cpu(), x[:, ::2]):
        with pytest.raises(err):
            o.add_rmsnorm_fp8(bad, None, torch.ones(bad.shape[1], device=DEV), 1e-6)
    for delta in (x[:2], x.half(), x.cpu()):
        with pytest.raises(err):
            o.add_rmsnorm_fp8(x, delta, torch.ones(64, device=DEV), 1e-6)
    for weight in (torch.ones(63, device=DEV), torch.ones(64, device=DEV, dtype=torch.float16)):
        with pytest.raises(err):
            o.add_rmsnorm_fp8(x, None, weight, 1e-6)
    with pytest.raises(err):
        o.add_rmsnorm_fp8(x, None, torch.ones(64, device=DEV), 1e-6, residual_out=x[:2])
    with pytest.raises(err):
        o.add_rmsnorm_fp8(torch.zeros(1, 786433, device=DEV), None, torch.ones(786433, device=DEV), 1e-6)
    assert o.linear_fp8(good, w).shape == (4, 256)
    wide = torch.zeros(4, 40, device=DEV).to(E4M3)
    scales = torch.ones(4, 1, device=DEV)
    for rows in (o.Fp8Rows(wide[:, :32], scales),             # a stride of 40
                 o.Fp8Rows(good.values, scales[:3]),           # scales missing
                 o.Fp8Rows(good.values, scales[:, 0]),         # of one dimension
                 o.Fp8Rows(good.values, torch.ones(4, 2, device=DEV)),
                 o.Fp8Rows(good.values, scales.double()),
                 o.Fp8Rows(good.values, scales.cpu()),
                 o.Fp8Rows(x, scales),                         # not e4m3
                 o.Fp8Rows(good.values.view(torch.uint8), scales),
                 o.Fp8Rows(good.values.t(), torch.ones(64, 1, device=DEV)),
                 o.Fp8Rows(torch.zeros(4, 128, device=DEV).to(E4M3)[:, 1:65], scales)):  # rows that start on byte 1
        with pytest.raises(err):
            o.linear_fp8(rows, w)
    short = o.quantize_blocks_fp8(torch.ones(256, 32, device=DEV))
    for call in (lambda: o.linear_fp8(x, w), lambda: o.linear_fp8(good, x), lambda: o.linear_fp8(good, good), lambda: o.linear_fp8(w, w), lambda: o.linear_fp8(good, short),
                 lambda: o.linear_fp8(good, o.Fp8Blocks(w.values, good.scales)), lambda: o.linear_fp8(good, w, torch.zeros(255, device=DEV)),
                 lambda: o.linear_fp8(good, w, torch.zeros(256, device=DEV).half()), lambda: o.linear_fp8(good, w, None, torch.float16), lambda: o.linear_fp8(good, w, None, E4M3),
                 lambda: o.gate_up_swiglu_fp8(good, o.quantize_blocks_fp8(torch.ones(128, 64, device=DEV))), lambda: o.gate_up_swiglu_fp8(good, w, features=129),
                 lambda: o.gate_up_swiglu_fp8(good, w, features=-1), lambda: o.gate_up_swiglu_fp8(good, w, None, torch.float8_e5m2), lambda: o.stack_gate_up_fp8(x, x[:2]),
                 lambda: o.gate_up_swiglu_fp8(good, w, plan=(1, 128, 1, 1)), lambda: o.gate_up_swiglu_fp8(good, w, plan=(1, 256, 2, 1)), lambda: o.gate_up_swiglu_fp8(good, w, plan=(0, 144, 1, 1))):
        with pytest.raises(err):
            call()
    none = o.quantize_rows_fp8(torch.empty(0, 64, device=DEV))
    assert o.linear_fp8(none, w).shape == (0, 256) and o.gate_up_swiglu_fp8(none, w, None, E4M3).shape == (0, 128)
    torch.cuda.synchronize()

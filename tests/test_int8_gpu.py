"""Rows of 8-bit integers: rounding to them and back, the norm that ends in them, products of them.

Tolerances, from the formulas.  A row's scale is a / 127 in one float32 division: half a unit in the last place, 2^-24.  A value
lands on the nearest step but for the rounding of v * (127 / a), two roundings of a number up to 127: at most 0.5 + 127 * 2^-23
steps off.  The norm adds the error of its factor: a float32 sum of squares in at most 110 additions a term (110 *
2^-24 of the sum, half of it in the root) and six single roundings, below 2^-17 of a value.  The sums of products are whole
numbers: what follows them is three float32 operations in a fixed order, so linear outputs are compared bit for bit.  The gated
unit's exponential and division are off by a few 2^-22 in the approximate form that bfloat16 outputs take, far below that type's
own half unit, 2^-9, and by a few 2^-24 in float32."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def ops():
    from slipstream_b200 import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def int8_rows(g, n, k, extra=0):
    """Random int8 rows (all 255 values), a stride of 16s with ``extra`` bytes more, rubbish between the rows."""
    stride = -(-k // 16) * 16 + extra
    store = torch.randint(-128, 128, (n, stride), generator=g, device=DEV, dtype=torch.int8)
    values = store[:, :k]
    values.clamp_(-127, 127)
    return ops().Int8Rows(values, torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4)


def sums_of(x, w):
    """Exact: whole numbers below 2^53."""
    return x.values.to(F64) @ w.values.to(F64).t()


def linear_of(x, w, bias):
    """Bit for bit what the kernels compute: the sum to float32, times the token's scale, times the feature's, plus the bias."""
    y = sums_of(x, w).to(F32) * x.scales[:, None] * w.scales
    return y if bias is None else y + bias.float()


def check_rows(rows, v, slack):
    """Every value on its nearest step (``slack`` of the value aside), scales right, the largest at 127."""
    top = v.abs().amax(dim=1)
    assert torch.all((rows.scales.to(F64) - top / 127).abs() <= top / 127 * (slack + 2.0 ** -23))
    q = rows.values.to(F64)
    assert q.abs().max() <= 127
    if (top > 0).any():
        assert torch.all(q.abs().amax(dim=1)[top > 0] == 127)
    off = (q * rows.scales.to(F64)[:, None] - v).abs()
    assert torch.all(off <= top[:, None] / 127 * (0.5 + 127 * 2.0 ** -22) + slack * v.abs())


WIDTHS = [1, 3, 16, 17, 64, 255, 896, 1001, 1537, 2051, 3584, 8193, 18944]


# --------------------------------------------------------------------------- rounding to int8 rows

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [*WIDTHS, 24001, 50000])
def test_quantize_rows(dtype, width):
    for rows, pad, shift in [(1, 0, 0), (5, 0, 0), (7, 8, 8), (6, 5, 1), (700 if width < 4000 else 301, 16, 0)]:
        store = normal(gen(width + rows), rows, width + pad, dtype=dtype)
        x = store[:, shift:shift + width]
        got = ops().quantize_rows_int8(x)
        assert got.values.shape == (rows, width) and got.scales.shape == (rows,)
        check_rows(got, x.to(F64), 0.0)
        # the definition in float32, operation for operation
        top = x.float().abs().amax(dim=1, keepdim=True)
        assert torch.equal(got.values, (x.float() * (torch.full_like(top, 127.0) / top)).round().to(torch.int8))
        assert torch.equal(got.scales, (top / torch.full_like(top, 127.0))[:, 0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width, pad", [(8, 0), (16, 8), (896, 0), (2048, 24), (3584, 0), (4100, 4), (5000, 3), (9736, 0), (12288, 0), (18944, 0), (24576, 0), (30000, 0)])
def test_quantize_many_rows(dtype, width, pad):
    """Rows enough for several a block, at widths on both sides of what the copies into shared memory take; a row of zeros, one of
    infinities and one of NaN among them change no other."""
    o = ops()
    x = normal(gen(width), 1301 if width > 9000 else 2600, width + pad, dtype=dtype)[:, :width]
    x[17], x[300], x[1184] = 0, float("inf"), float("nan")
    got = o.quantize_rows_int8(x)
    top = x.float().abs().amax(dim=1, keepdim=True)
    q = (x.float() * (torch.full_like(top, 127.0) / top)).round()
    fine = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    fine[[17, 300, 1184]] = False
    assert torch.equal(got.values[fine], q[fine].to(torch.int8))
    assert torch.equal(got.scales[fine], (top / torch.full_like(top, 127.0))[fine, 0])
    assert not got.values[~fine].any() and got.scales[17] == 0 and torch.isnan(got.scales[[300, 1184]]).all()
    assert torch.equal(o.dequantize_rows_int8(got, dtype)[fine], (got.values.float() * got.scales[:, None]).to(dtype)[fine])
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [33, 3584, 50000])
def test_quantize_rows_without_a_scale(dtype, width):
    x = normal(gen(1), 9, width, dtype=dtype)
    x[0] = 0
    x[1, width // 2] = float("inf")
    x[2, width - 1] = -float("inf")
    x[3, 0] = float("nan")
    x[4] = float("nan")
    x[5] *= 2.0 ** -110  # 127 / a would pass the largest float32 without care
    x[6] = 0
    x[6, 5] = -(2.0 ** -126)
    x[7] = torch.finfo(dtype).min
    got = ops().quantize_rows_int8(x)
    assert got.scales[0] == 0 and not got.values[0].any()
    assert torch.isnan(got.scales[1:5]).all() and not got.values[1:5].any()
    assert torch.isnan(got.dequantize(F32)[1:5]).all()
    fine = ops().Int8Rows(got.values[[5, 8]], got.scales[[5, 8]])
    check_rows(fine, x[[5, 8]].to(F64), 0.0)
    assert got.values[6, 5] == -127 and got.values[6].count_nonzero() == 1
    assert (got.values[7] == -127).all() and torch.isfinite(got.scales[7])


def test_widest_rows():
    """One row of as many elements as the kernels count, and one of one more.  Three elements are not zero, the first and the last
    among them."""
    o, widest = ops(), 2 ** 31 - 1 - 8192
    at = torch.tensor([0, 2 ** 30 + 1, widest - 1], device=DEV)
    values = torch.tensor([3.0, 1.0, -4.0], device=DEV)
    x = torch.zeros(1, widest, device=DEV, dtype=BF16)
    x[0, at] = values.to(BF16)
    rows = o.quantize_rows_int8(x)
    assert rows.scales.tolist() == [(torch.tensor(4.0) / 127).item()]
    assert rows.values[0, at].tolist() == [95, 32, -127] and rows.values.count_nonzero() == 3
    x.fill_(7.0)
    back = rows.dequantize(BF16)
    assert torch.equal(back[0, at], (rows.values[0, at].float() * rows.scales).to(BF16)) and back.count_nonzero() == 3
    del x, back, rows
    stream, weight = torch.zeros(1, widest, device=DEV), torch.ones(1, device=DEV, dtype=BF16).expand(widest).contiguous()
    stream[0, at] = values
    rows = o.add_rmsnorm_int8(stream, None, weight, 0.0)
    assert rows.values[0, at].tolist() == [95, 32, -127] and rows.values.count_nonzero() == 3
    assert abs(rows.scales.item() / (4 / (26 / widest) ** 0.5 / 127) - 1) < 2.0 ** -17
    del stream, weight, rows
    for wide in (torch.empty(1, widest + 1, device=DEV, dtype=BF16), torch.empty(1, 2 ** 31 - 8, device=DEV, dtype=BF16)):
        with pytest.raises(o.KernelError, match="elements at most"):
            o.quantize_rows_int8(wide)
    wide = torch.empty(1, widest + 1, device=DEV)
    with pytest.raises(o.KernelError, match="elements at most"):
        o.add_rmsnorm_int8(wide, None, wide[0], 1e-6)
    with pytest.raises(o.KernelError, match="elements at most"):
        o.dequantize_rows_int8(o.Int8Rows(wide.view(torch.int8)[:, :widest + 1], torch.ones(1, device=DEV)), BF16)
    torch.cuda.empty_cache()


def test_quantize_does_not_write_between_rows():
    o = ops()
    rows = o.int8_rows_like(6, 37, torch.device(DEV))
    assert rows.values.stride() == (48, 1) and rows.values.data_ptr() % 16 == 0
    assert o.quantize_rows_int8(torch.empty(0, 5, device=DEV)).shape == (0, 5)
    x = normal(gen(3), 6, 37, dtype=BF16)
    got = o.quantize_rows_int8(x)
    whole = torch.as_strided(got.values, (5, 48), (48, 1))
    before = whole[:, 37:].clone()
    again = o.quantize_rows_int8(x)
    assert torch.equal(got.values, again.values) and torch.equal(whole[:, 37:], before)


def marked(rows, width):
    """The address of memory as large as int8 rows are together with their scales, every byte of it 90, which the next ones get."""
    t = torch.full((rows * ((width + 15) // 16 * 16 + 4),), 90, dtype=torch.int8, device=DEV)
    return t.data_ptr()


def check_padding(rows, address):
    n, width = rows.values.shape
    stride = (width + 15) // 16 * 16
    assert rows.values.data_ptr() == address and rows.values.stride() == (stride, 1)
    assert (torch.as_strided(rows.values, (n, stride), (stride, 1))[:, width:] == 90).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width", [*((7, 33 + i) for i in range(16)), (700, 897), (700, 1001), (5, 24001), (5, 50005), (2400, 4100), (2400, 8200), (2400, 8204), (2400, 9736)])
def test_what_lies_between_rows_is_not_written(dtype, rows, width):
    """Every kernel that forms rows, at every number of bytes between two: what stood there stays, and behind the last row the scales."""
    o, eps = ops(), 1e-6
    store = normal(gen(width), rows, width + 3, dtype=dtype)
    weight, top = torch.ones(width, device=DEV), lambda t: t.float().abs().amax(dim=1)
    for x in (store[:, 3:], store[:, 3:].contiguous()):
        address = marked(rows, width)
        got = o.quantize_rows_int8(x)
        check_padding(got, address)
        assert torch.equal(got.scales, top(x) / torch.full_like(top(x), 127.0))
        del got
    stream = normal(gen(width), rows, width)
    expected = o.add_rmsnorm_int8(stream, x, weight, eps, residual_out=torch.empty_like(stream))
    want, scales = expected.values.clone(), expected.scales.clone()
    del expected
    address = marked(rows, width)
    got = o.add_rmsnorm_int8(stream, x, weight, eps)
    check_padding(got, address)
    assert torch.equal(got.values, want) and torch.equal(got.scales, scales)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", WIDTHS)
def test_dequantize_rows(dtype, width):
    for n in (1, 13):
        rows = int8_rows(gen(width), n, width, 32)
        got = ops().dequantize_rows_int8(rows, dtype)
        assert torch.equal(got, (rows.values.float() * rows.scales[:, None]).to(dtype))


# --------------------------------------------------------------------------- the norm

@pytest.mark.parametrize("dtype, w_dtype", [(BF16, BF16), (BF16, F32), (F32, F32), (None, BF16)])
@pytest.mark.parametrize("width", [1, 17, 64, 896, 1537, 3584, 5120, 8190, 20000, 40004])
def test_add_rmsnorm(dtype, w_dtype, width):
    o, eps = ops(), 1e-5
    for n in (1, 3, 310):
        g = gen(width + n)
        residual = normal(g, n, width) * 3
        delta = None if dtype is None else normal(g, n, width, dtype=dtype)
        weight = (1 + 0.1 * normal(g, width)).to(w_dtype)
        stream = residual if delta is None else residual + delta.float()
        x = stream.to(F64)
        v = x / (x.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.to(F64)
        out, before = torch.full_like(residual, 7.0), residual.clone()
        got = o.add_rmsnorm_int8(residual, delta, weight, eps, residual_out=out)
        assert torch.equal(out, stream) and torch.equal(residual, before)
        check_rows(got, v, 2.0 ** -17)
        again = o.add_rmsnorm_int8(residual, delta, weight, eps)  # in place
        assert torch.equal(residual, stream)
        assert torch.equal(again.values, got.values) and torch.equal(again.scales, got.scales)


@pytest.mark.parametrize("dtype, w_dtype", [(BF16, BF16), (BF16, F32), (F32, F32), (None, BF16)])
@pytest.mark.parametrize("width", [8, 64, 896, 1540, 3584, 4100, 5120, 8192, 12288, 16384])
def test_add_rmsnorm_many_rows(dtype, w_dtype, width):
    o, eps, n = ops(), 1e-6, 1301
    g = gen(width)
    residual = normal(g, n, width) * 3
    delta = None if dtype is None else normal(g, n, width, dtype=dtype)
    weight = (1 + 0.1 * normal(g, width)).to(w_dtype)
    residual[17] = 0
    if delta is not None:
        delta[17] = 0
    residual[300, 1], residual[1200, width - 1] = float("inf"), float("nan")
    stream = residual if delta is None else residual + delta.float()
    fine = torch.ones(n, dtype=torch.bool, device=DEV)
    fine[[300, 1200]] = False
    x = stream.to(F64)
    v = x / (x.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.to(F64)
    out = torch.full_like(residual, 7.0)
    got = o.add_rmsnorm_int8(residual, delta, weight, eps, residual_out=out)
    assert torch.equal(out[fine], stream[fine])
    check_rows(o.Int8Rows(got.values[fine], got.scales[fine]), v[fine], 2.0 ** -17)
    assert torch.isnan(got.scales[~fine]).all() and not got.values[~fine].any()
    again = o.add_rmsnorm_int8(residual, delta, weight, eps)  # in place
    assert torch.equal(residual[fine], stream[fine])
    assert torch.equal(again.values, got.values) and torch.equal(again.scales[fine], got.scales[fine])
    for rows in (1, 40, 400):  # a row does not depend on how many there are
        few = o.add_rmsnorm_int8(stream[fine][:rows].contiguous(), None, weight, eps)
        assert torch.equal(few.values, got.values[fine][:rows]) and torch.equal(few.scales, got.scales[fine][:rows])
    o.check_errors(torch.device(DEV))


def test_add_rmsnorm_rows_without_a_scale():
    g = gen(5)
    residual, weight = normal(g, 6, 512), normal(g, 512)
    residual[0] = 0
    residual[1, 3] = float("inf")
    residual[2, 9] = float("nan")
    residual[3] *= 1e-25  # the squares vanish beside eps, the values do not
    got = ops().add_rmsnorm_int8(residual, None, weight, 1e-6)
    assert got.scales[0] == 0 and not got.values[0].any()
    assert torch.isnan(got.dequantize(F32)[1:3]).all()
    x = residual[3:].to(F64)
    v = x / (x.square().mean(dim=1, keepdim=True) + 1e-6).sqrt() * weight.to(F64)
    check_rows(ops().Int8Rows(got.values[3:], got.scales[3:]), v, 2.0 ** -17)


# --------------------------------------------------------------------------- products

SHAPES = [(1, 1, 1), (1, 16, 8), (1, 33, 5), (1, 896, 1152), (2, 127, 129), (7, 4864, 896), (8, 3584, 512), (16, 2001, 130), (17, 640, 256), (31, 129, 1000),
          (33, 1536, 2048), (64, 1001, 77), (65, 256, 128), (100, 3581, 1153), (129, 777, 515), (203, 1024, 641), (256, 384, 300), (257, 300, 256),
          (300, 1111, 1000), (300, 128, 256), (70, 128, 64), (511, 896, 1152), (777, 2000, 333), (1025, 640, 2050), (2047, 512, 4608)]


@pytest.mark.parametrize("tokens, k, features", SHAPES)
def test_linear(tokens, k, features):
    o, g = ops(), gen(tokens * 7 + k)
    x, w = int8_rows(g, tokens, k, 16), int8_rows(g, features, k)
    for bias in (None, normal(g, features, dtype=BF16), normal(g, features)):
        ref = linear_of(x, w, bias)
        assert torch.equal(o.linear_int8(x, w, bias, F32), ref)
        assert torch.equal(o.linear_int8(x, w, bias), ref.to(BF16))
    o.check_errors(torch.device(DEV))


def plans(tokens, k, gated):
    few = max(16, min(256, (tokens + 15) // 16 * 16))
    out = [(0, tile, slices, per_sm, steps) for tile in {16, 32, 48, few, 128, 208} for slices in (1, 2, 5, 8) for per_sm, steps in ((1, 1), (2, 1), (4, 1), (1, 2), (2, 2))
           if tile <= 2 * few and steps * tile <= 256]
    return out + [(1, tile, 1, 1, steps) for tile in ((128, 256) if gated else (32, 96, 128, 224, 256)) for steps in (1, 2)]


@pytest.mark.parametrize("tokens, k, features", [(1, 200, 130), (19, 1500, 515), (150, 3584, 700), (515, 900, 1024), (33, 1152, 300)])
def test_linear_in_every_form(tokens, k, features):
    """The same bits from both kernels, whatever their tiles and however K is cut (more slices than there is K, too)."""
    o, g = ops(), gen(tokens)
    x, w, bias = int8_rows(g, tokens, k), int8_rows(g, features, k), normal(g, features)
    ref = linear_of(x, w, bias)
    for plan in plans(tokens, k, False):
        assert torch.equal(o.linear_int8(x, w, bias, F32, plan=plan), ref), plan
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("tokens", [3, 33, 257])
@pytest.mark.parametrize("features", [1, 2, 31, 33, 63, 94, 257, 258, 260, 264, 287, 513])
def test_many_tokens_with_output_rows_that_start_anywhere(tokens, features):
    """Rows of the output that start on 2, 4, 8 or 16 bytes, and tiles that end within their first or last run of 64 bytes."""
    o, g = ops(), gen(tokens * 1000 + features)
    x, w, bias = int8_rows(g, tokens, 200), int8_rows(g, features, 200), normal(g, features, dtype=BF16)
    gated = int8_rows(g, (features + 63) // 64 * 128, 200)
    x.scales.mul_(20.0 / 200 ** 0.5)
    for dtype in (F32, BF16):
        for tile in (32, 96, 256):
            assert torch.equal(o.linear_int8(x, w, bias, dtype, plan=(1, tile, 1, 1, 2)), linear_of(x, w, bias).to(dtype)), (dtype, tile)
        for tile in (128, 256):
            got = o.gate_up_swiglu_int8(x, gated, None, dtype, features=features, plan=(1, tile, 1, 1, 1))
            assert torch.equal(got, o.gate_up_swiglu_int8(x, gated, None, dtype, features=features, plan=(0, 32, 1, 1, 1))), (dtype, tile)
            assert gated_close(got, gated_of(x, gated, None, features))
    o.check_errors(torch.device(DEV))


def test_linear_largest_sums():
    """The longest K, every product 128 * 128: the sum stays below 2^31."""
    o = ops()
    k = 131071
    for tokens in (3, 300):
        x = o.int8_rows_like(tokens, k, torch.device(DEV))
        w = o.int8_rows_like(130, k, torch.device(DEV))
        for r in (x, w):
            r.values.fill_(-128)
            r.scales.fill_(1.0)
        w.values[1::2] = 127
        got = o.linear_int8(x, w, None, F32)
        assert torch.equal(got, linear_of(x, w, None)) and got.max() == float(128 * 128 * k) and got.min() == -float(127 * 128 * k)


def test_more_features_than_a_grid_has_rows_for_their_tiles():
    o, g = ops(), gen(12)
    features = 65536 * 128
    x, w = int8_rows(g, 3, 16), int8_rows(g, features, 16)
    for n in (features - 127, features):
        part = o.Int8Rows(w.values[:n], w.scales[:n])
        assert torch.equal(o.linear_int8(x, part, None, F32), linear_of(x, part, None))
    x.scales.mul_(5.0)
    assert gated_close(o.gate_up_swiglu_int8(x, w, None, F32), gated_of(x, w, None, features // 2))
    o.check_errors(torch.device(DEV))


def test_linear_scales_that_are_not_numbers():
    o, g = ops(), gen(11)
    for tokens in (4, 300):
        x, w = int8_rows(g, tokens, 256), int8_rows(g, 256, 256)
        x.scales[1] = float("nan")
        x.scales[2] = 0
        w.scales[5] = float("nan")
        got = o.linear_int8(x, w, None, F32)
        ref = linear_of(x, w, None)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))


def gated_of(x, w, bias, features):
    y = linear_of(x, w, bias).to(F64)
    runs = y.reshape(y.shape[0], -1, 2, 64)
    gate, up = (runs[:, :, i].reshape(y.shape[0], -1)[:, :features] for i in (0, 1))
    return gate * torch.sigmoid(gate) * up


def gated_close(got, ref):
    slack = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -20
    return torch.all((got.to(F64) - ref).abs() <= slack * ref.abs() + 1e-30)


@pytest.mark.parametrize("tokens, k, features", [(1, 896, 4864), (1, 33, 5), (8, 3584, 640), (16, 100, 64), (40, 1001, 1000), (130, 512, 130), (256, 768, 257),
                                                 (300, 640, 1024), (777, 333, 333), (2049, 512, 1536)])
def test_gate_up_swiglu(tokens, k, features):
    o, g = ops(), gen(tokens + k)
    x = int8_rows(g, tokens, k)
    w = int8_rows(g, -(-features // 64) * 128, k)
    x.scales.mul_(20.0 / k ** 0.5)
    for bias in (None, normal(g, w.shape[0], dtype=BF16), normal(g, w.shape[0])):
        ref = gated_of(x, w, bias, features)
        for dtype in (F32, BF16):
            got = o.gate_up_swiglu_int8(x, w, bias, dtype, features=features)
            assert got.shape == (tokens, features) and got.dtype == dtype and gated_close(got, ref)
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("tokens", [1, 24, 150, 515])
def test_gate_up_swiglu_in_every_form(tokens):
    o, g = ops(), gen(tokens)
    x, w, bias = int8_rows(g, tokens, 1500), int8_rows(g, 640, 1500), normal(g, 640)
    x.scales.mul_(0.5)
    first = {}
    for plan in plans(tokens, 1500, True):
        for dtype in (F32, BF16):
            got = o.gate_up_swiglu_int8(x, w, bias, dtype, plan=plan)
            assert torch.equal(got, first.setdefault(dtype, got)), plan
    assert gated_close(first[F32], gated_of(x, w, bias, 320)) and gated_close(first[BF16], gated_of(x, w, bias, 320))


def test_gate_far_out():
    """Gates whose exponential overflows or vanishes."""
    o = ops()
    for tokens in (2, 300):
        x, w = o.int8_rows_like(tokens, 16, torch.device(DEV)), o.int8_rows_like(128, 16, torch.device(DEV))
        x.values.zero_()
        w.values.zero_()
        x.values[:, 0] = 1
        w.values[:64, 0] = torch.arange(-32, 32, device=DEV, dtype=torch.int8) * 3
        w.values[64:, 0] = 100
        x.scales.fill_(1.0)
        w.scales.fill_(1.0)
        for dtype in (F32, BF16):
            got = o.gate_up_swiglu_int8(x, w, None, dtype)
            ref = gated_of(x, w, None, 64)
            # (far below, the unit's value vanishes; there an absolute 1e-30 is as good as the value)
            assert torch.isfinite(got).all() and gated_close(got, ref)


def test_stack_gate_up():
    o, g = ops(), gen(2)
    gate, up = normal(g, 100, 48), normal(g, 100, 48)
    stacked = o.stack_gate_up(gate, up)
    assert stacked.shape == (256, 48)
    assert torch.equal(stacked[:64], gate[:64]) and torch.equal(stacked[64:128], up[:64])
    assert torch.equal(stacked[128:164], gate[64:]) and torch.equal(stacked[192:228], up[64:])
    assert not stacked[164:192].any() and not stacked[228:].any()
    x = normal(g, 5, 48)
    got = o.gate_up_swiglu_int8(o.quantize_rows_int8(x), o.quantize_rows_int8(stacked), None, F32, features=100)
    xd, gd, ud = (o.quantize_rows_int8(t).dequantize(F32).to(F64) for t in (x, gate, up))
    a, b = xd @ gd.t(), xd @ ud.t()
    assert got.shape == (5, 100) and torch.all((got.to(F64) - a * torch.sigmoid(a) * b).abs() <= 2.0 ** -18 * (a * b).abs() + 1e-5)


# --------------------------------------------------------------------------- as a program calls them

def test_weights_rounded_right_in_front_of_their_product():
    """A product may read its weights early: not before the kernel that rounds them is through."""
    o, g = ops(), gen(9)
    x = int8_rows(g, 3, 4096)
    for seed in range(20):
        matrix = normal(gen(seed), 512, 4096, dtype=BF16)
        w = o.quantize_rows_int8(matrix)
        got = o.linear_int8(x, w, None, F32)
        assert torch.equal(got, linear_of(x, w, None))


@pytest.mark.parametrize("tokens", [3, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_turned_back_right_in_front_of_their_product(dtype, tokens):
    """The same for the product of the values: against the same product a second time, when everything in front of it is through.
    The weights' memory holds NaN before."""
    o, g = ops(), gen(10)
    x = normal(g, tokens, 4096, dtype=dtype)
    for seed in range(20):
        rows = int8_rows(gen(seed), 6144, 4096)
        torch.cuda.synchronize()
        weight = rows.dequantize(dtype)
        got = o.linear(x, weight)
        torch.cuda.synchronize()
        assert torch.equal(weight, (rows.values.float() * rows.scales[:, None]).to(dtype))
        assert torch.equal(got, o.linear(x, weight)), seed
        weight.fill_(float("nan"))
        del weight  # (the next one takes its memory)


@pytest.mark.parametrize("tokens", [3, 300])
@pytest.mark.parametrize("back", [False, True])
def test_weights_written_two_kernels_in_front_of_their_product(back, tokens):
    """Between the weights and the product stands a kernel that lets the one behind it go at once, as in a program: the norm whose
    rows the product takes, or the rounding of its activations.  Weights of both kernels that round: a block per row, and the ring."""
    o = ops()
    for seed in range(10):
        g, k = gen(seed), 8192 if seed % 2 else 4096
        matrix, stream, norm_w = normal(g, 2600 if seed % 2 else 512, k, dtype=BF16), normal(g, tokens, k), torch.ones(k, device=DEV)
        torch.cuda.synchronize()
        if back:
            rows = o.quantize_rows_int8(matrix)
            weight = rows.dequantize(BF16)
            x = o.quantize_rows_int8(stream, activations=True).dequantize(BF16, activations=True)
            got = o.linear(x, weight)
            torch.cuda.synchronize()
            assert torch.equal(weight, (rows.values.float() * rows.scales[:, None]).to(BF16))
            assert torch.equal(got, o.linear(x, weight))
        else:
            weight = o.quantize_rows_int8(matrix)
            x = o.add_rmsnorm_int8(stream, None, norm_w, 1e-6)
            got = o.linear_int8(x, weight, None, F32)
            assert torch.equal(got, linear_of(x, weight, None))
            weight.values.zero_()
            weight.scales.fill_(float("nan"))
        del weight  # (the next one may take its memory)


def test_layer_on_another_stream_and_in_a_graph():
    """Norm, product, rounding, gated product, product: on a stream of its own, and captured and replayed with other inputs."""
    o, g = ops(), gen(21)
    hidden, inter = 512, 640
    norm_w = 1 + 0.1 * normal(g, hidden)
    w1, w2 = int8_rows(g, 2 * inter, hidden), int8_rows(g, hidden, inter)
    residual, delta = normal(g, 9, hidden), normal(g, 9, hidden, dtype=BF16)

    def layer():
        x = o.add_rmsnorm_int8(residual, delta, norm_w, 1e-6, residual_out=stream_out)
        hidden_rows = o.quantize_rows_int8(o.gate_up_swiglu_int8(x, w1), activations=True)
        return o.linear_int8(hidden_rows, w2)

    stream_out = torch.empty_like(residual)
    torch.cuda.synchronize()
    expected = layer()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = layer()
    side.synchronize()
    assert torch.equal(there, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for seed in (1, 2):
        residual.copy_(normal(gen(seed), 9, hidden))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, layer())
    o.check_errors(torch.device(DEV))


def test_two_blocks_share_an_sm_where_the_plan_says_so():
    from slipstream_b200.ops import int8

    one, two = int8._resident(0)
    sms = ops().sm_count(0)
    assert one[0] == sms and two[0] == 2 * sms and all(b > a for a, b in zip(one, two))
    assert int8._plan_on(8, 37888, 3584, 1, 0)[:4] == (0, 16, 1, 2)


@pytest.mark.parametrize("plan", [[0, 16, 1, 1, 1], (0, 16, 1, 1), (0, 16, 1, 1, 1, 1), (0, 16.0, 1, 1, 1), (0, 2 ** 32 + 16, 1, 1, 1), (0, 16, 2 ** 70, 1, 1),
                                  (0, -16, 1, 1, 1), (-1, 32, 1, 1, 1), 16, "01111"])
def test_plans_that_are_none(plan):
    o = ops()
    rows, w = o.quantize_rows_int8(torch.ones(4, 64, device=DEV)), o.quantize_rows_int8(torch.ones(128, 64, device=DEV))
    with pytest.raises(o.KernelError):
        o.linear_int8(rows, w, plan=plan)
    with pytest.raises(o.KernelError):
        o.gate_up_swiglu_int8(rows, w, plan=plan)


def test_launches_are_counted_where_there_are_any():
    o = ops()
    x, weight = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    rows, w = o.quantize_rows_int8(x), o.quantize_rows_int8(torch.ones(128, 64, device=DEV))
    none = o.quantize_rows_int8(x[:0])

    def counted(call):
        before = o.launch_count()
        try:
            call()
        except o.KernelError:
            pass
        return o.launch_count() - before

    for call in (lambda: o.quantize_rows_int8(x), lambda: rows.dequantize(F32), lambda: o.add_rmsnorm_int8(x, None, weight, 1e-6),
                 lambda: o.linear_int8(rows, w), lambda: o.gate_up_swiglu_int8(rows, w)):
        assert counted(call) == 1
    for call in (lambda: o.quantize_rows_int8(x[:0]), lambda: none.dequantize(F32), lambda: o.add_rmsnorm_int8(x[:0], None, weight, 1e-6),
                 lambda: o.linear_int8(none, w), lambda: o.gate_up_swiglu_int8(none, w), lambda: o.gate_up_swiglu_int8(rows, w, features=0)):
        assert counted(call) == 0
    for call in (lambda: o.quantize_rows_int8(x.half()), lambda: rows.dequantize(torch.float16), lambda: o.add_rmsnorm_int8(x, None, weight[:5], 1e-6),
                 lambda: o.linear_int8(rows, w, weight), lambda: o.linear_int8(rows, w, plan=(0, 24, 1, 1, 1)), lambda: o.gate_up_swiglu_int8(rows, rows)):
        assert counted(call) == 0


def test_refusals():
    o = ops()
    err = o.KernelError
    x = torch.zeros(4, 64, device=DEV)
    good, w = o.quantize_rows_int8(x), o.quantize_rows_int8(torch.ones(128, 64, device=DEV))
    with pytest.raises(err):
        o.quantize_rows_int8(x.half())
    with pytest.raises(err):
        o.quantize_rows_int8(x.cpu())
    with pytest.raises(err):
        o.quantize_rows_int8(x.t())
    with pytest.raises(err):
        o.quantize_rows_int8(x[:, :0])
    with pytest.raises(err):
        o.quantize_rows_int8(x[0])
    with pytest.raises(err):
        o.dequantize_rows_int8(good, torch.float16)
    with pytest.raises(err):
        o.dequantize_rows_int8(x, F32)
    for bad in (x.double(), x.cpu(), x[:, ::2]):
        with pytest.raises(err):
            o.add_rmsnorm_int8(bad, None, torch.ones(bad.shape[1], device=DEV), 1e-6)
    for delta in (x[:2], x.half(), x.cpu()):
        with pytest.raises(err):
            o.add_rmsnorm_int8(x, delta, torch.ones(64, device=DEV), 1e-6)
    for weight in (torch.ones(63, device=DEV), torch.ones(64, device=DEV, dtype=torch.float16)):
        with pytest.raises(err):
            o.add_rmsnorm_int8(x, None, weight, 1e-6)
    with pytest.raises(err):
        o.add_rmsnorm_int8(x, None, torch.ones(64, device=DEV), 1e-6, residual_out=x[:2])
    assert o.linear_int8(good, w).shape == (4, 128)
    wide = torch.zeros(4, 40, device=DEV, dtype=torch.int8)
    scales = torch.ones(4, device=DEV)
    for rows in (o.Int8Rows(wide[:, :32], scales),            # a stride of 40
                 o.Int8Rows(good.values, scales[:3]),          # scales missing
                 o.Int8Rows(good.values, scales.double()),
                 o.Int8Rows(x, scales),                        # not int8
                 o.Int8Rows(good.values.t(), torch.ones(64, device=DEV)),
                 o.Int8Rows(torch.zeros(4, 128, device=DEV, dtype=torch.int8)[:, 1:65], scales)):  # rows that start on byte 1
        with pytest.raises(err):
            o.linear_int8(rows, w)
    for call in (lambda: o.linear_int8(x, w), lambda: o.linear_int8(good, x), lambda: o.linear_int8(good, o.quantize_rows_int8(x[:, :32].contiguous())),
                 lambda: o.linear_int8(good, w, torch.zeros(127, device=DEV)), lambda: o.linear_int8(good, w, torch.zeros(128, device=DEV).half()),
                 lambda: o.linear_int8(good, w, None, torch.float16), lambda: o.gate_up_swiglu_int8(good, good),
                 lambda: o.gate_up_swiglu_int8(good, w, features=65), lambda: o.stack_gate_up(x, x[:2]),
                 lambda: o.linear_int8(good, w, plan=(0, 24, 1, 1, 1)), lambda: o.linear_int8(good, w, plan=(0, 16, 9, 1, 1)), lambda: o.linear_int8(good, w, plan=(0, 16, 1, 1, 3)),
                 lambda: o.linear_int8(good, w, plan=(1, 48, 1, 1, 1)), lambda: o.gate_up_swiglu_int8(good, w, plan=(1, 96, 1, 1, 1))):
        with pytest.raises(err):
            call()
    assert o.linear_int8(o.quantize_rows_int8(torch.empty(0, 64, device=DEV)), w).shape == (0, 128)
    torch.cuda.synchronize()

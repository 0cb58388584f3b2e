"""What the kernels of the 8-bit layers do when a wait gives up: they say so in the error word, write nothing, wait for what is in
flight to them and end, and the device goes on.  Shown by a build whose waits give up without a look (WAIT_POLLS=0), called through its
entry points; the copies of that build are real ones, and its blocks wait for them before they end, with the limit of the ordinary build."""

import ctypes
from ctypes import c_double, c_int64, c_void_p

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
WAIT_LIMIT = 8  # SS_ERR_WAIT_LIMIT


class RowsCall(ctypes.Structure):  # csrc/int8_calls.h, Int8RowsCall
    _fields_ = [("x", c_void_p), ("stride", c_int64), ("q", c_void_p), ("q_stride", c_int64), ("scales", c_void_p), ("rows", c_int64),
                ("width", c_int64), ("dtype", c_int64), ("early", c_int64), ("y", c_void_p), ("delta", c_void_p), ("weight", c_void_p),
                ("w_f32", c_int64), ("eps", c_double), ("err", c_void_p), ("stream", c_void_p)]


class ProductCall(ctypes.Structure):  # Int8Call
    _fields_ = [("x", c_void_p), ("ldx", c_int64), ("x_scale", c_void_p), ("w", c_void_p), ("ldw", c_int64), ("w_scale", c_void_p),
                ("bias", c_void_p), ("bias_f32", c_int64), ("out", c_void_p)]
    _fields_ += [(name, c_int64) for name in ("ldc", "out_f32", "tokens", "features", "K", "gated", "out_features", "many", "bn", "slices", "per_sm", "steps")]
    _fields_ += [("err", c_void_p), ("stream", c_void_p)]


def without_waits(name, source):
    from slipstream_b200.ops.library import compile_library

    return ctypes.CDLL(str(compile_library(name, [source], {"WAIT_POLLS": 0})))


@pytest.fixture(scope="module")
def rows_library():
    return without_waits("slipstream_int8_rows", "ops_int8.cu")


@pytest.fixture(scope="module")
def products_library():
    return without_waits("slipstream_int8_products", "gemm_int8.cu")


def ran(entry, call):
    """The entry point's status, and the error word behind it."""
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    call.err, call.stream = err.data_ptr(), torch.cuda.current_stream().cuda_stream
    assert entry(ctypes.byref(call)) == 0
    torch.cuda.synchronize()
    return int(err.item())


def int8_results(rows, width):
    return torch.full((rows, (width + 15) & -16), 55, dtype=torch.int8, device=DEV), torch.full((rows,), 7.0, device=DEV)


@pytest.mark.parametrize("early", [0, 1])
@pytest.mark.parametrize("dtype, width", [(F32, 4096), (BF16, 8192), (F32, 12288), (BF16, 18944)])
def test_rounding_of_many_rows(rows_library, dtype, width, early):
    from slipstream_b200 import ops

    rows = 2400
    x = torch.randn(rows, width, device=DEV).to(dtype)
    q, scales = int8_results(rows, width)
    call = RowsCall(x=x.data_ptr(), stride=width, q=q.data_ptr(), q_stride=q.stride(0), scales=scales.data_ptr(), rows=rows, width=width,
                    dtype=int(dtype == BF16), early=early)
    assert ran(rows_library.ss_quantize_rows_int8, call) == WAIT_LIMIT
    assert (q == 55).all() and (scales == 7).all()
    top = x.float().abs().amax(dim=1, keepdim=True)
    assert torch.equal(ops.quantize_rows_int8(x).values, (x.float() * (torch.full_like(top, 127.0) / top)).round().to(torch.int8))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("delta, width", [(None, 4096), (BF16, 3584), (F32, 5120), (BF16, 8192)])
def test_norm_of_many_rows(rows_library, delta, width, in_place):
    from slipstream_b200 import ops

    rows = 2400
    residual, weight = torch.randn(rows, width, device=DEV), torch.ones(width, device=DEV)
    d = None if delta is None else torch.randn(rows, width, device=DEV).to(delta)
    out = residual if in_place else torch.full_like(residual, 7.0)
    before = out.clone()
    q, scales = int8_results(rows, width)
    call = RowsCall(x=residual.data_ptr(), stride=width, q=q.data_ptr(), q_stride=q.stride(0), scales=scales.data_ptr(), rows=rows, width=width,
                    dtype=int(delta != F32), y=out.data_ptr(), delta=None if d is None else d.data_ptr(), weight=weight.data_ptr(), w_f32=1, eps=1e-6)
    assert ran(rows_library.ss_add_rmsnorm_int8, call) == WAIT_LIMIT
    assert torch.equal(out, before) and (q == 55).all() and (scales == 7).all()
    stream = residual.clone()
    ops.add_rmsnorm_int8(stream, d, weight, 1e-6)
    assert torch.equal(stream, residual if d is None else residual + d.float())
    ops.check_errors(torch.device(DEV))


def gives_up(library, tokens, k, features, plan, gated, dtype):
    """A product with the build that gives up, then with the ordinary one."""
    from slipstream_b200 import ops

    def int8_rows(n):
        store = torch.randint(-127, 128, (n, (k + 15) & -16), device=DEV, dtype=torch.int8)
        return ops.Int8Rows(store[:, :k], torch.rand(n, device=DEV))

    x, w = int8_rows(tokens), int8_rows(features)
    columns = features // 2 if gated else features
    out = torch.full((tokens, columns), 7.0, device=DEV, dtype=dtype)
    many, bn, slices, per_sm, steps = plan
    call = ProductCall(x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), w=w.values.data_ptr(), ldw=w.values.stride(0),
                       w_scale=w.scales.data_ptr(), out=out.data_ptr(), ldc=columns, out_f32=int(dtype == F32), tokens=tokens, features=features,
                       K=k, gated=int(gated), out_features=columns, many=many, bn=bn, slices=slices, per_sm=per_sm, steps=steps)
    assert ran(library.ss_gemm_int8, call) == WAIT_LIMIT
    assert (out == 7).all()
    if not gated:
        sums = x.values.to(torch.float64) @ w.values.to(torch.float64).t()
        assert torch.equal(ops.linear_int8(x, w, None, F32, plan=plan), sums.to(F32) * x.scales[:, None] * w.scales)
    ops.check_errors(torch.device(DEV))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens, k, plan", [(1, 100, (0, 16, 1, 1, 1)), (9, 3584, (0, 16, 1, 2, 2)), (200, 18944, (0, 208, 1, 1, 1)), (100, 2000, (0, 48, 1, 1, 2)),
                                             (16, 3584, (0, 16, 4, 2, 2)), (33, 896, (0, 48, 2, 1, 1)), (250, 18944, (0, 256, 5, 1, 1)), (60, 300, (0, 32, 8, 1, 1))])
def test_products_of_few_tokens(products_library, tokens, k, plan, gated, dtype):
    gives_up(products_library, tokens, k, 1152, plan, gated, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens, k, features, plan", [(1, 100, 128, (1, 128, 1, 1, 1)), (300, 896, 1152, (1, 256, 1, 1, 2)), (2047, 3584, 4608, (1, 256, 1, 1, 1)),
                                                       (4099, 300, 9728, (1, 128, 1, 1, 2)), (515, 18944, 3584, (1, 256, 1, 1, 1))])
def test_products_of_many_tokens(products_library, tokens, k, features, plan, gated, dtype):
    gives_up(products_library, tokens, k, features, plan, gated, dtype)

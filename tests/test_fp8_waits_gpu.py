"""What the kernels of layers in 8-bit floats do when a wait gives up: they say so in the error word, write nothing, wait for what is in
flight to them and end, and the device goes on.  Shown by a build whose waits give up without a look (WAIT_POLLS=0), called through its
entry points; the copies of that build are real ones, and its blocks wait for them before they end, with the limit of the ordinary build."""

import ctypes
from ctypes import c_double, c_int64, c_void_p

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
WAIT_LIMIT = 8  # SS_ERR_WAIT_LIMIT


class RowsCall(ctypes.Structure):  # csrc/fp8_calls.h, Fp8RowsCall
    _fields_ = [("x", c_void_p), ("stride", c_int64), ("q", c_void_p), ("q_stride", c_int64), ("scales", c_void_p)]
    _fields_ += [(name, c_int64) for name in ("scale_row", "scale_block", "rows", "width", "dtype", "blocks", "early")]
    _fields_ += [("y", c_void_p), ("delta", c_void_p), ("weight", c_void_p), ("w_f32", c_int64), ("eps", c_double), ("err", c_void_p), ("stream", c_void_p)]


class ProductCall(ctypes.Structure):  # Fp8Call
    _fields_ = [("x", c_void_p), ("ldx", c_int64), ("x_scale", c_void_p), ("x_row", c_int64), ("x_block", c_int64), ("w", c_void_p), ("ldw", c_int64),
                ("w_scale", c_void_p), ("w_row", c_int64), ("w_block", c_int64), ("bias", c_void_p), ("bias_f32", c_int64), ("out", c_void_p), ("ldc", c_int64),
                ("out_type", c_int64), ("out_scale", c_void_p)]
    _fields_ += [(name, c_int64) for name in ("tokens", "features", "K", "gated", "out_features", "many", "bn", "slices", "per_sm")]
    _fields_ += [("err", c_void_p), ("stream", c_void_p), ("parts", c_void_p)]


@pytest.fixture(scope="module")
def library():
    from slipstream_b200.ops.library import FP8_SOURCES, compile_library

    return ctypes.CDLL(str(compile_library("slipstream_fp8", FP8_SOURCES, {"WAIT_POLLS": 0})))


def ran(entry, call):
    """The entry point's status, and the error word behind it."""
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    call.err, call.stream = err.data_ptr(), torch.cuda.current_stream().cuda_stream
    assert entry(ctypes.byref(call)) == 0
    torch.cuda.synchronize()
    return int(err.item())


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("delta, width", [(None, 4096), (BF16, 3584), (F32, 5120), (BF16, 8192), (F32, 6144)])
def test_norm_of_many_rows(library, delta, width, in_place):
    from slipstream_b200 import ops

    rows = 2400
    residual, weight = torch.randn(rows, width, device=DEV), torch.ones(width, device=DEV)
    d = None if delta is None else torch.randn(rows, width, device=DEV).to(delta)
    out = residual if in_place else torch.full_like(residual, 7.0)
    before = out.clone()
    blocks = -(-width // 128)
    q, scales = torch.full((rows, width), 55, dtype=torch.uint8, device=DEV), torch.full((blocks, rows), 7.0, device=DEV)
    call = RowsCall(x=residual.data_ptr(), stride=width, q=q.data_ptr(), q_stride=width, scales=scales.data_ptr(), scale_row=1, scale_block=rows, rows=rows,
                    width=width, dtype=int(delta != F32), y=out.data_ptr(), delta=None if d is None else d.data_ptr(), weight=weight.data_ptr(), w_f32=1, eps=1e-6)
    assert ran(library.ss_add_rmsnorm_fp8, call) == WAIT_LIMIT
    assert torch.equal(out, before) and (q == 55).all() and (scales == 7).all()
    stream = residual.clone()
    ops.add_rmsnorm_fp8(stream, d, weight, 1e-6)
    assert torch.equal(stream, residual if d is None else residual + d.float())
    ops.check_errors(torch.device(DEV))


def gives_up(library, tokens, k, features, plan, gated, dtype):
    """A product with the build that gives up, then with the ordinary one."""
    from slipstream_b200 import ops

    def values(n):
        store = torch.randint(0, 120, (n, (k + 15) & -16), device=DEV, dtype=torch.uint8).view(E4M3)
        return store[:, :k]

    blocks = -(-k // 128)
    x, w = ops.Fp8Rows(values(tokens), torch.rand(blocks, tokens, device=DEV).t()), ops.Fp8Blocks(values(features), torch.rand(-(-features // 128), blocks, device=DEV))
    columns = features // 2 if gated else features
    pitch = (columns + 15) & -16 if dtype == E4M3 else columns
    out = torch.full((tokens, pitch), 7, device=DEV, dtype=torch.uint8) if dtype == E4M3 else torch.full((tokens, pitch), 7.0, device=DEV, dtype=dtype)
    out_scale = torch.full((-(-columns // 128), tokens), 7.0, device=DEV)
    bias = torch.ones(features, device=DEV)
    many, bn, slices, per_sm = plan
    parts = torch.empty(slices, tokens, (features + 3) & -4, device=DEV)
    call = ProductCall(x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), x_row=1, x_block=tokens, w=w.values.data_ptr(),
                       ldw=w.values.stride(0), w_scale=w.scales.data_ptr(), w_row=blocks, w_block=1, bias=bias.data_ptr(), bias_f32=1, out=out.data_ptr(), ldc=pitch,
                       out_type={F32: 0, BF16: 1, E4M3: 2}[dtype], out_scale=out_scale.data_ptr(), tokens=tokens, features=features, K=k, gated=int(gated),
                       out_features=columns, many=many, bn=bn, slices=slices, per_sm=per_sm, parts=parts.data_ptr())
    assert ran(library.ss_gemm_fp8, call) == WAIT_LIMIT
    assert (out == 7).all() and (out_scale == 7).all()
    got = ops.gate_up_swiglu_fp8(x, w, bias, dtype, plan=plan) if gated else ops.linear_fp8(x, w, bias, dtype, plan=plan)
    assert got.shape == (tokens, columns)
    ops.check_errors(torch.device(DEV))


TYPES = [(False, F32), (False, BF16), (True, F32), (True, BF16), (True, E4M3)]


@pytest.mark.parametrize("gated, dtype", TYPES)
@pytest.mark.parametrize("tokens, k, plan", [(1, 100, (0, 16, 1, 1)), (9, 3584, (0, 16, 1, 2)), (100, 18944, (0, 128, 1, 1)), (90, 2000, (0, 48, 1, 1)),
                                             (16, 3584, (0, 16, 4, 2)), (33, 896, (0, 48, 2, 1)), (95, 18944, (0, 96, 5, 1)), (60, 1100, (0, 32, 8, 1))])
def test_products_of_few_tokens(library, tokens, k, plan, gated, dtype):
    gives_up(library, tokens, k, 1280, plan, gated, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens, k, features, plan", [(256, 18944, 3584, (1, 256, 5, 1)), (100, 300, 1279, (1, 128, 2, 1)), (700, 2000, 5000, (1, 128, 8, 1))])
def test_products_of_many_tokens_in_slices(library, tokens, k, features, plan, dtype):
    gives_up(library, tokens, k, features, plan, False, dtype)


@pytest.mark.parametrize("gated, dtype", TYPES)
@pytest.mark.parametrize("tokens, k, features, tile", [(1, 100, 256, 64), (300, 896, 1280, 128), (2047, 3584, 4608, 256), (4099, 300, 9728, 128), (515, 18944, 3584, 64)])
def test_products_of_many_tokens(library, tokens, k, features, tile, gated, dtype):
    gives_up(library, tokens, k, features, (1, 256 if gated else tile, 1, 1), gated, dtype)

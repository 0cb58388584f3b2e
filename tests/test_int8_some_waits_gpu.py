"""What the int8 products of few tokens do when the waits of some blocks give up and those of others do not: nothing is written that was
formed from what they did not form, all else is, and the error word says so.  Shown by a build in which the waits of a second slice of K and
of blocks 2 and 3 of a row of blocks give up without a look (SOME_WAITS_GIVE_UP), called through its entry points."""

import ctypes

import pytest
import torch

from test_int8_waits_gpu import BF16, DEV, F32, WAIT_LIMIT, ProductCall, ran

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def library():
    from slipstream_b200.ops.library import compile_library

    return ctypes.CDLL(str(compile_library("slipstream_int8_products", ["gemm_int8.cu"], {"SOME_WAITS_GIVE_UP": 1})))


def products(library, tokens, k, features, plan, gated, dtype):
    """(what the build leaves in an output of sevens, what the ordinary one makes of the same operands)"""
    from slipstream_b200 import ops

    gen = torch.Generator(device=DEV).manual_seed(tokens + k)

    def int8_rows(n):
        store = torch.randint(-127, 128, (n, (k + 15) & -16), device=DEV, dtype=torch.int8, generator=gen)
        return ops.Int8Rows(store[:, :k], torch.rand(n, device=DEV, generator=gen) / 1000)

    x, w = int8_rows(tokens), int8_rows(features)
    columns = features // 2 if gated else features
    out = torch.full((tokens, columns), 7.0, device=DEV, dtype=dtype)
    many, bn, slices, per_sm, steps = plan
    call = ProductCall(x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), w=w.values.data_ptr(), ldw=w.values.stride(0),
                       w_scale=w.scales.data_ptr(), out=out.data_ptr(), ldc=columns, out_f32=int(dtype == F32), tokens=tokens, features=features,
                       K=k, gated=int(gated), out_features=columns, many=many, bn=bn, slices=slices, per_sm=per_sm, steps=steps)
    assert ran(library.ss_gemm_int8, call) == WAIT_LIMIT
    whole = ops.gate_up_swiglu_int8(x, w, None, dtype, plan=plan) if gated else ops.linear_int8(x, w, None, dtype, plan=plan)
    ops.check_errors(torch.device(DEV))
    return out, whole


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens, k, plan", [(16, 3584, (0, 16, 4, 2, 2)), (33, 896, (0, 48, 2, 1, 1)), (250, 18944, (0, 256, 5, 1, 1)), (60, 1100, (0, 32, 8, 1, 1)),
                                             (1, 300, (0, 16, 3, 1, 1))])
def test_a_slice_of_few_tokens(library, tokens, k, plan, gated, dtype):
    """Every tile has a slice whose block gives up, so no block writes, whichever columns it owns."""
    out, _ = products(library, tokens, k, 1152, plan, gated, dtype)
    assert (out == 7).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens, k, tile", [(70, 3584, 16), (100, 300, 32), (200, 2000, 48)])
def test_tiles_of_few_tokens(library, tokens, k, tile, gated, dtype):
    """Tiles of tokens 2 and 3 give up; the others are right."""
    out, whole = products(library, tokens, k, 1152, (0, tile, 1, 1, 1), gated, dtype)
    lost = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    lost[2 * tile: 4 * tile] = True
    assert (out[lost] == 7).all() and torch.equal(out[~lost], whole[~lost])

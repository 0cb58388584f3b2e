"""What the products of 8-bit floats do when the waits of some blocks give up and those of others do not: nothing is written that was formed
from what they did not form, all else is, and the error word says so.  Shown by a build in which the waits of a second slice of K and of
blocks 2 and 3 of a row of blocks give up without a look (SOME_WAITS_GIVE_UP), called through its entry points."""

import ctypes

import pytest
import torch

from test_fp8_waits_gpu import BF16, DEV, E4M3, F32, TYPES, WAIT_LIMIT, ProductCall, ran

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def library():
    from slipstream_b200.ops.library import FP8_SOURCES, compile_library

    return ctypes.CDLL(str(compile_library("slipstream_fp8", FP8_SOURCES, {"SOME_WAITS_GIVE_UP": 1})))


def products(library, tokens, k, features, plan, gated, dtype, word=0):
    """(what the build leaves in an output of sevens, its scales, what the ordinary one makes of the same operands, its scales)
    ``word``: an error that stands in the error word already; the build is then the ordinary one."""
    from slipstream_b200 import ops

    blocks, gen = -(-k // 128), torch.Generator(device=DEV).manual_seed(tokens + k)

    def values(n):
        store = torch.randint(0, 120, (n, (k + 15) & -16), device=DEV, dtype=torch.uint8, generator=gen).view(E4M3)
        return store[:, :k]

    x = ops.Fp8Rows(values(tokens), torch.rand(blocks, tokens, device=DEV, generator=gen).t())
    w = ops.Fp8Blocks(values(features), torch.rand(-(-features // 128), blocks, device=DEV, generator=gen))
    columns = features // 2 if gated else features
    pitch = (columns + 15) & -16 if dtype == E4M3 else columns
    out = torch.full((tokens, pitch), 7, device=DEV, dtype=torch.uint8) if dtype == E4M3 else torch.full((tokens, pitch), 7.0, device=DEV, dtype=dtype)
    out_scale = torch.full((-(-columns // 128), tokens), 7.0, device=DEV)
    many, bn, slices, per_sm = plan
    parts = torch.zeros(slices, tokens, (features + 3) & -4, device=DEV)
    call = ProductCall(x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), x_row=1, x_block=tokens, w=w.values.data_ptr(),
                       ldw=w.values.stride(0), w_scale=w.scales.data_ptr(), w_row=blocks, w_block=1, out=out.data_ptr(), ldc=pitch,
                       out_type={F32: 0, BF16: 1, E4M3: 2}[dtype], out_scale=out_scale.data_ptr(), tokens=tokens, features=features, K=k, gated=int(gated),
                       out_features=columns, many=many, bn=bn, slices=slices, per_sm=per_sm, parts=parts.data_ptr())
    if word:
        err = torch.full((1,), word, dtype=torch.int32, device=DEV)
        call.err, call.stream = err.data_ptr(), torch.cuda.current_stream().cuda_stream
        assert library.ss_gemm_fp8(ctypes.byref(call)) == 0
        assert int(err.item()) == word
    else:
        assert ran(library.ss_gemm_fp8, call) == WAIT_LIMIT
    whole = ops.gate_up_swiglu_fp8(x, w, None, dtype, plan=plan) if gated else ops.linear_fp8(x, w, None, dtype, plan=plan)
    ops.check_errors(torch.device(DEV))
    if dtype == E4M3:
        return out[:, :columns], out_scale, whole.values.view(torch.uint8), whole.scales.t()
    return out, out_scale, whole, out_scale


@pytest.mark.parametrize("gated, dtype", TYPES)
@pytest.mark.parametrize("tokens, k, plan", [(16, 3584, (0, 16, 4, 1)), (33, 896, (0, 48, 2, 1)), (95, 18944, (0, 32, 5, 1)), (60, 1100, (0, 32, 8, 1)), (1, 300, (0, 16, 3, 1))])
def test_a_slice_of_few_tokens(library, tokens, k, plan, gated, dtype):
    """Every tile has a slice whose block gives up, so no block writes, whichever columns it owns."""
    out, scale, _, _ = products(library, tokens, k, 1280, plan, gated, dtype)
    assert (out == 7).all() and (scale == 7).all()


@pytest.mark.parametrize("gated, dtype", TYPES)
@pytest.mark.parametrize("tokens, k, tile", [(70, 3584, 16), (100, 300, 32), (200, 2000, 48)])
def test_tiles_of_few_tokens(library, tokens, k, tile, gated, dtype):
    """Tiles of tokens 2 and 3 give up; the others are right."""
    out, scale, whole, whole_scale = products(library, tokens, k, 1280, (0, tile, 1, 1), gated, dtype)
    lost = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    lost[2 * tile: 4 * tile] = True
    assert (out[lost] == 7).all() and torch.equal(out[~lost], whole[~lost])
    if dtype == E4M3:
        assert (scale[:, lost] == 7).all() and torch.equal(scale[:, ~lost], whole_scale[:, ~lost])


SLICED = [(256, 18944, 3584, (1, 256, 5, 1)), (100, 300, 1279, (1, 128, 2, 1)), (700, 2000, 5000, (1, 128, 8, 1))]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens, k, features, plan", SLICED)
def test_a_pair_of_many_tokens_in_slices(library, tokens, k, features, plan, dtype):
    """A pair of blocks gives up: tiles of which it forms a part are left as they are, the others are right."""
    out, _, whole, _ = products(library, tokens, k, features, plan, False, dtype)
    _, tile, slices, _ = plan
    blocks = -(-k // 128)
    slices = -(-blocks // -(-blocks // slices))  # (that have any K)
    down = -(-tokens // 256)
    tiles = down * -(-features // tile)
    pairs = min(tiles * slices, torch.cuda.get_device_properties(DEV).multi_processor_count // 2)
    lost = torch.zeros(tokens, features, dtype=torch.bool, device=DEV)
    for t in range(1, tiles * slices, pairs):
        m, f = t % tiles % down * 256, t % tiles // down * tile
        lost[m: m + 256, f: f + tile] = True
    assert lost.any() and (out[lost] == 7).all() and torch.equal(out[~lost], whole[~lost])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens, k, features, plan", SLICED)
def test_an_error_of_another_call(tokens, k, features, plan, dtype):
    """A wait of another call gave up, and nobody has read the error word yet: this call's result is whole all the same."""
    from slipstream_b200.ops.functions import fp8_library

    out, _, whole, _ = products(fp8_library(), tokens, k, features, plan, False, dtype, word=WAIT_LIMIT)
    assert torch.equal(out, whole)

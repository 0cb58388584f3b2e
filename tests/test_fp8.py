"""Layers in 8-bit floats on the host: the products' plans, the layout of stacked weights, what is refused before a kernel is looked for."""

import pytest
import torch

from slipstream_b200.ops.fp8 import FP8_BLOCK, Fp8Blocks, Fp8Rows, dequantize_fp8, fp8_plan, gate_up_swiglu_fp8, linear_fp8, stack_gate_up_fp8
from slipstream_b200.ops.functions import KernelError

RESIDENT = ((148, 74, 45, 33, 26, 22, 15, 15), (296, 148, 93, 71, 56, 45, 37, 33))


@pytest.mark.parametrize("resident", [None, RESIDENT, ((1,) * 8, (1,) * 8)])
@pytest.mark.parametrize("sms", [1, 2, 80, 148])
def test_plans_are_forms_that_the_kernels_have(sms, resident):
    for gated in (False, True):
        parts = 2 if gated else 1
        for tokens in (1, 2, 15, 16, 17, 100, 129, 255, 256, 257, 640, 641, 5000, 100000):
            for features, k in ((256, 1), (256, 17), (256, 128), (1280, 896), (4608, 3584), (3584, 18944), (37888, 3584), (256, 1000000)):
                many, tile, slices, per = fp8_plan(tokens, features, k, sms, gated, resident)
                if many:
                    assert tile in (64, 128, 256) and tokens > 32 and (not gated or tile == 256)
                    assert slices == 1 or (not gated and tile > 64 and 2 <= slices <= min(8, -(-k // 256)) and per == 1)
                else:
                    assert tile % 16 == 0 and 16 <= tile <= 256 // parts and 1 <= slices <= min(8, -(-k // 128)) and tokens <= 640
                    assert per == 1 or (per == 2 and tile <= 64 // parts)
                    # what the kernel keeps in shared memory: two stages of the ring, the factors, and where K is cut the sums that it owns
                    half = next(c for c in (8, 16, 32, 64, 128) if 2 * c >= tile)
                    floats = (8 if parts * half <= 32 else 4) * -(-(half + parts) // 4) * 4 + 2 * parts * half
                    rest = 1536 + 32 * floats + (slices * -(-tile // slices) * 512 * parts if slices > 1 else 0)
                    assert 2 * (128 * parts + tile) * 128 + rest <= 232448


def test_plans_of_more_features_than_a_grid_has_rows_for_their_tiles():
    """The kernel for few tokens has its tiles of features along grid.y: up to 65,535 of them."""
    for tokens in (1, 32, 65, 640, 700):
        assert tokens > 32 or fp8_plan(tokens, 65535 * 128, 16, 148, False, RESIDENT)[0] == 0
        assert fp8_plan(tokens, 65535 * 128 + 128, 16, 148, False, RESIDENT)[0] == 1


def test_plans_do_not_change_within_a_step_of_tokens():
    for tokens in (1, 17, 300, 1000):
        step = 16 if tokens <= 640 else 256
        upto = -(-tokens // step) * step
        assert fp8_plan(tokens, 4608, 3584, 148, False, RESIDENT) == fp8_plan(upto, 4608, 3584, 148, False, RESIDENT)


def test_stacked_gate_and_up_rows():
    for rows in (1, 127, 128, 129, 400):
        gate, up = torch.randn(rows, 3), torch.randn(rows, 3)
        stacked = stack_gate_up_fp8(gate, up)
        runs = stacked.reshape(-1, 2, FP8_BLOCK, 3)
        assert torch.equal(runs[:, 0].reshape(-1, 3)[:rows], gate) and torch.equal(runs[:, 1].reshape(-1, 3)[:rows], up)
        assert not runs[:, 0].reshape(-1, 3)[rows:].any() and not runs[:, 1].reshape(-1, 3)[rows:].any()
    assert stack_gate_up_fp8(torch.ones(5), torch.zeros(5)).shape == (256,)
    with pytest.raises(KernelError):
        stack_gate_up_fp8(torch.ones(5), torch.ones(6))


def test_operands_of_the_wrong_kind():
    values, scales = torch.zeros(128, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    rows, blocks = Fp8Rows(values, scales.expand(128, 1)), Fp8Blocks(values, scales)
    assert rows.shape == (128, 128) and blocks.nbytes() == 128 * 128 + 4
    for call in (lambda: linear_fp8(values, blocks), lambda: linear_fp8(rows, values), lambda: linear_fp8(blocks, blocks), lambda: linear_fp8(rows, rows),
                 lambda: gate_up_swiglu_fp8(rows, rows), lambda: linear_fp8(rows, blocks, None, torch.float8_e4m3fn), lambda: dequantize_fp8(values, torch.float32)):
        with pytest.raises(KernelError):
            call()

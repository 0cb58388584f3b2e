"""The host side of the 8-bit float operators' calls: what is counted."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_launches_of_products_in_slices():
    """A product of many tokens with K in slices is two kernels, a plan that is refused none."""
    from slipstream_b200 import ops

    rows, w = ops.quantize_rows_fp8(torch.ones(40, 512, device=DEV)), ops.quantize_blocks_fp8(torch.ones(256, 512, device=DEV))
    for plan, launches in (((1, 128, 1, 1), 1), ((1, 128, 2, 1), 2), ((1, 256, 4, 1), 2)):
        before = ops.launch_count()
        ops.linear_fp8(rows, w, plan=plan)
        assert ops.launch_count() - before == launches
    for call in (lambda: ops.linear_fp8(rows, w, plan=(1, 64, 2, 1)), lambda: ops.linear_fp8(rows, w, plan=(1, 128, 9, 1)),
                 lambda: ops.gate_up_swiglu_fp8(rows, w, plan=(1, 256, 2, 1))):
        before = ops.launch_count()
        with pytest.raises(ops.KernelError):
            call()
        assert ops.launch_count() == before

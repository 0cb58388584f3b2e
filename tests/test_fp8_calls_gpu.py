"""The host side of the 8-bit float operators' calls: what is counted, how wide a weight may be."""

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


def test_weights_of_more_than_65535_blocks_a_row():
    """Rounded by the definition, back, and a product of them: ones in the last 300 elements, 300 of them counted."""
    from slipstream_b200 import ops
    from test_fp8_gpu import check_definition

    width = 65536 * 128 + 100
    x = torch.randn(3, width, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).to(torch.bfloat16)
    got = ops.quantize_blocks_fp8(x)
    assert got.scales.shape == (1, 65537)
    check_definition(got, x, 128)
    ones = torch.zeros(2, width, device=DEV, dtype=torch.bfloat16)
    ones[:, -300:] = 1
    w, rows = ops.quantize_blocks_fp8(ones), ops.quantize_rows_fp8(ones)
    assert torch.equal(w.dequantize(torch.bfloat16), ones)
    # (448 * (1 / 448) is 1 but for two roundings of 2^-24 a factor, and three blocks are added)
    assert ((ops.linear_fp8(rows, w, out_dtype=torch.float32) - 300).abs() <= 300 * 8 * 2.0 ** -24).all()

"""The host side of the 8-bit float operators' calls: what is counted, how wide a weight may be, NaN in products with K in slices."""

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


def test_scales_that_are_nan_in_slices():
    """They make their rows and features NaN, whatever their bits (those that the kernels mark unformed sums with among them)."""
    from slipstream_b200 import ops

    gen = torch.Generator(device=DEV).manual_seed(3)
    x, w = (f(torch.randn(n, 1000, device=DEV, generator=gen)) for f, n in ((ops.quantize_rows_fp8, 70), (ops.quantize_blocks_fp8, 700)))
    plan = (1, 128, 4, 1)
    whole = ops.linear_fp8(x, w, None, torch.float32, plan=plan)
    for bits in (0x7FC0BEEF, 0x7FFFFFFF, 0x7F800001):
        nan = torch.tensor([bits], dtype=torch.int32, device=DEV).view(torch.float32)
        scales = x.scales.clone()
        scales[33, 2] = nan
        out = ops.linear_fp8(ops.Fp8Rows(x.values, scales), w, None, torch.float32, plan=plan)
        assert out[33].isnan().all() and torch.equal(out[:33], whole[:33]) and torch.equal(out[34:], whole[34:])
        scales = w.scales.clone()
        scales[1, 7] = nan
        out = ops.linear_fp8(x, ops.Fp8Blocks(w.values, scales), None, torch.float32, plan=plan)
        assert out[:, 128:256].isnan().all() and torch.equal(out[:, :128], whole[:, :128]) and torch.equal(out[:, 256:], whole[:, 256:])

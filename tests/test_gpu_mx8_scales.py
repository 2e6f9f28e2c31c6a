"""Every scale byte of the 8-bit form is read as what it stands for, also those the kernels themselves do not write."""

import pytest
import torch

from helpers import DTYPES, announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 35])
def test_all_scale_bytes(gpu, dtype, width):
    """code * 2^(scale - 133) has seven magnitude bits and is no smaller than 2^-133: exact in fp32 and bf16 (whose smallest
    number is 2^-133).  fp16: the value rounded once, to nearest even, and its largest finite number beyond the range."""
    from cute_kernels import mx8_dequantize_cute, mx8_dequantize_torch

    announce("mx8 scale bytes", dtype, width)
    blocks = -(-width // 32)
    scales = torch.arange(255, dtype=torch.uint8).view(255, 1).expand(255, blocks).contiguous()
    codes = torch.arange(255 * width).remainder(255).sub(127).to(torch.int8).view(255, width)
    codes[:, :4] = torch.tensor([127, -127, 1, 0], dtype=torch.int8)
    exact = codes.double() * torch.pow(2.0, scales.double()[:, :1] - 133)
    want = exact.clamp(-65504.0, 65504.0).to(dtype) if dtype == torch.float16 else exact.to(dtype)
    if dtype != torch.float16:
        assert torch.equal(want.double(), exact) and int((want[:7] != 0).sum()) > 7 * 28
    values = mx8_dequantize_cute(codes.to(gpu), scales.to(gpu), dtype)
    assert values.dtype == dtype and torch.equal(values.cpu(), want)
    assert torch.equal(mx8_dequantize_torch(codes, scales, dtype), want)
    scales[:] = 255
    assert mx8_dequantize_cute(codes.to(gpu), scales.to(gpu), dtype).isnan().all()


def test_products_of_small_blocks(gpu):
    """The routing weights' gradient from expert outputs whose scale bytes are below 7: sums of code * 2^(scale - 133) * dy, with
    dy a power of two that brings them back among the normal numbers."""
    from cute_kernels.kernels.scattermoe.ops import moe_combine_backward_gates_mx8

    announce("mx8 small blocks")
    codes = torch.arange(2 * 7 * 32).remainder(255).sub(127).to(torch.int8).view(2, 7, 32)
    scales = torch.arange(7, dtype=torch.uint8).view(1, 7, 1).expand(2, 7, 1).contiguous()
    dy = torch.full((2, 32), 2.0 ** 100)
    want = (codes.double() * torch.pow(2.0, scales.double() - 133) * 2.0 ** 100).sum(-1)
    d_gates = torch.empty(2, 7, device=gpu)
    moe_combine_backward_gates_mx8(codes.to(gpu), scales.to(gpu), dy.to(gpu), d_gates)
    assert torch.equal(d_gates.cpu().double(), want)  # whole numbers times a power of two: no rounding anywhere

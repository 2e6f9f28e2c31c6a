"""Activations in 8 bits: MXINT8 of the OCP microscaling formats, for what a training step keeps between forward and backward.

A block is 32 consecutive elements of a row (the last one of a row may be shorter).  It has one scale byte ``b`` and an int8
code ``q`` in [-127, 127] per element, which stands for ``q * 2 ** (b - 133)``.  ``b`` is the smallest exponent (7 .. 254; smaller
ones written elsewhere are read too) for which the block's largest magnitude rounds to at most 127 steps, so an element is off by at most half a step: 1/254 to 1/127 of that
magnitude.  Scaling by a power of two is exact: codes depend on nothing but the values, and writing what was read
back changes nothing.  A block with a NaN or an infinity has scale byte 255 and stands for NaNs.

The pair here is for what a caller keeps itself.  ``swiglu_cute``, ``swiglu_unchunked_cute``, ``rmsnorm_cute`` and
``fused_residual_add_rmsnorm_cute`` take ``checkpoint_8bit=True`` and ``MoE_HIP`` has the attribute ``checkpoint_8bit``: their
forward writes the 8-bit form in the pass that computes the result, and their backward works from it.

The reference has no counterpart; its nearest relative is ``memory_efficient`` of its RMSNorm
(cute_kernels/kernels/rmsnorm/__init__.py:11-106), which recomputes 1 / rms instead of saving it.
"""

import torch

from .. import _C, _native
from ..constants import LIBRARY_NAME
from ..utils import cute_op


def mx8_quantize_torch(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    H = x.size(-1)
    blocks = torch.nn.functional.pad(x.float(), (0, -H % _C.MX8_BLOCK)).unflatten(-1, (-1, _C.MX8_BLOCK))
    finite = blocks.isfinite().all(dim=-1, keepdim=True)
    blocks = torch.where(finite, blocks, torch.zeros_like(blocks))
    largest = blocks.abs().amax(dim=-1, keepdim=True)
    # the addend carries into the exponent where the largest magnitude would round to 128 steps
    exponent = ((largest.view(torch.int32) + 0x10000) >> 23).clamp(7, 254)
    inverse = ((260 - exponent) << 23).view(torch.float32)
    codes = (blocks * inverse).round().clamp(-127, 127).to(torch.int8)
    scales = torch.where(finite, exponent, torch.full_like(exponent, 255)).to(torch.uint8)
    return codes.flatten(-2)[..., :H].contiguous(), scales.squeeze(-1)


def mx8_dequantize_torch(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    H = codes.size(-1)
    exponent = scales.to(torch.int32)
    # 2 ** (exponent - 133): below 7 a subnormal number, one bit of the mantissa
    bits = torch.where(exponent < 7, 1 << (exponent.clamp(max=6) + 16), (exponent.clamp(min=7) - 6) << 23)
    steps = torch.where(exponent == 255, float("nan"), bits.to(torch.int32).view(torch.float32))
    x = codes.float() * steps.repeat_interleave(_C.MX8_BLOCK, dim=-1)[..., :H]
    if dtype == torch.float16:
        x = x.clamp(-65504.0, 65504.0)
    return x.to(dtype)


def new_mx8(shape, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    """Memory for the codes and scale bytes of a tensor of this shape (two dimensions or more)."""
    return (
        torch.empty(shape, dtype=torch.int8, device=device),
        torch.empty(*shape[:-1], _C.mx8_blocks(shape[-1]), dtype=torch.uint8, device=device),
    )


def new_kept(rows: int, H: int, device: torch.device, with_rstd: bool = False) -> torch.Tensor:
    """Memory for what an operator keeps of ``rows`` rows of H elements: one buffer, laid out by ``_C.mx8_kept_offsets``."""
    return torch.empty(_C.mx8_kept_offsets(rows, H, with_rstd)[2], dtype=torch.int8, device=device)


def kept_pair(kept: torch.Tensor, shape) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes and scale bytes inside a buffer of ``new_kept`` for rows that lie in this shape."""
    H = shape[-1]
    rows = 1
    for n in shape[:-1]:
        rows *= n
    start, end, _ = _C.mx8_kept_offsets(rows, H, False)
    codes = kept[: rows * H].view(shape)
    return codes, kept[start:end].view(torch.uint8).view(*shape[:-1], _C.mx8_blocks(H))


@cute_op(f"{LIBRARY_NAME}::mx8_quantize_hip", mutates_args={"codes", "scales"})
def mx8_quantize_hip(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> None:
    _C.mx8_quantize(x, codes, scales)


@cute_op(f"{LIBRARY_NAME}::mx8_dequantize_hip", mutates_args={"output"})
def mx8_dequantize_hip(codes: torch.Tensor, scales: torch.Tensor, output: torch.Tensor) -> None:
    _C.mx8_dequantize(codes, scales, output)


def mx8_quantize_cute(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)``: int8 of x's shape, and uint8 ``[..., ceil(H / 32)]``.  float32, float16 or bfloat16; not
    differentiable (a checkpoint is read in a backward, not differentiated through)."""
    functions = _native.functions_for(x)
    if functions is not None:
        return functions.mx8_quantize(x)
    if x.dim() == 0:
        raise ValueError("mx8_quantize_cute: x needs at least one dimension")
    rows = x.detach().unsqueeze(0) if x.dim() == 1 else x.detach()
    rows = rows.contiguous()
    codes, scales = new_mx8(rows.shape, x.device)
    mx8_quantize_hip(rows, codes, scales)
    return (codes.squeeze(0), scales.squeeze(0)) if x.dim() == 1 else (codes, scales)


def mx8_dequantize_cute(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values ``(codes, scales)`` stand for: exact in float32 and bfloat16, rounded to float16 where they lie among its
    subnormal numbers (beyond its range: its largest finite number)."""
    functions = _native.functions_for(codes)
    if functions is not None:
        return functions.mx8_dequantize(codes, scales, dtype)
    if codes.dim() == 0:
        raise ValueError("mx8_dequantize_cute: codes need at least one dimension")
    is_1d = codes.dim() == 1
    if is_1d:
        codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
    output = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    mx8_dequantize_hip(codes.contiguous(), scales.contiguous(), output)
    return output.squeeze(0) if is_1d else output

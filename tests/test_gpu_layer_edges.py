"""Edges of the MoE layer and of the operators with an 8-bit checkpoint."""

import pytest
import torch

from helpers import DTYPES, announce
from test_gpu_mx8 import _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint_8bit", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_tokens(gpu, dtype, checkpoint_8bit):
    """A batch without tokens gives empty results and zero weight gradients, also where the output's gradient is an expanded
    tensor, as a sum's is (its strides are zero, and empty tensors count as contiguous)."""
    announce("layer without tokens", dtype, checkpoint_8bit)
    for H, I in ((64, 128), (72, 40)):
        moe, x, dy = _layer(gpu, dtype, 4, H, I, 4, 2, 121)
        moe.checkpoint_8bit = checkpoint_8bit
        for dense in (True, False):
            moe.zero_grad()
            v = x[:0].to(gpu).requires_grad_(True)
            y, logits = moe(v)
            balance, z, counts = moe.balance_loss(logits)
            if dense:
                torch.autograd.backward((y, balance), (dy[:0].to(gpu), None))
            else:
                (y.sum() + balance).backward()
            assert y.shape == (0, H) and v.grad.shape == (0, H) and not counts.any()
            assert all(not p.grad.any() for p in moe.parameters())


def test_refusals_are_those_of_the_ordinary_call(gpu):
    """Odd rows of a one-tensor SwiGLU and tensors without a dimension, with and without the checkpoint, traced and eager."""
    import cute_kernels as ck
    from cute_kernels.utils import set_cute_tracing

    announce("refusals of the checkpoints")
    odd = torch.randn(4, 63, device=gpu, requires_grad=True)
    scalar = torch.tensor(1.0, device=gpu, requires_grad=True)
    for tracing in (False, True):
        set_cute_tracing(tracing)
        try:
            for checkpoint_8bit in (False, True):
                with pytest.raises(AssertionError, match="even"):
                    ck.swiglu_unchunked_cute(odd, checkpoint_8bit=checkpoint_8bit)
                with pytest.raises(IndexError):
                    ck.rmsnorm_cute(scalar, None, 1e-5, checkpoint_8bit=checkpoint_8bit)
            with pytest.raises(ValueError, match="one dimension"):
                ck.swiglu_cute(scalar, scalar.detach(), checkpoint_8bit=True)
        finally:
            set_cute_tracing(False)

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

"""SwiGLU in fp32 far down the negative gates, where the sigmoid is small: the result keeps its relative accuracy there.

y = up * gate * sigmoid(gate) with sigmoid(x) = e / (1 + e), e = exp(x), for x < 0.  Every factor is known relative to itself:
the exponential to 1 ulp (2^-23), the addition, the division and the three products to 2^-24 each, so y is off by at most
7 * 2^-24 < 2^-21 of itself; dup = dy * gate * sigmoid likewise.  dgate = dy * up * (s + gate * s * (1 - s)): s and 1 - s by
5 * 2^-24 each, and five more operations: 2^-20 of the magnitudes that are added."""

import pytest
import torch

from helpers import announce, randn
from test_gpu_mx8 import assert_rounded, kept64, swiglu64

pytestmark = pytest.mark.gpu


def _far_gates():
    """Gates from -0.5 down to -80 (exp is a normal number down to -87.3), and a few beside them that are not negative."""
    gate = torch.linspace(-80.0, -0.5, 33 * 64 + 5)
    gate = torch.cat([gate, torch.tensor([-8.0, -10.0, -14.0, -17.0, -18.0, -40.0, 0.0, 0.25, 3.0, 20.0, 90.0])])
    gate = gate[: gate.numel() // 4 * 4].view(4, -1).contiguous()
    return gate, randn(gate.shape, torch.float32, 91), randn(gate.shape, torch.float32, 92)


@pytest.mark.parametrize("one_tensor", [False, True])
@pytest.mark.parametrize("checkpoint_8bit", [False, True])
def test_far_gates_fp32(gpu, checkpoint_8bit, one_tensor):
    from cute_kernels import swiglu_cute, swiglu_unchunked_cute

    announce("swiglu far gates", checkpoint_8bit, one_tensor)
    gate, up, dy = _far_gates()
    if one_tensor:
        x = torch.cat([up, gate], dim=-1).to(gpu).requires_grad_(True)
        y = swiglu_unchunked_cute(x, checkpoint_8bit=checkpoint_8bit)
        d_up, d_gate = torch.autograd.grad(y, x, dy.to(gpu))[0].chunk(2, dim=-1)
    else:
        g, u = gate.to(gpu, copy=True).requires_grad_(True), up.to(gpu, copy=True).requires_grad_(True)
        y = swiglu_cute(g, u, checkpoint_8bit=checkpoint_8bit)
        d_gate, d_up = torch.autograd.grad(y, (g, u), dy.to(gpu))
    d64 = dy.double()
    g, u = gate.double(), up.double()
    assert_rounded(y, swiglu64(g, u), torch.float32, 2.0 ** -21, what="y")
    if checkpoint_8bit:
        g, u = kept64(gate), kept64(up)
    s = torch.sigmoid(g)
    assert_rounded(d_up, d64 * g * s, torch.float32, 2.0 ** -21, what="d_up")
    assert_rounded(d_gate, d64 * u * (s + g * s * (1 - s)), torch.float32, 2.0 ** -20,
                   (d64 * u).abs() * (s + (g * s * (1 - s)).abs()), what="d_gate")

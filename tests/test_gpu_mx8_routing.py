"""The routing weights' share of the 8-bit layer's backward, step by step: the gradient of the routing weights from the kept
expert outputs, and the router's weight gradient from it."""

import pytest
import torch

from helpers import DTYPES, announce
from test_gpu_mx8 import _layer, assert_rounded, kept64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(100, 64, 128, 4, 2), (96, 72, 40, 5, 3)])
def test_routing_gradients(gpu, dtype, shape, monkeypatch):
    """d_gates[t, s] = <kept y[t, s], dy[t]> with the expert outputs the layer kept: fp32 evaluation as in the kernel's own test
    (a lane adds 8, the wave 6 more), rounded once.  Then, with g the softmax of the selected logits,
    d_logits[t, s] = g (d_gates - sum g d_gates), rounded, and d_weight[e] = sum_t d_logits[t, e] x[t], rounded.  A rounding is
    half a step, u = eps / 2 of the value: d_logits is off by u g (|d| + sum g |d|) for d_gates' rounding, u of itself for its
    own, and 2^-20 of those magnitudes for the softmax in fp32; d_weight by that times |x| summed over the tokens, 2^-16 of its
    terms for the fp32 sum (100 of them), and u of itself."""
    from cute_kernels.kernels.scattermoe import ops

    T, H, I, E, k = shape
    announce("layer 8-bit routing", dtype, shape)
    moe, x, dy = _layer(gpu, dtype, T, H, I, E, k, 111)
    moe.checkpoint_8bit = True
    kept = []
    quantize = ops.mx8_quantize_hip
    monkeypatch.setattr(ops, "mx8_quantize_hip", lambda rows, *out: kept.append(rows.detach().cpu()) or quantize(rows, *out))
    routing = []
    route = moe._compute_routing_weights

    def routed(rows):
        logits, weights, selected = route(rows)
        weights.retain_grad()
        routing.append((logits.detach().cpu(), weights, selected.cpu()))
        return logits, weights, selected

    monkeypatch.setattr(moe, "_compute_routing_weights", routed)
    y, _ = moe(x.to(gpu))
    y.backward(dy.to(gpu))
    (logits, weights, selected), outputs = routing[0], kept[1]
    assert len(kept) == 2 and outputs.shape == (T, k, H)

    u = torch.finfo(dtype).eps / 2
    terms = kept64(outputs) * dy.double().unsqueeze(1)
    d = terms.sum(-1)
    evaluation = (8 * -(-H // 512) + 8) * 2.0 ** -24
    assert_rounded(weights.grad, d, dtype, evaluation, terms.abs().sum(-1), "d_gates")

    g = torch.softmax(logits.double().gather(1, selected), dim=-1)
    inner = (g * d).sum(-1, keepdim=True)
    size = g * (d.abs() + (g * d.abs()).sum(-1, keepdim=True))
    exact = g * (d - inner)
    lost = g * evaluation * (terms.abs().sum(-1) + (g * terms.abs().sum(-1)).sum(-1, keepdim=True))
    off = u * size + u * exact.abs() + 2.0 ** -20 * size + lost
    if dtype == torch.float16:
        off = off + 2.0 ** -25 * (1 + 2 * g)  # half of fp16's smallest step, for d_gates and for d_logits
    rows = lambda values: torch.zeros(T, E, dtype=torch.float64).scatter_(1, selected, values)
    x64 = x.double()
    want = rows(exact).t() @ x64
    allowed = rows(off).t() @ x64.abs() + u * want.abs() + 2.0 ** -16 * (rows(exact).abs().t() @ x64.abs())
    error = (moe.gate.weight.grad.cpu().double() - want).abs()
    assert (error <= allowed).all(), float((error / allowed).max())
    # (tight enough to see a routing gradient that is missing or another token's)
    assert (allowed.norm() < 0.2 * want.norm()) and (want.norm() > 0)

"""Further GPU test bodies of the 8-bit checkpoints, the balance loss and the operators they share code with, on the CPU
emulation of the kernels."""

import inspect

import pytest
import torch

import test_gpu_layer_balance as layer_balance
import test_gpu_layer_edges as edges
import test_gpu_mx8_routing as routing
import test_gpu_mx8_scales as small_scales
import test_gpu_second_derivatives as second
import test_gpu_swiglu_far_gates as far_gates
from test_emulated_device import emulated, library  # noqa: F401 (fixtures)

CASES = []


def case(function, **arguments):
    label = function.__name__[5:] + "-" + "-".join(str(v).replace("torch.", "") for v in arguments.values())
    CASES.append(pytest.param(function, arguments, id=label[:90]))


for checkpoint_8bit in (False, True):
    for one_tensor in (False, True):
        case(far_gates.test_far_gates_fp32, checkpoint_8bit=checkpoint_8bit, one_tensor=one_tensor)
for experts, top_k in [(8, 2), (12, 1), (40, 6), (100, 70), (66, 65)]:
    for fuse_router in (True, False):
        case(layer_balance.test_counts_are_those_of_the_routing, experts=experts, top_k=top_k, fuse_router=fuse_router)
case(layer_balance.test_one_token_and_one_expert_of_any_stride)
for name in ("rmsnorm", "residual", "residual-both", "swiglu", "unchunked", "balance", "z-loss"):
    for path in ("python", "traced"):
        case(second.test_operators, name=name, path=path)
case(second.test_layer)
for dtype in (torch.float32, torch.float16, torch.bfloat16):
    for width in (32, 35):
        case(small_scales.test_all_scale_bytes, dtype=dtype, width=width)
case(small_scales.test_products_of_small_blocks)
for dtype in (torch.float32, torch.float16, torch.bfloat16):
    case(routing.test_routing_gradients, dtype=dtype, shape=(100, 64, 128, 4, 2))
case(routing.test_routing_gradients, dtype=torch.bfloat16, shape=(96, 72, 40, 5, 3))
for dtype in (torch.float32, torch.bfloat16):
    for checkpoint_8bit in (False, True):
        case(edges.test_no_tokens, dtype=dtype, checkpoint_8bit=checkpoint_8bit)
case(edges.test_refusals_are_those_of_the_ordinary_call)


@pytest.mark.parametrize("function,arguments", CASES)
def test_gpu_test_body_on_the_emulated_device(emulated, monkeypatch, function, arguments):  # noqa: F811
    if "monkeypatch" in inspect.signature(function).parameters:
        arguments = dict(arguments, monkeypatch=monkeypatch)
    function(emulated, **arguments)

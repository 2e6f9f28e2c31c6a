"""Gradients that the kernels compute say nothing about how they depend on what they came from.  Differentiating through the
8-bit checkpoints' and the balance loss's is an error wherever they run - the compiled host path, the Python autograd functions, the
layer -, also where the rest of a sum could be differentiated."""

import pytest
import torch

from helpers import announce, randn

pytestmark = pytest.mark.gpu

MESSAGE = "no derivative of its own"


def _calls(gpu):
    import cute_kernels as ck

    res, w = randn((5, 64), torch.float32, 61).to(gpu), randn((64,), torch.float32, 62).to(gpu)
    ids = torch.tensor([[0], [1], [2], [3], [4]], device=gpu)
    return {
        "rmsnorm": lambda v: ck.rmsnorm_cute(v, w, 1e-5, checkpoint_8bit=True).square().sum(),
        "residual": lambda v: ck.fused_residual_add_rmsnorm_cute(v, res, None, 1e-5, checkpoint_8bit=True)[0].square().sum(),
        "residual-both": lambda v: sum(t.square().sum() for t in
                                       ck.fused_residual_add_rmsnorm_cute(res, v, w, 1e-5, checkpoint_8bit=True)),
        "swiglu": lambda v: ck.swiglu_cute(v, res, checkpoint_8bit=True).square().sum(),
        "unchunked": lambda v: ck.swiglu_unchunked_cute(v, checkpoint_8bit=True).square().sum(),
        "balance": lambda v: ck.moe_balance_loss_cute(v, ids)[0].square(),
        "z-loss": lambda v: ck.moe_balance_loss_cute(v, ids)[1].square(),
    }


def _check(call, leaf):
    """The first derivative with and without a graph alike; the second an error, alone and beside a term
    that has one, by grad and by backward."""
    def fresh():
        return leaf.detach().clone().requires_grad_(True)

    v = fresh()
    (first,) = torch.autograd.grad(call(v), v)
    (again,) = torch.autograd.grad(call(v), v, create_graph=True)
    assert torch.equal(first, again.detach()) and again.requires_grad
    for loss in (lambda g, v: g.square().sum(), lambda g, v: (g.square() + v.pow(3)).sum()):
        v = fresh()
        (g,) = torch.autograd.grad(call(v), v, create_graph=True)
        with pytest.raises(RuntimeError, match=MESSAGE):
            torch.autograd.grad(loss(g, v), v)
        v = fresh()
        (g,) = torch.autograd.grad(call(v), v, create_graph=True)
        with pytest.raises(RuntimeError, match=MESSAGE):
            loss(g, v).backward()


@pytest.mark.parametrize("path", ["eager", "python", "traced"])
@pytest.mark.parametrize("name", ["rmsnorm", "residual", "residual-both", "swiglu", "unchunked", "balance", "z-loss"])
def test_operators(gpu, name, path, monkeypatch):
    from cute_kernels import _native
    from cute_kernels.utils import set_cute_tracing

    announce("second derivative", name, path)
    if path == "python":
        monkeypatch.setattr(_native, "functions_for", lambda tensor: None)
    set_cute_tracing(path == "traced")
    try:
        _check(_calls(gpu)[name], randn((5, 64), torch.float32, 60).to(gpu))
    finally:
        set_cute_tracing(False)


def test_layer(gpu):
    import cute_kernels as ck

    announce("second derivative of the layer")
    moe = ck.MoE_HIP(num_experts=4, num_experts_per_tok=2, hidden_size=64, intermediate_size=128,
                     activation_function=ck.swiglu_unchunked_cute, is_glu=True, add_bias=False, std=0.05)
    with torch.no_grad():
        for i, p in enumerate(moe.parameters()):
            p.copy_(randn(p.shape, torch.float32, 90 + i, 0.1))
    moe = moe.to(device=gpu, dtype=torch.bfloat16)
    moe.checkpoint_8bit = True
    x = randn((20, 64), torch.bfloat16, 95).to(gpu)
    _check(lambda v: moe(v)[0].float().square().sum(), x)
    # through a weight of the experts
    for weight in (moe.c_fc.weight, moe.c_proj.weight):
        (g,) = torch.autograd.grad(moe(x)[0].float().square().sum(), weight, create_graph=True)
        with pytest.raises(RuntimeError, match=MESSAGE):
            torch.autograd.grad((g.float().square() + weight.float().pow(3)).sum(), weight)

"""``MoE_HIP.balance_loss`` counts the experts that the layer's forward sent its tokens to, whichever selection it routes by."""

import pytest
import torch

from helpers import announce, randn
from test_gpu_moe_balance import reference

pytestmark = pytest.mark.gpu


def _layer(gpu, E, k, dtype, H=64):
    import cute_kernels as ck

    moe = ck.MoE_HIP(num_experts=E, num_experts_per_tok=k, hidden_size=H, intermediate_size=64,
                     activation_function=ck.swiglu_unchunked_cute, is_glu=True, add_bias=False, std=0.05)
    with torch.no_grad():
        for i, p in enumerate(moe.parameters()):
            p.copy_(randn(p.shape, torch.float32, 70 + i, 0.1))
        # few distinct whole numbers as logits: equal ones on every row, at the border of the selection too
        moe.gate.weight.zero_()
        moe.gate.weight[:, 0] = torch.arange(E).remainder(3).float()
        moe.gate.weight[:, 1] = torch.arange(E).remainder(2).float()
    return moe.to(device=gpu, dtype=dtype)


# (experts, top_k): the last two are beyond the selection kernel
@pytest.mark.parametrize("fuse_router", [True, False])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (12, 1), (40, 6), (100, 70), (66, 65)])
def test_counts_are_those_of_the_routing(gpu, experts, top_k, fuse_router, monkeypatch):
    announce("layer balance", experts, top_k, fuse_router)
    dtype = torch.bfloat16
    moe = _layer(gpu, experts, top_k, dtype)
    moe.fuse_router = fuse_router
    routed = []
    inner = moe._compute_experts
    monkeypatch.setattr(moe, "_compute_experts",
                        lambda rows, weights, selected: routed.append(selected) or inner(rows, weights, selected))
    x = randn((3, 40, 64), torch.float32, 75).sign().to(dtype).to(gpu).requires_grad_(True)
    mask = torch.ones(3, 40, dtype=torch.bool, device=gpu)
    mask[2, 17:] = False
    _, router_logits = moe(x)
    want = reference(router_logits.detach().cpu(), routed[0].cpu(), mask.view(-1).cpu(), 1.0, 0.0)
    assert (torch.topk(router_logits.detach().float(), min(top_k + 1, experts)).values.diff(dim=-1)[:, -1] == 0).any()
    for call in [lambda: moe.balance_loss(router_logits, mask),
                 lambda: moe.balance_loss(router_logits, mask, selected_experts=routed[0]),
                 lambda: moe.balance_loss(router_logits.view(3, 40, experts), mask, routed[0].view(3, 40, top_k))]:
        balance, z, counts = call()
        assert torch.equal(counts.cpu().long(), want[2])
        assert abs(float(balance.detach()) - float(want[0])) <= 2.0 ** -19 * float(want[0])
        (d,) = torch.autograd.grad(balance, router_logits, retain_graph=True)
        error = (d.cpu().double() - want[3]).abs()
        assert (error <= 2.0 ** -8 * want[3].abs() + 2.0 ** -18 * want[4]).all()  # (bf16 rounding, and the fp32 evaluation)


def test_one_token_and_one_expert_of_any_stride(gpu):
    """Along a dimension of one element a tensor's stride can be any number; the selection takes it as the losses do."""
    from cute_kernels import moe_balance_loss_cute

    announce("balance strides of one")
    wide = randn((20, 8), torch.float32, 80)
    views = [
        (lambda t: t[:1, :5].t(), 1),  # five tokens, one expert, the next column a row away
        (lambda t: t[:1].expand(20, 8)[:1], 2),  # one token of an expanded row: stride 0
        (lambda t: t[0].view(8, 1).t(), 2),  # one token, stride 1
        (lambda t: t[3:4, 2:3], 1),
        (lambda t: t[:, 1:2], 1),
        (lambda t: t[7], 2),
    ]
    for view, top_k in views:
        z = wide.to(gpu, copy=True).requires_grad_(True)
        logits = view(z)
        host = view(wide).reshape(-1, logits.size(-1))
        ids = host.topk(top_k, dim=-1).indices
        want = reference(host, ids, None, 1.0, 1.0)
        balance, z_loss, counts = moe_balance_loss_cute(logits, top_k=top_k)
        assert torch.equal(counts.cpu().long(), want[2])
        assert abs(float(balance.detach()) - float(want[0])) <= 2.0 ** -19 * float(want[0])
        (d,) = torch.autograd.grad(balance + z_loss, logits)
        error = (d.cpu().double().reshape(want[3].shape) - want[3]).abs()
        assert (error <= 2.0 ** -23 * want[3].abs() + 2.0 ** -18 * want[4]).all()

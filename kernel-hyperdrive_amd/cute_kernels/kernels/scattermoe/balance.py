"""Balance loss, z-loss and per-expert counts of an MoE router.

The layer returns its router logits (cute_kernels/kernels/scattermoe/torch_implementation.py:10-199) so that the caller can
put an auxiliary loss on them; the reference has none.  With ``p`` the softmax over the E experts, ``lse`` the log-sum-exp of
the logits, N counting tokens and c_e the selections of expert e by them::

    balance = E * sum_e c_e / (N k) * mean_t p_te            (1 when the load is even)
    z       = mean_t lse_t ** 2

Gradients reach the logits through p and lse; the counts are whole numbers and have none.
"""

import torch

from ... import _C, _native
from ...constants import LIBRARY_NAME
from ...utils import cute_op


def moe_balance_loss_torch(
    router_logits: torch.Tensor, selected_experts: torch.Tensor, token_mask: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    E, k = router_logits.size(-1), selected_experts.size(-1)
    logits = router_logits.reshape(-1, E).float()
    selected = selected_experts.reshape(-1, k)
    if token_mask is not None:
        keep = token_mask.reshape(-1)
        logits, selected = logits[keep], selected[keep]
    n = max(1, logits.size(0))
    valid = selected[(selected >= 0) & (selected < E)]
    counts = torch.bincount(valid, minlength=E).to(torch.int32)
    dead = (logits <= torch.finfo(router_logits.dtype).min).all(dim=-1)
    alive = logits[~dead]
    balance = E * (counts / (n * k) * alive.softmax(dim=-1).sum(dim=0) / n).sum()
    return balance, alive.logsumexp(dim=-1).square().sum() / n, counts


@cute_op(f"{LIBRARY_NAME}::moe_balance_loss_forward_hip", mutates_args={"balance", "z", "counts", "shares"})
def moe_balance_loss_forward_hip(
    logits: torch.Tensor,
    selected: torch.Tensor,
    mask: torch.Tensor | None,
    balance: torch.Tensor,
    z: torch.Tensor,
    counts: torch.Tensor,
    shares: torch.Tensor,
) -> None:
    nbytes = _C.moe_balance_loss_workspace_size(logits.size(0), logits.size(1))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes > 0 else None
    _C.moe_balance_loss_forward(logits, selected, mask, balance, z, counts, shares, workspace)


@cute_op(f"{LIBRARY_NAME}::moe_balance_loss_backward_hip", mutates_args={"d_logits"})
def moe_balance_loss_backward_hip(
    logits: torch.Tensor,
    mask: torch.Tensor | None,
    shares: torch.Tensor,
    balance_grad: torch.Tensor | None,
    z_grad: torch.Tensor | None,
    d_logits: torch.Tensor,
) -> None:
    _C.moe_balance_loss_backward(logits, mask, shares, balance_grad, z_grad, d_logits)


class _MoEBalanceLoss_Cute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, selected, mask):
        device = logits.device
        balance = torch.empty((), dtype=torch.float32, device=device)
        z = torch.empty((), dtype=torch.float32, device=device)
        counts = torch.empty(logits.size(1), dtype=torch.int32, device=device)
        shares = torch.empty(logits.size(1) + 1, dtype=torch.float32, device=device)
        moe_balance_loss_forward_hip(logits, selected, mask, balance, z, counts, shares)
        ctx.save_for_backward(logits, mask, shares)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return balance, z, counts

    @staticmethod
    def backward(ctx, balance_grad, z_grad, _counts_grad):
        logits, mask, shares = ctx.saved_tensors
        if balance_grad is None and z_grad is None:
            return None, None, None
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        moe_balance_loss_backward_hip(logits, mask, shares, balance_grad, z_grad, d_logits)
        return _native.not_differentiable(d_logits, None, None)


def moe_balance_loss_cute(
    router_logits: torch.Tensor,
    selected_experts: torch.Tensor | None = None,
    token_mask: torch.Tensor | None = None,
    top_k: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(balance, z, expert_counts)`` - two float32 scalars and int32 ``[E]`` - of ``router_logits [..., E]`` (float32,
    float16 or bfloat16, E <= 1024).

    ``selected_experts [..., k]``: the experts each token went to (an id outside [0, E), a dropped slot, counts nowhere); None:
    the ``top_k`` (at most 64) largest logits, equal ones in the order of their positions, as the layer's router selects them.
    ``token_mask [...]`` bool: False for padding, which takes no part whatever its logits and ids hold.  Without a counting
    token both losses are 0.  A token whose logits are all -inf or the type's lowest value has no probabilities and no
    log-sum-exp: it counts in N, and its selections in the counts."""
    E = router_logits.size(-1)
    logits = router_logits if router_logits.dim() == 2 else router_logits.reshape(-1, E)
    if (E > 1 and logits.stride(1) != 1) or (logits.size(0) > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    if selected_experts is None:
        if top_k is None:
            raise ValueError("moe_balance_loss_cute: selected_experts or top_k")
        from .moe_hip import router_topk_softmax_forward_hip  # (moe_hip's layer has this function as a method)

        selected_experts = router_topk_softmax_forward_hip(logits.detach(), top_k)[2]
    else:
        if selected_experts.shape[:-1] != router_logits.shape[:-1]:
            raise ValueError(
                f"moe_balance_loss_cute: selected_experts {tuple(selected_experts.shape)} do not go with logits "
                f"{tuple(router_logits.shape)}"
            )
        if top_k is not None and selected_experts.size(-1) != top_k:
            raise ValueError("moe_balance_loss_cute: top_k is not the number of selected experts")
        selected_experts = _C._index_i64(selected_experts, "selected_experts")
        if selected_experts.dim() != 2:
            selected_experts = selected_experts.view(-1, selected_experts.size(-1))
    if token_mask is not None:
        if token_mask.dtype != torch.bool or token_mask.shape != router_logits.shape[:-1]:
            raise ValueError("moe_balance_loss_cute: token_mask is one bool per token")
        token_mask = token_mask.reshape(-1).contiguous()
    functions = _native.functions_for(logits)
    if functions is None:
        return _MoEBalanceLoss_Cute.apply(logits, selected_experts, token_mask)
    return functions.moe_balance_loss(logits, selected_experts, token_mask)

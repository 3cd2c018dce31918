"""Routing to experts from logits (``csrc/route.cu``), with the gradient of the logits.

The reference's router (rwkv_mlx/moe.py:51-86) takes the softmax over the selected logits of at
most 32 experts and is served by :func:`rwkv_mlx_b200.moe.router_forward`.  :func:`route_experts`
is the form that larger expert layers are trained with: sigmoid or softmax scores, a bias that
balances the load and enters the selection only, selection limited to the best groups of experts,
and weights that are renormalised over the selection or not.  It has no counterpart in the
reference.
"""

from __future__ import annotations

import torch

from . import _native as nat

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 512, 32, 32


def _forward(logits, top_k, sigmoid, bias, n_groups, topk_groups, top2, renormalize, scale, want_counts):
    n, E = logits.shape
    dev = logits.device
    shape, pitch = (n, top_k), (top_k, 1)  # (empty_strided costs less than empty on the host)
    inds = torch.empty_strided(shape, pitch, dtype=torch.int32, device=dev)
    weights = torch.empty_strided(shape, pitch, dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev) if want_counts else None
    L = nat.lib()
    with nat.on_device(dev):
        rc = L.rwkv_route_experts(nat.ptr(logits), nat.row_stride(logits), nat.ptr(bias), nat.ptr(inds),
                                  nat.ptr(weights), nat.ptr(counts), n, E, top_k, n_groups, topk_groups, top2, sigmoid,
                                  renormalize, scale, nat.dtype_code(logits), nat.stream_ptr(dev))
    nat.check(rc, "rwkv_route_experts")
    return inds, weights, counts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, sigmoid, bias, n_groups, topk_groups, top2, renormalize, scale, want_counts):
        inds, weights, counts = _forward(logits, top_k, sigmoid, bias, n_groups, topk_groups, top2, renormalize, scale,
                                         want_counts)
        ctx.save_for_backward(logits, inds, weights)
        ctx.opts = (sigmoid, renormalize, scale)
        ctx.mark_non_differentiable(inds, *([] if counts is None else [counts]))
        ctx.set_materialize_grads(False)  # no zero tensors for the integer outputs
        return inds, weights, counts

    @staticmethod
    @nat.first_order
    def backward(ctx, _dinds, dweights, _dcounts=None):
        if dweights is None:
            return (None,) * 10
        logits, inds, weights = ctx.saved_tensors
        sigmoid, renormalize, scale = ctx.opts
        n, E = logits.shape
        dev = logits.device
        dlogits = torch.empty((n, E), device=dev, dtype=logits.dtype)
        dw = dweights.to(torch.float32).contiguous()
        L = nat.lib()
        with nat.on_device(dev):
            rc = L.rwkv_route_experts_backward(nat.ptr(logits), nat.row_stride(logits), nat.ptr(inds), nat.ptr(weights),
                                               nat.ptr(dw), nat.ptr(dlogits), n, E, inds.shape[1], sigmoid, renormalize,
                                               scale, nat.dtype_code(logits), nat.stream_ptr(dev))
        nat.check(rc, "rwkv_route_experts_backward")
        return (dlogits,) + (None,) * 9


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  n_groups: int = 1, topk_groups: int = 1, group_score: str = "top2", renormalize: bool = True,
                  scale: float = 1.0, return_counts: bool = False):
    """Choose ``top_k`` experts for each row of ``logits`` (..., E), fp32 / fp16 / bf16.

    Scores s are ``softmax(logits)`` or ``sigmoid(logits)`` in fp32.  Experts are compared by
    s + ``bias`` ((E,) fp32, no gradient; softmax without a bias compares the logits, which have the
    same order), after all but the ``topk_groups`` best of ``n_groups`` equal runs of experts are left
    out; a run counts by its largest key (``group_score="max"``) or the sum of its two largest
    (``"top2"``).  Ties go to the lower index.

    Returns ``(inds, weights)`` or ``(inds, weights, counts)``: int32 (..., top_k) in descending order
    of the key, fp32 ``scale * s / sum of the selected s`` (``scale * s`` without ``renormalize``), and
    int32 (E,) rows given to each expert.  A row whose selected scores sum to 0 (all logits -inf) has
    weights 0; a NaN logit ranks first and its weight is NaN.  Differentiable in ``logits``.
    """
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"route_experts: score must be 'softmax' or 'sigmoid', not {score!r}")
    if group_score not in ("top2", "max"):
        raise ValueError(f"route_experts: group_score must be 'top2' or 'max', not {group_score!r}")
    E = logits.shape[-1]
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"route_experts: 1 to {MAX_EXPERTS} experts, not {E}")
    if not 1 <= n_groups <= MAX_GROUPS or E % n_groups or not 1 <= topk_groups <= n_groups:
        raise ValueError(f"route_experts: {n_groups} groups of which {topk_groups} stay do not fit {E} experts "
                         f"(at most {MAX_GROUPS} equal groups)")
    if not 1 <= top_k <= min(MAX_TOP_K, topk_groups * (E // n_groups)):
        raise ValueError(f"route_experts: top_k must be 1 to {min(MAX_TOP_K, topk_groups * (E // n_groups))} here, not {top_k}")
    if bias is not None:
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError("route_experts: bias must be (E,) on the logits' device")
        bias = bias.detach().to(torch.float32).contiguous()
    nat.dtype_code(logits)
    lead = logits.shape[:-1]
    l2 = nat.rows_2d(logits)
    args = (l2, int(top_k), int(score == "sigmoid"), bias, int(n_groups), int(topk_groups), int(group_score == "top2"),
            int(bool(renormalize)), float(scale), bool(return_counts))
    if logits.requires_grad and torch.is_grad_enabled():
        inds, weights, counts = _Route.apply(*args)
    else:
        inds, weights, counts = _forward(*args)
    if len(lead) != 1:
        inds, weights = inds.view(*lead, top_k), weights.view(*lead, top_k)
    return (inds, weights, counts) if return_counts else (inds, weights)


def update_balance_bias(bias: torch.Tensor, counts: torch.Tensor, rate: float) -> torch.Tensor:
    """Move each expert's bias by ``rate`` towards an even load, in place: up where ``counts`` is
    below the mean, down where it is above.  Run once a step, outside autograd."""
    with torch.no_grad():
        c = counts.to(torch.float32)
        return bias.add_(torch.sign(c.mean() - c).to(bias.dtype), alpha=rate)

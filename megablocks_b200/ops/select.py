"""Expert selection: scores, a balancing bias, expert groups, top-k and renormalised weights.

With ``s`` the softmax or sigmoid of a token's logits over the experts and ``c = s + bias``

* a group (``experts / groups`` consecutive experts) is worth the sum of its two largest ``c``, and the best
  ``top_groups`` groups stay;
* the ``top_k`` largest ``c`` of those groups are chosen, in descending order;
* their weights are ``scale * s / ||s_chosen||_p`` (``norm_p`` 1 or 2), or ``scale * s`` without ``norm_p``;
* ``scores = s / sum(s)``, a distribution over the experts, is what a load-balancing loss takes.

Equal values go to the lowest id, of experts and of groups.  The order is that of the exact values: closer
pairs than fp32 tells apart are compared in 64 bits, and without a bias the logits are compared, whose order
the scores have.  The bias has a part in the choice only: no gradient reaches it, and the weights are those
of the unbiased scores.  It is moved by :func:`update_expert_bias`, against the load, so that a layer is
balanced without an auxiliary loss.

A bias of -inf takes an expert out, one of +inf puts it before all others; a group with both as its largest is
worth +inf, and one with a single expert that is not taken out -inf.

A token whose logits hold NaN (softmax: or +inf) gets distinct valid ids and NaN weights.  An expert with
a logit of -inf has score 0; where every chosen score is 0, so are the weights.

On CUDA the forward and the backward pass are one kernel each (``csrc/select_experts.cu``); forward-mode tangents
and functional transforms take PyTorch ops.
"""

import math
from typing import Optional, Tuple

import torch

from megablocks_b200._ext import ext, transformed

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 32, 32
_SCORES = ('softmax', 'sigmoid')
_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(logits, top_k, bias, groups, top_groups):
    if logits.dim() != 2 or logits.dtype not in (torch.float16, torch.bfloat16, torch.float32, torch.float64):
        raise ValueError('select_experts expects floating-point logits[tokens, experts]')
    experts = logits.shape[1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f'select_experts takes 1 to {MAX_EXPERTS} experts, got {experts}')
    if not 1 <= groups <= MAX_GROUPS or experts % groups:
        raise ValueError(f'groups must divide the {experts} experts and be at most {MAX_GROUPS}, got {groups}')
    if not 1 <= top_groups <= groups:
        raise ValueError(f'top_groups must lie in [1, {groups}], got {top_groups}')
    if not 1 <= top_k <= min(MAX_TOP_K, top_groups * (experts // groups)):
        raise ValueError(f'top_k must lie in [1, {min(MAX_TOP_K, top_groups * (experts // groups))}] (at most '
                         f'{MAX_TOP_K}, and what the chosen groups hold), got {top_k}')
    if bias is not None and (bias.shape != (experts,) or bias.dtype != torch.float32 or bias.device != logits.device):
        raise ValueError('bias must be a float32 vector with one entry per expert, on the device of the logits')


def select_experts(logits: torch.Tensor, top_k: int, *, score: str = 'softmax', bias: Optional[torch.Tensor] = None,
                   groups: int = 1, top_groups: Optional[int] = None, norm_p: Optional[int] = None,
                   scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(scores[tokens, experts], weights[tokens, top_k], experts[tokens, top_k])`` of ``logits[tokens, experts]``.

    Scores and weights have the type of the logits, the ids are int64.  ``bias`` is fp32; ``top_groups`` is by
    default all of them.  Up to 1024 experts, 32 groups and ``top_k`` 32."""
    top_groups = groups if top_groups is None else top_groups
    if score not in _SCORES:
        raise ValueError(f'score must be one of {_SCORES}, got {score!r}')
    if norm_p not in (None, 0, 1, 2):
        raise ValueError(f'norm_p must be None, 1 or 2, got {norm_p!r}')
    norm_p = int(norm_p or 0)
    if logits.is_cuda and logits.dtype in _KERNEL_DTYPES and not transformed(logits):
        return tuple(ext().select_experts(logits, top_k, score == 'sigmoid', bias, groups, top_groups, norm_p, scale))
    _check(logits, top_k, bias, groups, top_groups)
    return _composed(logits, top_k, score, None if bias is None else bias.detach(), groups, top_groups, norm_p, scale)


def _scores(x: torch.Tensor, score: str) -> torch.Tensor:
    if score == 'sigmoid':
        return torch.sigmoid(x)
    top = x.amax(dim=-1, keepdim=True).detach()
    e = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(dim=-1, keepdim=True)
    return e / total.masked_fill(total == 0, 1.0)


def _composed(logits, top_k, score, bias, groups, top_groups, norm_p, scale):
    """The same from PyTorch ops."""
    with torch.no_grad():
        wide = logits.detach().double()
        order = wide
        if bias is not None or top_groups < groups:
            choice = _scores(wide, score)
            if bias is not None:
                choice = order = choice + bias.double()
            choice = choice.masked_fill(choice.isnan(), math.inf)
        order = order.masked_fill(order.isnan(), math.inf)
        out = torch.zeros_like(order, dtype=torch.bool)
        if top_groups < groups:
            size = logits.shape[1] // groups
            value = choice.view(-1, groups, size).topk(min(2, size), dim=-1).values.sum(dim=-1)
            value = value.masked_fill(value.isnan(), math.inf)
            kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
            out = torch.ones_like(value, dtype=torch.bool).scatter_(1, kept, False).repeat_interleave(size, dim=1)
        # Experts of other groups behind all others, also behind those that are worth -inf.
        ranked = order.sort(dim=-1, descending=True, stable=True).indices
        ranked = ranked.gather(1, out.gather(1, ranked).to(torch.int8).sort(dim=-1, stable=True).indices)
        experts = ranked[:, :top_k].contiguous()
    wide = logits if logits.dtype == torch.float64 else logits.float()
    s = _scores(wide, score)
    weights = s.gather(1, experts)
    if norm_p:
        norm = torch.linalg.vector_norm(weights, ord=norm_p, dim=-1, keepdim=True)
        weights = weights / norm.masked_fill(norm == 0, math.inf)
    weights = weights * scale
    total = s.sum(dim=-1, keepdim=True)
    scores = s if score == 'softmax' else s / total.masked_fill(total == 0, math.inf)
    return scores.to(logits.dtype), weights.to(logits.dtype), experts


@torch.no_grad()
def update_expert_bias(bias: torch.Tensor, load: torch.Tensor, rate: float) -> torch.Tensor:
    """``bias += rate * sign(mean(load) - load)`` in place: experts with less than the mean load get a larger
    bias, those with more a smaller one.  ``load[experts]``: tokens per expert since the last update."""
    if bias.shape != load.shape or bias.dim() != 1:
        raise ValueError('bias and load must be vectors with one entry per expert')
    # sum(load) - experts * load keeps whole numbers whole: no expert at the mean moves by a rounding.
    load = load.to(torch.float64)
    return bias.add_(torch.sign(load.sum() - load.numel() * load).to(bias.dtype), alpha=rate)

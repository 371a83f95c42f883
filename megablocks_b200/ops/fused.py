"""Fused row-wise ops for the transformer around the MoE layers.

* :func:`cross_entropy` - mean softmax cross-entropy over ``[rows, vocab]`` logits.
  On CUDA the forward reads the 16-bit logits once (no fp32 copy) and the backward
  overwrites the logits buffer with the gradient in place, so a 3.3 GB logits tensor
  costs three passes instead of the dozen of the eager float() / log_softmax /
  nll_loss chain.  The logits tensor must not be used after the loss (it is the
  gradient afterwards).
* :func:`distillation_loss` / :func:`linear_distillation_loss` - distillation from a teacher's top logits
  (optionally mixed with the targets' cross entropy), loss and gradient in one pass over the student's logits.
* :func:`layer_norm` - LayerNorm whose backward reduces the weight and bias
  gradients through shared memory in the same pass that produces ``dx``.

* :func:`rms_norm` / :class:`RMSNorm` - the same kernels without centring and bias (Mixtral-style
  models), including the fused residual add.
* :func:`rope` - rotary position embedding of ``[batch, heads, seq, head_dim]`` queries / keys in
  one pass (rotation of the pairs ``(i, i + d/2)`` in fp32, no fp32 copies of the tensor).
* :func:`load_balancing_loss` - the auxiliary loss of all layers in one reduction kernel and its
  gradient in one broadcast kernel.

* :func:`linear` / :class:`Linear` - ``nn.Linear`` whose bias gradient is one column-sum kernel
  at memory bandwidth (the library route reduces the same tensor at a third of that).

All fall back to the PyTorch ops on CPU tensors.
"""

import math
import os
from typing import Any

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from megablocks_b200._ext import ext, transformed


class _CrossEntropy(torch.autograd.Function):

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, targets: torch.Tensor):
        loss, lse = ext().cross_entropy_forward(logits, targets)
        ctx.save_for_backward(logits, targets, lse)
        return loss.mean()

    @staticmethod
    def backward(ctx: Any, grad_out: torch.Tensor):
        logits, targets, lse = ctx.saved_tensors
        scale = grad_out.detach().float().reshape(1)
        ext().cross_entropy_backward_(logits, targets, lse, scale, 1.0 / logits.shape[0])
        return logits, None


class _LinearCrossEntropy(torch.autograd.Function):
    """``mean(cross_entropy(hidden @ weight^T, targets))`` with the loss and the gradient of the logits
    taken in ONE pass over the logits (they are overwritten with ``(softmax - onehot) / rows``).  The
    incoming gradient, a scalar, is then applied to the two small products of the backward pass
    instead of to the logits."""

    @staticmethod
    def forward(ctx: Any, hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor):
        logits = hidden @ weight.t()
        loss = ext().cross_entropy_fused_(logits, targets, 1.0 / logits.shape[0])
        ctx.save_for_backward(hidden, weight, logits)
        return loss.mean()

    @staticmethod
    def backward(ctx: Any, grad_out: torch.Tensor):
        hidden, weight, dlogits = ctx.saved_tensors
        scale = grad_out.detach().float()       # a 0-dim fp32 tensor: multiplies in fp32, result in the tensor's type
        dh = dw = None
        if ctx.needs_input_grad[0]:
            dh = (dlogits @ weight).mul_(scale)
        if ctx.needs_input_grad[1]:
            dw = (dlogits.t() @ hidden).mul_(scale)
        return dh, dw, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Mean cross entropy of ``hidden[rows, h] @ weight[vocab, h]^T`` against ``targets[rows]``: the
    language-model head and its loss.  On CUDA the logits are written once and read once."""
    # Not for fp16: there the loss scale has to reach the logit gradient before it is rounded (the
    # unscaled (softmax - onehot) / rows underflows), and the scale is only known in backward.
    if (hidden.is_cuda and hidden.dtype in (torch.bfloat16, torch.float32) and hidden.dim() == 2
            and weight.dtype == hidden.dtype and not torch.is_autocast_enabled()
            and os.environ.get('MB200_FUSED_LM_LOSS', '1') != '0'):
        return _LinearCrossEntropy.apply(hidden.contiguous(), weight, targets.contiguous())
    return cross_entropy(F.linear(hidden, weight), targets)


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Mean cross entropy of ``logits[rows, vocab]`` against ``targets[rows]`` (int64)."""
    if logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float16, torch.float32) and logits.is_contiguous():
        return _CrossEntropy.apply(logits, targets.contiguous())
    return F.cross_entropy(logits.float(), targets)


class _LinearDistillation(torch.autograd.Function):
    """The language-model head and the loss: the gradient of the logits over the logits, as in
    :class:`_LinearCrossEntropy`."""

    @staticmethod
    def forward(ctx: Any, hidden, weight, values, ids, targets, temperature, hard_weight):
        logits = hidden @ weight.t()
        loss, dlogits = ext().distill_in_place(logits, values, ids, targets, temperature, hard_weight)
        ctx.save_for_backward(hidden, weight, dlogits)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_out: torch.Tensor):
        hidden, weight, dlogits = ctx.saved_tensors
        scale = grad_out.detach().float()
        dh = (dlogits @ weight).mul_(scale) if ctx.needs_input_grad[0] else None
        dw = (dlogits.t() @ hidden).mul_(scale) if ctx.needs_input_grad[1] else None
        return dh, dw, None, None, None, None, None


MAX_TEACHER_TOP = 1024
_DISTILL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_distillation(rows, device, teacher_logits, teacher_ids, temperature, targets, hard_weight):
    if teacher_logits.dim() != 2 or teacher_logits.shape != teacher_ids.shape or teacher_logits.shape[0] != rows:
        raise ValueError('distillation expects the teacher\'s logits and ids as [rows, top], one row per row of logits')
    if not 1 <= teacher_logits.shape[1] <= MAX_TEACHER_TOP:
        raise ValueError(f'distillation takes 1 to {MAX_TEACHER_TOP} teacher logits a row')
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError('the teacher\'s ids must be int32 or int64')
    if teacher_logits.dtype not in (torch.float16, torch.bfloat16, torch.float32, torch.float64):
        raise ValueError('the teacher\'s logits must be floating-point')
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f'the temperature must be positive, got {temperature}')
    if not (math.isfinite(hard_weight) and hard_weight >= 0):
        raise ValueError(f'hard_weight must not be negative, got {hard_weight}')
    if hard_weight and targets is None:
        raise ValueError('hard_weight needs targets')
    if targets is not None and (targets.shape != (rows,) or targets.dtype != torch.int64):
        raise ValueError('targets must be int64 with one entry per row')
    if any(t is not None and t.device != device for t in (teacher_logits, teacher_ids, targets)):
        raise ValueError('the teacher\'s logits, its ids and the targets must be on the device of the logits')


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                      temperature: float = 1.0, targets=None, hard_weight: float = 0.0) -> torch.Tensor:
    """Mean over the rows of ``T^2 KL(p || q) + hard_weight * cross_entropy(logits, targets)``.

    ``q = softmax(logits[rows, vocab] / T)`` and ``p`` is the softmax of a row's ``teacher_logits[rows, top] / T``
    over the columns that ``teacher_ids[rows, top]`` (int32 or int64) names: the teacher's kept logits, taken as
    its whole distribution.  Ids outside the vocabulary mark unused slots, a column named twice counts twice;
    a row without a used slot has no such term, one whose target lies outside the vocabulary no cross
    entropy, and a row with neither has a gradient of zero, whatever its logits.  Every row counts in the mean.  A
    used slot of NaN makes the loss and the row's gradient NaN.
    The teacher gets no gradient; the logits stay as they are."""
    if (logits.is_cuda and logits.dtype in _DISTILL_DTYPES and teacher_logits.dtype != torch.float64
            and not transformed(logits)):
        return ext().distillation_loss(logits, teacher_logits, teacher_ids, targets, temperature, hard_weight)
    if logits.dim() != 2 or not logits.is_floating_point() or logits.shape[1] < 1:
        raise ValueError('distillation expects floating-point logits[rows, vocab]')
    _check_distillation(logits.shape[0], logits.device, teacher_logits, teacher_ids, temperature, targets, hard_weight)
    return _composed_distillation(logits, teacher_logits, teacher_ids, temperature, targets, hard_weight)


def _composed_distillation(logits, teacher_logits, teacher_ids, temperature, targets, hard_weight):
    """The same from PyTorch ops."""
    rows, vocab = logits.shape
    z = logits if logits.dtype == torch.float64 else logits.float()
    ids = teacher_ids.long()
    used = (ids >= 0) & (ids < vocab)
    def shifted(x):                                 # by the maximum, before a small temperature overflows
        top = x.detach().amax(dim=-1, keepdim=True)
        return (x - top.masked_fill(top == -math.inf, 0.0)) / temperature

    values = teacher_logits.detach().to(z.dtype).masked_fill(~used, -math.inf)
    used = used & (values != -math.inf)
    values = shifted(values)
    live = used.any(dim=-1)
    logp = values.masked_fill(~live.unsqueeze(1), 0.0).log_softmax(dim=-1).masked_fill(~used, 0.0)
    p = logp.exp() * used
    # Rows that teach nothing take no part at all, so that nothing of their logits reaches a gradient.
    hard = torch.zeros_like(live)
    if targets is not None and hard_weight:
        hard = (targets >= 0) & (targets < vocab)
    z = z.masked_fill(~(live | hard).unsqueeze(1), 0.0)
    logq = shifted(z).log_softmax(dim=-1).gather(1, ids.masked_fill(~used, 0))
    loss = temperature**2 * torch.where(p != 0, p * (logp - logq), 0.0).sum()         # p log p is 0 there
    if targets is not None and hard_weight:
        ce = -z.log_softmax(dim=-1).gather(1, targets.masked_fill(~hard, 0).unsqueeze(1)).squeeze(1)
        loss = loss + hard_weight * torch.where(hard, ce, 0.0).sum()
    return loss / max(rows, 1)


def linear_distillation_loss(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                             teacher_ids: torch.Tensor, temperature: float = 1.0, targets=None,
                             hard_weight: float = 0.0) -> torch.Tensor:
    """:func:`distillation_loss` of ``hidden[rows, h] @ weight[vocab, h]^T``: the language-model head and its loss.
    On CUDA the logits are written once, and once overwritten with their gradient."""
    if (hidden.is_cuda and hidden.dtype in (torch.bfloat16, torch.float32) and hidden.dim() == 2
            and weight.dtype == hidden.dtype and teacher_logits.dtype != torch.float64 and not transformed(hidden, weight)
            and not torch.is_autocast_enabled() and os.environ.get('MB200_FUSED_LM_LOSS', '1') != '0'):
        if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
            return _LinearDistillation.apply(hidden.contiguous(), weight, teacher_logits, teacher_ids, targets,
                                             temperature, hard_weight)
    return distillation_loss(F.linear(hidden, weight), teacher_logits, teacher_ids, temperature, targets, hard_weight)


class _LayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        y, mean, rstd, _ = ext().layernorm_forward(x2, weight, bias, eps, None, None)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.shape = shape
        return y.view(shape)

    @staticmethod
    def backward(ctx: Any, dy: torch.Tensor):
        x2, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = ext().layernorm_backward(dy.reshape(x2.shape).contiguous(), x2, weight, mean, rstd, None, False)
        return dx.view(ctx.shape), dw, db, None


class _AddLayerNorm(torch.autograd.Function):
    """``s = a + b [+ b_bias]; y = LayerNorm(s)`` in one pass; the backward adds ``ds`` while it writes
    ``dx``.  ``b_bias`` is a per-column vector that belongs to ``b`` (the output bias of the layer that
    produced it): its add rides in the forward kernel and its gradient is one column sum of ``dx``."""

    @staticmethod
    def forward(ctx: Any, a: torch.Tensor, b: torch.Tensor, b_bias, weight: torch.Tensor, bias: torch.Tensor,
                eps: float):
        shape = a.shape
        a2 = a.reshape(-1, shape[-1]).contiguous()
        b2 = b.reshape(-1, shape[-1]).contiguous()
        y, mean, rstd, s = ext().layernorm_forward(a2, weight, bias, eps, b2, b_bias)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.shape = shape
        ctx.bias_grad = b_bias is not None and ctx.needs_input_grad[2]
        return s.view(shape), y.view(shape)

    @staticmethod
    def backward(ctx: Any, ds, dy):
        s, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            d2 = ds.reshape(s.shape).contiguous()
            return ds, ds, (ext().column_sum(d2) if ctx.bias_grad else None), None, None, None
        dres = ds.reshape(s.shape).contiguous() if ds is not None else None
        dx, dw, db = ext().layernorm_backward(dy.reshape(s.shape).contiguous(), s, weight, mean, rstd, dres, False)
        dbias = ext().column_sum(dx) if ctx.bias_grad else None
        dx = dx.view(ctx.shape)
        return dx, dx, dbias, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    cols = x.shape[-1]
    fused = (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16, torch.float32) and weight.dtype == x.dtype
             and bias is not None and (cols * x.element_size()) % 16 == 0 and cols <= 6144)
    if fused:
        return _LayerNorm.apply(x, weight, bias, eps)
    return F.layer_norm(x, (cols,), weight, bias, eps)


def add_layer_norm(a: torch.Tensor, b, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5, b_bias=None):
    """``(a + b, LayerNorm(a + b))``; ``b`` may be ``None``.  On CUDA the add rides in the norm's kernels.

    ``b_bias`` (optional, one value per column) is added to ``b`` in the same pass."""
    if b is None:
        return a, layer_norm(a, weight, bias, eps)
    cols = a.shape[-1]
    if b_bias is not None and not (b_bias.is_cuda and b_bias.dtype == a.dtype and b_bias.numel() == cols):
        b, b_bias = b + b_bias, None
    fused = (a.is_cuda and b.is_cuda and a.dtype == b.dtype == weight.dtype and bias is not None
             and a.shape == b.shape and a.dtype in (torch.bfloat16, torch.float16, torch.float32)
             and ext().layernorm_can_fuse(a.reshape(-1, cols)))
    if fused:
        return _AddLayerNorm.apply(a, b, b_bias, weight, bias, eps)
    s = a + b if b_bias is None else a + b + b_bias
    return s, layer_norm(s, weight, bias, eps)


class LayerNorm(torch.nn.LayerNorm):
    """``nn.LayerNorm`` (same parameters and state dict) running the fused kernels on CUDA."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def add_forward(self, a: torch.Tensor, b, b_bias=None):
        """``(a + b [+ b_bias], self(...))`` with the adds fused into the kernels; ``b`` may be ``None``."""
        return add_layer_norm(a, b, self.weight, self.bias, self.eps, b_bias)


class _RMSNorm(torch.autograd.Function):
    """``y = x * rsqrt(mean(x^2) + eps) * weight`` on the LayerNorm kernels (no centring, no bias)."""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor, eps: float):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        y, mean, rstd, _ = ext().layernorm_forward(x2, weight, None, eps, None, None)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.shape = shape
        return y.view(shape)

    @staticmethod
    def backward(ctx: Any, dy: torch.Tensor):
        x2, weight, mean, rstd = ctx.saved_tensors
        dx, dw, _ = ext().layernorm_backward(dy.reshape(x2.shape).contiguous(), x2, weight, mean, rstd, None, True)
        return dx.view(ctx.shape), dw, None


class _AddRMSNorm(torch.autograd.Function):
    """``s = a + b; y = RMSNorm(s)`` in one pass; the backward adds ``ds`` while it writes ``dx``."""

    @staticmethod
    def forward(ctx: Any, a: torch.Tensor, b: torch.Tensor, weight: torch.Tensor, eps: float):
        shape = a.shape
        a2 = a.reshape(-1, shape[-1]).contiguous()
        b2 = b.reshape(-1, shape[-1]).contiguous()
        y, mean, rstd, s = ext().layernorm_forward(a2, weight, None, eps, b2, None)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.shape = shape
        return s.view(shape), y.view(shape)

    @staticmethod
    def backward(ctx: Any, ds, dy):
        s, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            return ds, ds, None, None
        dres = ds.reshape(s.shape).contiguous() if ds is not None else None
        dx, dw, _ = ext().layernorm_backward(dy.reshape(s.shape).contiguous(), s, weight, mean, rstd, dres, True)
        dx = dx.view(ctx.shape)
        return dx, dx, dw, None


def _norm_kernel_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    cols = x.shape[-1]
    return (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16, torch.float32) and weight.dtype == x.dtype
            and (cols * x.element_size()) % 16 == 0 and cols <= 6144)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    if _norm_kernel_ok(x, weight):
        return _RMSNorm.apply(x, weight, eps)
    return F.rms_norm(x, (x.shape[-1],), weight, eps)


def add_rms_norm(a: torch.Tensor, b, weight: torch.Tensor, eps: float = 1e-5):
    """``(a + b, RMSNorm(a + b))``; ``b`` may be ``None``.  On CUDA the add rides in the norm's kernels."""
    if b is None:
        return a, rms_norm(a, weight, eps)
    cols = a.shape[-1]
    fused = (a.is_cuda and b.is_cuda and a.dtype == b.dtype == weight.dtype and a.shape == b.shape
             and a.dtype in (torch.bfloat16, torch.float16, torch.float32)
             and ext().layernorm_can_fuse(a.reshape(-1, cols)))
    if fused:
        return _AddRMSNorm.apply(a, b, weight, eps)
    s = a + b
    return s, rms_norm(s, weight, eps)


class RMSNorm(torch.nn.Module):
    """Root-mean-square norm (weight only) running the fused kernels on CUDA."""

    def __init__(self, dim: int, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.weight, self.eps)

    def add_forward(self, a: torch.Tensor, b, b_bias=None):
        if b is not None and b_bias is not None:
            b = b + b_bias
        return add_rms_norm(a, b, self.weight, self.eps)


class _Rope(torch.autograd.Function):

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
        ctx.save_for_backward(cos, sin)
        return ext().rope(x, cos, sin, False)

    @staticmethod
    def backward(ctx: Any, dy: torch.Tensor):
        cos, sin = ctx.saved_tensors
        if dy.stride(-1) != 1:
            dy = dy.contiguous()
        return ext().rope(dy, cos, sin, True), None, None


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotary embedding of ``x[batch, seq, heads, dim]`` (any strides with a unit one in ``dim``) with
    fp32 tables ``cos`` / ``sin`` of shape ``[seq, dim / 2]``; pairs are ``(i, i + dim / 2)``.
    Returns a contiguous tensor."""
    d = x.shape[-1]
    elem = x.element_size()
    ok = (x.is_cuda and x.dim() == 4 and x.dtype in (torch.bfloat16, torch.float16, torch.float32)
          and x.stride(-1) == 1 and d % (2 * (16 // elem)) == 0 and x.data_ptr() % 16 == 0
          and all((st * elem) % 16 == 0 for st in x.stride()[:3]) and cos.dtype == torch.float32)
    if ok:
        return _Rope.apply(x, cos.contiguous(), sin.contiguous())
    half = d // 2
    x1, x2 = x[..., :half].float(), x[..., half:].float()
    c, s = cos[:x.shape[1]].unsqueeze(1), sin[:x.shape[1]].unsqueeze(1)     # [seq, 1, dim / 2]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)


class _LoadBalancingLoss(torch.autograd.Function):

    @staticmethod
    def forward(ctx: Any, scale: float, layers: int, *tensors):
        scores, counts = list(tensors[:layers]), list(tensors[layers:])
        ctx.scale, ctx.layers = scale, layers
        ctx.save_for_backward(*tensors)
        return ext().lbl_forward(scores, counts, scale)

    @staticmethod
    def backward(ctx: Any, gout: torch.Tensor):
        tensors = ctx.saved_tensors
        scores, counts = list(tensors[:ctx.layers]), list(tensors[ctx.layers:])
        grads = ext().lbl_backward(scores, counts, ctx.scale, gout.detach().float().reshape(1).contiguous())
        return (None, None) + tuple(grads) + (None,) * ctx.layers


def load_balancing_loss_supported(scores, counts) -> bool:
    first = scores[0]
    return (len(scores) <= 64 and all(s.is_cuda and s.is_contiguous() and s.dim() == 2 and s.shape == first.shape
                                      and s.dtype == first.dtype for s in scores)
            and first.dtype in (torch.bfloat16, torch.float16, torch.float32) and first.shape[0] > 0
            and all(c.is_cuda and c.dtype == torch.int32 and c.is_contiguous() for c in counts))


def load_balancing_loss(scores, counts, scale: float) -> torch.Tensor:
    """``scale * sum_l <counts[l], column sums of scores[l]>`` over the layers, as one fp32 scalar.

    One reduction kernel forward (fp32 accumulation, deterministic), one broadcast kernel backward.
    """
    return _LoadBalancingLoss.apply(float(scale), len(scores), *scores, *counts)


class _Linear(torch.autograd.Function):
    """``x @ w.T + b`` with library GEMMs; the bias gradient is the fused column sum."""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor):
        ctx.save_for_backward(x, weight)
        return F.linear(x, weight, bias)

    @staticmethod
    def backward(ctx: Any, dy: torch.Tensor):
        x, weight = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = (dy2 @ weight).view(x.shape)
        if ctx.needs_input_grad[1]:
            dw = dy2.t() @ x.reshape(-1, x.shape[-1])
        if ctx.needs_input_grad[2]:
            db = ext().column_sum(dy2)
        return dx, dw, db


def linear(x: torch.Tensor, weight: torch.Tensor, bias=None) -> torch.Tensor:
    """``F.linear`` with the bias gradient computed by one bandwidth-bound kernel on CUDA."""
    fused = (bias is not None and x.is_cuda and x.dtype in (torch.bfloat16, torch.float16)
             and weight.dtype == x.dtype and bias.dtype == x.dtype and (weight.shape[0] * x.element_size()) % 16 == 0
             and not torch.is_autocast_enabled())
    if fused:
        return _Linear.apply(x, weight, bias)
    return F.linear(x, weight, bias)


class Linear(torch.nn.Linear):
    """``nn.Linear`` (same parameters and state dict) routed through :func:`linear`."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear(x, self.weight, self.bias)

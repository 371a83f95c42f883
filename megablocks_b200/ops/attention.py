"""Causal attention inside a sliding window, with a few first tokens that stay visible.

Query ``i`` sees key ``j`` when ``j <= i`` and (``i - j < window`` or ``j < sinks``).  ``window=None`` is plain
causal attention.  Queries may share keys (``heads`` a multiple of ``kv_heads``: query head ``h`` reads key head
``h * kv_heads // heads``).

* :func:`window_attention` - whole sequences, differentiable, with the lengths of a padded batch;
* :func:`window_attention_decode` - one new token per sequence over a key-value cache.

On CUDA, 16-bit tensors with head sizes up to 128 (multiples of 8) run on the tensor cores
(``csrc/window_attention*.cu``): nothing of the size ``seq x seq`` is stored, keys outside the window are not
read, and the gradients are the same in every run.  Everything else, calls with forward-mode tangents or under
functional transforms among it, is composed of PyTorch ops, which do store the scores.

Products are taken over whole tiles, with probabilities of zero for pairs that are hidden by the window: NaN or an
infinity in ``v`` (in any input, for the gradients) may reach other tokens of the sequence than those that see it.
Behind a sequence's end, and out of sight of a decoded token, anything may stand.
"""

import math
from typing import Optional

import torch

from megablocks_b200._ext import ext, transformed

_KERNEL_DTYPES = (torch.bfloat16, torch.float16)


def _check(q, k, v, window, sinks, lengths, scale, batch):
    tensors = (q, k, v) if lengths is None else (q, k, v, lengths)
    if any(t.device != q.device for t in tensors):
        raise ValueError('q, k, v and lengths must be on one device')
    if not q.dtype == k.dtype == v.dtype or not q.is_floating_point():
        raise ValueError('q, k and v must have one floating-point type')
    if k.shape != v.shape or k.shape[2] < 1 or q.shape[-2] < 1 or q.shape[-2] % k.shape[2]:
        raise ValueError('k and v must have one shape, and the query heads must be a multiple of the key heads')
    if q.shape[-1] != k.shape[-1] or q.shape[-1] < 1:
        raise ValueError('q, k and v must have one head size')
    if window is not None and window < 1:
        raise ValueError(f'window must be at least 1 (or None), got {window}')
    if sinks < 0:
        raise ValueError(f'sinks must not be negative, got {sinks}')
    if lengths is not None and (lengths.shape != (batch,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError('lengths must be int32 or int64 with one entry per sequence')
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f'scale must be positive, got {scale}')


def _kernel_dim(q: torch.Tensor) -> bool:
    return q.is_cuda and q.dtype in _KERNEL_DTYPES and q.shape[-1] % 8 == 0 and q.shape[-1] <= 128


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of ``q[batch, seq, heads, dim]`` over ``k, v[batch, seq, kv_heads, dim]``; returns a contiguous
    tensor like ``q``.

    ``lengths[batch]``: valid tokens of each sequence of a padded batch (clamped to ``[0, seq]``); rows behind
    them are zero, have no gradient, and are not looked at.  ``scale`` is by default ``dim ** -0.5``.  Any
    strides; views of a fused projection with 16-byte aligned rows are read in place, others are copied.  On CUDA
    fewer than 65536 sequences and heads and 2^22 tokens, and differentiable once."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or q.shape[:2] != k.shape[:2]:
        raise ValueError('window_attention expects q[batch, seq, heads, dim] and k, v[batch, seq, kv_heads, dim]')
    scale = q.shape[-1]**-0.5 if scale is None else float(scale)
    _check(q, k, v, window, sinks, lengths, scale, q.shape[0])
    window = max(q.shape[1], 1) if window is None else int(window)
    if not _kernel_dim(q) or q.numel() == 0 or transformed(q, k, v):
        return _composed(q, k, v, window, int(sinks), lengths, scale)
    return ext().window_attention(q, k, v, window, int(sinks), lengths, scale)


def _attend(q, k, v, seen, scale):
    """``q[b, rows, heads, d]`` over ``k, v[b, keys, kv_heads, d]`` with the visible pairs
    ``seen[b or 1, rows, keys]``; rows that see nothing are zero."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    ratio = q.shape[2] // k.shape[2]
    qs = q.to(wide).transpose(1, 2)
    ks, vs = (t.to(wide).transpose(1, 2).repeat_interleave(ratio, dim=1) for t in (k, v))
    seen = seen.unsqueeze(1)
    scores = (qs @ ks.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    some = seen.any(dim=-1, keepdim=True)
    probs = scores.masked_fill(~some, 0.0).softmax(dim=-1) * some
    return (probs @ vs).transpose(1, 2).to(q.dtype).contiguous()


def _composed(q, k, v, window, sinks, lengths, scale):
    batch, seq = q.shape[:2]
    pos = torch.arange(seq, device=q.device)
    gap = pos[:, None] - pos[None, :]
    seen = ((gap >= 0) & ((gap < window) | (pos < sinks)[None, :])).unsqueeze(0)
    if lengths is not None:
        valid = pos < lengths.view(-1, 1)                       # padding may hold anything
        seen = seen & valid.unsqueeze(1) & valid.unsqueeze(2)
        pad = ~valid.view(batch, seq, 1, 1)
        q, k, v = (t.masked_fill(pad, 0.0) for t in (q, k, v))
        return _attend(q, k, v, seen, scale).masked_fill(pad, 0.0)
    return _attend(q, k, v, seen, scale)


def window_attention_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
                            window: Optional[int] = None, sinks: int = 0,
                            scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token per sequence, ``q[batch, heads, dim]``, over the caches
    ``k, v[batch, capacity, kv_heads, dim]``, which hold its own key and value already.

    ``lengths[batch]``: valid tokens, the new one included (clamped to ``[0, capacity]``); an idle slot of length
    0 gives zeros.  Only visible keys are read.  The caches may have any strides; where their rows do not start
    on 16 bytes the visible ones are gathered by PyTorch ops.  On CUDA fewer than 65536 sequences and heads and
    2^30 tokens.  Not differentiable."""
    if q.dim() != 3 or k.dim() != 4 or v.dim() != 4 or q.shape[0] != k.shape[0]:
        raise ValueError('window_attention_decode expects q[batch, heads, dim] and k, v[batch, capacity, kv_heads, dim]')
    if lengths is None:
        raise ValueError('window_attention_decode needs lengths')
    scale = q.shape[-1]**-0.5 if scale is None else float(scale)
    _check(q, k, v, window, sinks, lengths, scale, q.shape[0])
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise ValueError('window_attention_decode is not differentiable: call it without gradients')
    window = max(k.shape[1], 1) if window is None else int(window)
    if (_kernel_dim(q) and q.numel() and k.numel() and not transformed(q, k, v)
            and all(ext().window_attention_in_place(t) for t in (k, v))):
        q = q.contiguous()
        return ext().window_attention_decode(q if q.data_ptr() % 4 == 0 else q.clone(), k, v, lengths, window,
                                             int(sinks), scale)
    return _composed_decode(q, k, v, lengths, window, int(sinks), scale)


def _composed_decode(q, k, v, lengths, window, sinks, scale):
    batch, capacity = k.shape[:2]
    if capacity == 0 or batch == 0:
        return torch.zeros_like(q, memory_format=torch.contiguous_format)
    length = lengths.long().clamp(0, capacity).view(-1, 1)
    lo = (length - window).clamp(min=0)
    first = torch.arange(min(sinks, capacity), device=q.device).expand(batch, -1)
    near = lo + torch.arange(min(window, capacity), device=q.device)
    keys = torch.cat([first, near], dim=1)
    seen = torch.cat([first < lo, near < length], dim=1)
    at = keys.clamp(max=capacity - 1)
    rows = torch.arange(batch, device=q.device).view(-1, 1)
    k, v = (t[rows, at].masked_fill(~seen.view(*seen.shape, 1, 1), 0.0) for t in (k, v))
    return _attend(q.unsqueeze(1), k, v, seen.unsqueeze(1), scale).squeeze(1)

"""Decoder-only transformers whose feed-forward blocks are dMoE / MoE layers.

The reference ships no model code: its experiment scripts train GPT-2 style
models through a Megatron-LM fork that replaces every FFN with a dMoE layer
(exp/dmoe/dmoe_125m_8gpu.sh:53-72,143-148).  This module provides that model
family natively so the library can be trained and benchmarked stand-alone:

* ``gpt2`` flavour: LayerNorm, learned positions, GELU experts, tied LM head;
* ``mixtral`` flavour: RMSNorm, rotary positions, grouped-query attention,
  SwiGLU experts (``mlp_type='glu'``), untied LM head.

Attention uses the library fused attention (``scaled_dot_product_attention``), or this library's windowed
attention where ``attention_window`` or ``attention_sinks`` is set and wherever a key-value cache is;
everything MoE runs this library's kernels.  Inputs are ``[batch, seq]`` token ids.

Beside training (``loss``, ``distillation_loss``) a model answers: ``prefill`` fills a :class:`KVCache` from a
batch of prompts, ``decode`` takes one token per sequence further, ``generate`` does both greedily.  No token is
dropped in an answer, whatever the model's capacity factor.
"""

import contextlib
import dataclasses
import math
from functools import partial
from typing import List, NamedTuple, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from megablocks_b200.layers.arguments import Arguments
from megablocks_b200.layers.dmoe import dMoE
from megablocks_b200.layers.moe import MoE, batched_load_balancing_loss, clear_load_balancing_loss
from megablocks_b200.layers.router import batched_router_zloss, clear_router_zloss
from megablocks_b200.ops import fused
from megablocks_b200.ops.attention import window_attention, window_attention_decode


@dataclasses.dataclass
class TransformerConfig:
    flavour: str = 'gpt2'               # 'gpt2' | 'mixtral'
    vocab_size: int = 51200
    max_seq_len: int = 1024
    num_layers: int = 12
    hidden_size: int = 768
    num_heads: int = 12
    num_kv_heads: Optional[int] = None  # grouped-query attention when < num_heads
    ffn_hidden_size: int = 3072
    moe_num_experts: int = 64
    moe_top_k: int = 1
    moe_loss_weight: float = 0.1
    moe_zloss_weight: float = 0.0
    moe_capacity_factor: int = 1
    dropless: bool = True
    mlp_impl: str = 'grouped'
    memory_optimized_mlp: bool = True
    rope_theta: float = 10000.0
    init_std: float = 0.02
    activation_checkpointing: bool = False
    dtype: torch.dtype = torch.bfloat16
    device: Optional[torch.device] = None
    # expert parallelism
    expert_parallel_group: Optional[object] = None
    ep_fused_comm: Optional[bool] = None
    ep_inflight_microbatches: int = 1
    # pipeline parallelism: this process builds stage `pipeline_stage` of `pipeline_stages`
    pipeline_stages: int = 1
    pipeline_stage: int = 0
    # selection of the experts (see Arguments)
    moe_router_score: str = 'softmax'
    moe_router_bias: bool = False
    moe_router_groups: int = 1
    moe_router_top_groups: Optional[int] = None
    moe_router_scale: float = 1.0
    # attention: a token sees itself and the `attention_window` - 1 before it (None: all), and the first
    # `attention_sinks` tokens
    attention_window: Optional[int] = None
    attention_sinks: int = 0

    @property
    def kv_heads(self) -> int:
        return self.num_kv_heads or self.num_heads

    def moe_arguments(self) -> Arguments:
        glu = self.flavour == 'mixtral'
        return Arguments(
            hidden_size=self.hidden_size,
            ffn_hidden_size=self.ffn_hidden_size,
            num_layers=self.num_layers,
            bias=not glu,
            return_bias=True,      # the bias add rides in the next norm kernel (Block.forward)
            activation_fn=F.silu if glu else partial(F.gelu, approximate='tanh'),
            moe_num_experts=self.moe_num_experts,
            moe_top_k=self.moe_top_k,
            moe_capacity_factor=self.moe_capacity_factor,
            moe_loss_weight=self.moe_loss_weight,
            moe_zloss_weight=self.moe_zloss_weight,
            moe_lbl_in_fp32=True,
            moe_normalize_expert_weights=1 if glu else None,
            moe_expert_model_parallelism=self.expert_parallel_group is not None,
            expert_parallel_group=self.expert_parallel_group,
            memory_optimized_mlp=self.memory_optimized_mlp,
            mlp_type='glu' if glu else 'mlp',
            mlp_impl=self.mlp_impl,
            fp16=self.dtype == torch.float16,
            bf16=self.dtype == torch.bfloat16,
            device=self.device if self.device is not None else torch.device('cpu'),
            init_method=partial(nn.init.normal_, mean=0.0, std=self.init_std),
            output_layer_init_method=partial(nn.init.normal_, mean=0.0,
                                             std=self.init_std / math.sqrt(2.0 * self.num_layers)),
            ep_fused_comm=self.ep_fused_comm,
            ep_inflight_microbatches=self.ep_inflight_microbatches,
            pipeline_model_parallel_size=self.pipeline_stages,
            moe_router_score=self.moe_router_score,
            moe_router_bias=self.moe_router_bias,
            moe_router_groups=self.moe_router_groups,
            moe_router_top_groups=self.moe_router_top_groups,
            moe_router_scale=self.moe_router_scale,
        )


# Named configurations: the dMoE family trained by the reference's experiment
# scripts (exp/dmoe/*.sh: 64 experts, top-1, ffn = 4 x hidden, seq 1024) and a
# Mixtral-8x7B-shaped model.
PRESETS = {
    'dmoe-46m': dict(num_layers=6, hidden_size=512, num_heads=8, ffn_hidden_size=2048),
    'dmoe-125m': dict(num_layers=12, hidden_size=768, num_heads=12, ffn_hidden_size=3072),
    'dmoe-356m': dict(num_layers=24, hidden_size=1024, num_heads=16, ffn_hidden_size=4096),
    'dmoe-760m': dict(num_layers=24, hidden_size=1536, num_heads=16, ffn_hidden_size=6144),
    'dmoe-1315m': dict(num_layers=24, hidden_size=2048, num_heads=16, ffn_hidden_size=8192),
    'mixtral-8x7b': dict(flavour='mixtral', vocab_size=32000, max_seq_len=4096, num_layers=32, hidden_size=4096,
                         num_heads=32, num_kv_heads=8, ffn_hidden_size=14336, moe_num_experts=8, moe_top_k=2,
                         rope_theta=1e6),
    'tiny': dict(vocab_size=512, max_seq_len=64, num_layers=2, hidden_size=128, num_heads=4, ffn_hidden_size=256,
                 moe_num_experts=8, moe_top_k=2),
    'tiny-mixtral': dict(flavour='mixtral', vocab_size=512, max_seq_len=64, num_layers=2, hidden_size=128,
                         num_heads=4, num_kv_heads=2, ffn_hidden_size=256, moe_num_experts=4, moe_top_k=2),
}


def preset(name: str, **overrides) -> TransformerConfig:
    cfg = dict(PRESETS[name])
    cfg.update(overrides)
    return TransformerConfig(**cfg)


RMSNorm = fused.RMSNorm


class Teacher(NamedTuple):
    """A teacher's kept logits of a batch, for :meth:`MoETransformer.distillation_loss`."""
    logits: torch.Tensor                # [batch, seq, top]
    ids: torch.Tensor                   # [batch, seq, top] int32 or int64; outside the vocabulary: unused
    temperature: float = 1.0
    hard_weight: float = 0.0            # of the targets' cross entropy


@dataclasses.dataclass
class KVCache:
    """Keys and values of every layer, ``[batch, capacity, kv_heads, head_dim]`` each, and the valid tokens of
    every sequence.  ``used`` is the longest sequence's length as far as the host knows it."""
    keys: List[torch.Tensor]
    values: List[torch.Tensor]
    lengths: torch.Tensor               # int32 [batch]
    used: int = 0

    @property
    def capacity(self) -> int:
        return self.keys[0].shape[1]


def _rope_tables(seq_len: int, head_dim: int, theta: float, device):
    inv = 1.0 / (theta**(torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    ang = torch.outer(torch.arange(seq_len, device=device, dtype=torch.float32), inv)
    return ang.cos().contiguous(), ang.sin().contiguous()


class Attention(nn.Module):

    def __init__(self, cfg: TransformerConfig):
        super().__init__()
        self.cfg = cfg
        self.head_dim = cfg.hidden_size // cfg.num_heads
        kw = dict(device=cfg.device, dtype=cfg.dtype)
        bias = cfg.flavour == 'gpt2'
        qkv_out = (cfg.num_heads + 2 * cfg.kv_heads) * self.head_dim
        self.qkv = fused.Linear(cfg.hidden_size, qkv_out, bias=bias, **kw)
        self.proj = fused.Linear(cfg.hidden_size, cfg.hidden_size, bias=bias, **kw)
        nn.init.normal_(self.qkv.weight, std=cfg.init_std)
        nn.init.normal_(self.proj.weight, std=cfg.init_std / math.sqrt(2.0 * cfg.num_layers))
        if bias:
            nn.init.zeros_(self.qkv.bias)
            nn.init.zeros_(self.proj.bias)

    def _project(self, x: torch.Tensor, rope):
        """Queries, keys and values ``[batch, seq, heads, head_dim]``, rotated."""
        b, s, _ = x.shape
        cfg = self.cfg
        q_dim, kv_dim = cfg.num_heads * self.head_dim, cfg.kv_heads * self.head_dim
        q, k, v = self.qkv(x).split([q_dim, kv_dim, kv_dim], dim=-1)
        q = q.view(b, s, cfg.num_heads, self.head_dim)
        k = k.view(b, s, cfg.kv_heads, self.head_dim)
        if rope is not None:     # rotate the [batch, seq, heads, dim] views of the fused projection in one pass each
            q, k = fused.rope(q, *rope), fused.rope(k, *rope)
        return q, k, v.view(b, s, cfg.kv_heads, self.head_dim)

    def prefill(self, x: torch.Tensor, rope, keys: torch.Tensor, values: torch.Tensor,
                lengths: torch.Tensor) -> torch.Tensor:
        """Whole prompts; their keys and values go to the start of the caches."""
        b, s, _ = x.shape
        q, k, v = self._project(x, rope)
        keys[:, :s].copy_(k)
        values[:, :s].copy_(v)
        out = window_attention(q, k, v, self.cfg.attention_window, self.cfg.attention_sinks, lengths)
        return self.proj(out.reshape(b, s, -1))

    def decode(self, x: torch.Tensor, rope, keys: torch.Tensor, values: torch.Tensor, at: torch.Tensor,
               lengths: torch.Tensor) -> torch.Tensor:
        """One token per sequence (``x[1, batch, hidden]``, the batch in the place of the positions, as the
        rotary tables have it) at position ``at[batch]`` of the caches, ``lengths`` with it."""
        q, k, v = (t.squeeze(0).to(keys.dtype) for t in self._project(x, rope))        # autocast may differ
        rows = torch.arange(at.shape[0], device=at.device)
        keys[rows, at] = k
        values[rows, at] = v
        out = window_attention_decode(q, keys, values, lengths, self.cfg.attention_window, self.cfg.attention_sinks)
        return self.proj(out.reshape(1, at.shape[0], -1))

    def forward(self, x: torch.Tensor, rope) -> torch.Tensor:
        b, s, _ = x.shape
        cfg = self.cfg
        q, k, v = self._project(x, rope)
        if cfg.attention_window is not None or cfg.attention_sinks:
            out = window_attention(q, k, v, cfg.attention_window, cfg.attention_sinks)
            return self.proj(out.reshape(b, s, -1))
        q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
        out = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=cfg.kv_heads != cfg.num_heads)
        return self.proj(out.transpose(1, 2).reshape(b, s, -1))


def _add_norm(norm: nn.Module, x: torch.Tensor, delta, delta_bias=None):
    """``(x + delta [+ delta_bias], norm(...))``; ``delta_bias`` is the per-column output bias of the
    layer that produced ``delta``."""
    if hasattr(norm, 'add_forward'):
        return norm.add_forward(x, delta, delta_bias)
    if delta is not None:
        x = x + delta if delta_bias is None else x + delta + delta_bias
    return x, norm(x)


class Block(nn.Module):

    def __init__(self, cfg: TransformerConfig, moe_args: Arguments):
        super().__init__()
        kw = dict(device=cfg.device, dtype=cfg.dtype)
        norm = RMSNorm if cfg.flavour == 'mixtral' else fused.LayerNorm
        self.ln1 = norm(cfg.hidden_size, **kw)
        self.attn = Attention(cfg)
        self.ln2 = norm(cfg.hidden_size, **kw)
        self.moe = (dMoE if cfg.dropless else MoE)(moe_args)

    def forward(self, x: torch.Tensor, delta, delta_bias, rope, attend=None):
        """The residual stream arrives as ``x + delta + delta_bias`` (``delta`` may be ``None``;
        ``delta_bias`` is the previous MoE layer's output bias, one value per column, or ``None``)
        and leaves the same way, so every residual add rides in the following norm's kernels.
        ``attend`` (optional) takes the place of the attention layer's forward pass."""
        x, normed = _add_norm(self.ln1, x, delta, delta_bias)
        x, normed = _add_norm(self.ln2, x, self.attn(normed, rope) if attend is None else attend(self.attn, normed))
        # The MoE layer is token-wise: it flattens every leading dimension, so the
        # [batch, seq, hidden] activations go in as they are (no transpose copy).
        out = self.moe(normed)
        if isinstance(out, tuple):        # return_bias: (output without the bias, bias vector)
            return x, out[0], out[1]
        return x, out, None


class MoETransformer(nn.Module):
    """Token ids ``[batch, seq]`` -> logits ``[batch, seq, vocab]`` (and the training loss)."""

    def __init__(self, cfg: TransformerConfig):
        super().__init__()
        self.cfg = cfg
        self.moe_args = cfg.moe_arguments()
        kw = dict(device=cfg.device, dtype=cfg.dtype)
        # A pipeline stage owns a contiguous slice of the blocks; the first stage also owns the
        # embeddings, the last one the final norm and the LM head (which is then a matrix of its
        # own: the tied GPT-2 head would need the embedding of another process).
        from megablocks_b200.parallel.pipeline import stage_layers
        if cfg.pipeline_stages > 1 and cfg.num_layers % cfg.pipeline_stages:
            raise ValueError('num_layers must be divisible by pipeline_stages (the load-balancing loss expects '
                             'num_layers / pipeline_stages terms per stage)')
        self.is_first_stage = cfg.pipeline_stage == 0
        self.is_last_stage = cfg.pipeline_stage == cfg.pipeline_stages - 1
        self.wte = self.wpe = self.ln_f = self.lm_head = None
        if self.is_first_stage:
            self.wte = nn.Embedding(cfg.vocab_size, cfg.hidden_size, **kw)
            nn.init.normal_(self.wte.weight, std=cfg.init_std)
            if cfg.flavour == 'gpt2':
                self.wpe = nn.Embedding(cfg.max_seq_len, cfg.hidden_size, **kw)
                nn.init.normal_(self.wpe.weight, std=cfg.init_std)
        layers = stage_layers(cfg.num_layers, cfg.pipeline_stages, cfg.pipeline_stage)
        self.blocks = nn.ModuleList([Block(cfg, self.moe_args) for _ in layers])
        norm = RMSNorm if cfg.flavour == 'mixtral' else fused.LayerNorm
        if self.is_last_stage:
            self.ln_f = norm(cfg.hidden_size, **kw)
            if cfg.flavour == 'mixtral' or not self.is_first_stage:
                self.lm_head = nn.Linear(cfg.hidden_size, cfg.vocab_size, bias=False, **kw)
                nn.init.normal_(self.lm_head.weight, std=cfg.init_std)
        self._ropes = {}             # device -> rotary tables, each at least twice as long as the one before

    def _rope_for(self, seq: int, device):
        """Rotary tables of at least ``seq`` positions, cut to them.  Tables that are replaced stay alive: a recorded
        step or decode call reads them where they are."""
        if self.cfg.flavour != 'mixtral':
            return None
        kept = self._ropes.setdefault(device, [])
        if not kept or kept[-1][0].shape[0] < seq:
            size = max(seq, self.cfg.max_seq_len, 2 * kept[-1][0].shape[0] if kept else 0)
            with torch.inference_mode(False):                   # training may use them next
                tables = _rope_tables(size, self.cfg.hidden_size // self.cfg.num_heads, self.cfg.rope_theta, device)
            if tables[0].is_cuda and torch.cuda.is_current_stream_capturing():
                return tables[0][:seq], tables[1][:seq]         # filled by the replays only: not for others
            kept.append(tables)
        return kept[-1][0][:seq], kept[-1][1][:seq]

    def _embed(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.wte(tokens)
        if self.wpe is not None:
            x = x + self.wpe(torch.arange(tokens.shape[1], device=tokens.device))
        return x

    def _run_blocks(self, x: torch.Tensor, attend=None):
        """Residual stream through this process's blocks; returns ``(x, delta, delta_bias)`` with the
        last block's output (and its bias vector, if any) still to be added.  ``attend(layer, attention,
        normed)`` takes the place of the attention layers' forward pass."""
        delta = delta_bias = None
        if attend is not None:
            for i, block in enumerate(self.blocks):
                x, delta, delta_bias = block(x, delta, delta_bias, None, partial(attend, i))
            return x, delta, delta_bias
        rope = self._rope_for(x.shape[1], x.device)
        for block in self.blocks:
            if self.cfg.activation_checkpointing and self.training:
                x, delta, delta_bias = checkpoint(block, x, delta, delta_bias, rope, use_reentrant=False)
            else:
                x, delta, delta_bias = block(x, delta, delta_bias, rope)
        return x, delta, delta_bias

    def hidden_states(self, tokens: torch.Tensor) -> torch.Tensor:
        x, delta, delta_bias = self._run_blocks(self._embed(tokens))
        return _add_norm(self.ln_f, x, delta, delta_bias)[1]

    def _aux_loss(self):
        """This stage's auxiliary losses of the forward pass just run (``None`` when there are none);
        clears the per-step accumulators."""
        aux = None
        if self.training and self.moe_args.moe_loss_weight > 0:
            aux = batched_load_balancing_loss(self.moe_args)
        if self.training and self.moe_args.moe_zloss_weight > 0:
            z = batched_router_zloss(self.moe_args).sum()
            aux = z if aux is None else aux + z
        clear_load_balancing_loss()
        clear_router_zloss()
        return aux

    # -- pipeline stages ---------------------------------------------------------------
    def stage_forward(self, inp: torch.Tensor):
        """One pipeline stage: token ids (first stage) or the previous stage's activations in,
        ``(activations for the next stage, auxiliary loss of this stage or None)`` out.  The last
        stage returns the un-normalised residual stream for :meth:`stage_loss`."""
        x, delta, delta_bias = self._run_blocks(self._embed(inp) if self.is_first_stage else inp)
        if delta is not None:
            x = x + delta if delta_bias is None else x + delta + delta_bias
        return x, self._aux_loss()

    def stage_loss(self, hidden: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """Last stage: final norm, LM head and cross entropy."""
        return self._lm_loss(self.ln_f(hidden), targets)

    def _lm_loss(self, hidden: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """Language-model head and mean cross entropy (the logits are written once and read once)."""
        weight = self.lm_head.weight if self.lm_head is not None else self.wte.weight
        return fused.linear_cross_entropy(hidden.reshape(-1, hidden.shape[-1]), weight, targets.reshape(-1))

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        weight = self.lm_head.weight if self.lm_head is not None else self.wte.weight
        return F.linear(hidden, weight)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return self.logits(self.hidden_states(tokens))

    def loss(self, tokens: torch.Tensor, targets: torch.Tensor):
        """Next-token cross entropy plus the MoE auxiliary losses.

        Returns ``(total, lm_loss)``.  Clears the per-step loss accumulators.
        """
        if self.cfg.pipeline_stages > 1:
            raise RuntimeError('a pipeline stage is driven through stage_forward / stage_loss')
        lm = self._lm_loss(self.hidden_states(tokens), targets)
        aux = self._aux_loss()
        total = lm if aux is None else lm + aux
        return total, lm.detach()

    def distillation_loss(self, tokens: torch.Tensor, teacher: Teacher, targets: Optional[torch.Tensor] = None):
        """The loss against a teacher's kept logits (:func:`fused.linear_distillation_loss`), with
        ``teacher.hard_weight`` times the targets' cross entropy, plus the MoE auxiliary losses.

        Returns ``(total, distillation loss)``.  Clears the per-step loss accumulators.
        """
        if self.cfg.pipeline_stages > 1:
            raise RuntimeError('a pipeline stage is driven through stage_forward / stage_loss')
        top = teacher.logits.shape[-1]
        if teacher.logits.shape[:-1] != tokens.shape or teacher.ids.shape != teacher.logits.shape:
            raise ValueError('a teacher has logits and ids [batch, seq, top] for tokens [batch, seq]')
        hidden = self.hidden_states(tokens)
        weight = self.lm_head.weight if self.lm_head is not None else self.wte.weight
        loss = fused.linear_distillation_loss(
            hidden.reshape(-1, hidden.shape[-1]), weight, teacher.logits.reshape(-1, top),
            teacher.ids.reshape(-1, top), teacher.temperature, None if targets is None else targets.reshape(-1),
            teacher.hard_weight)
        aux = self._aux_loss()
        return loss if aux is None else loss + aux, loss.detach()

    # -- answering -----------------------------------------------------------------------
    def new_cache(self, batch: int, capacity: int) -> KVCache:
        """An empty key-value cache for ``batch`` sequences of up to ``capacity`` tokens."""
        cfg = self.cfg
        if cfg.pipeline_stages > 1:
            raise RuntimeError('a pipeline stage does not answer by itself')
        if batch < 1 or capacity < 1:
            raise ValueError('a cache holds at least one sequence of one token')
        if self.wpe is not None and capacity > cfg.max_seq_len:
            raise ValueError(f'the model has {cfg.max_seq_len} positions, a cache of {capacity} does not fit')
        weight = self.wte.weight
        self._rope_for(capacity, weight.device)         # before a call is recorded
        shape = (batch, capacity, cfg.kv_heads, cfg.hidden_size // cfg.num_heads)
        with torch.inference_mode(False):               # a cache may be written in any mode
            buffers = [[torch.zeros(shape, dtype=weight.dtype, device=weight.device) for _ in self.blocks]
                       for _ in range(2)]
            return KVCache(*buffers, torch.zeros(batch, dtype=torch.int32, device=weight.device))

    @contextlib.contextmanager
    def _answering(self, capacity_factor: float):
        """Without gradients and, whatever mode the model is in, without what only training does: the layers'
        loss accumulators and load counts, jitter, and tokens that are dropped, which would make an answer depend on
        the padding and on the other sequences."""
        training = [m for m in self.modules() if m.training] if self.training else []
        for m in training:
            m.training = False
        factor = self.moe_args.moe_capacity_factor
        if not self.cfg.dropless:
            self.moe_args.moe_capacity_factor = capacity_factor
        try:
            with torch.no_grad():
                yield
        finally:
            self.moe_args.moe_capacity_factor = factor
            for m in training:
                m.training = True

    def prefill(self, tokens: torch.Tensor, cache: KVCache, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Fill the cache from prompts ``tokens[batch, seq]`` (``lengths[batch]`` valid tokens each, at least one;
        ``None``: all); returns the logits ``[batch, vocab]`` behind each prompt's last token."""
        with self._answering(0):            # as many places as the fullest expert needs
            return self._prefill(tokens, cache, lengths)

    def _prefill(self, tokens, cache, lengths):
        b, s = tokens.shape
        if b != cache.lengths.shape[0] or not 1 <= s <= cache.capacity:
            raise ValueError(f'prompts of {s} tokens for {b} sequences do not fit a cache of {cache.capacity} tokens '
                             f'for {cache.lengths.shape[0]}')
        if lengths is None:
            lengths = torch.full((b,), s, dtype=torch.int32, device=tokens.device)
        elif lengths.shape != (b,):
            raise ValueError('lengths must have one entry per sequence')
        cache.lengths.copy_(lengths.clamp(1, s))
        cache.used = s
        rope = self._rope_for(s, tokens.device)
        valid = cache.lengths.clone()

        def attend(layer, attention, normed):
            return attention.prefill(normed, rope, cache.keys[layer], cache.values[layer], valid)

        x, delta, delta_bias = self._run_blocks(self._embed(tokens), attend)
        hidden = _add_norm(self.ln_f, x, delta, delta_bias)[1]
        last = (cache.lengths - 1).long()
        return self.logits(hidden[torch.arange(b, device=tokens.device), last])

    def decode(self, tokens: torch.Tensor, cache: KVCache) -> torch.Tensor:
        """Take every sequence one token further: ``tokens[batch]`` go to the end of the cache; returns the logits
        ``[batch, vocab]`` behind them.

        A recorded call may be replayed: lengths advance on the device, and a token for which a sequence has no
        room takes the place of its last one."""
        # A place for every token with every expert, which takes no look at the counts and so can be recorded (2^-20:
        # whatever the products round to, no place less).
        with self._answering(self.cfg.moe_num_experts / self.cfg.moe_top_k * (1 + 2.0**-20)):
            return self._decode(tokens, cache)

    def _decode(self, tokens, cache):
        if tokens.shape != cache.lengths.shape:
            raise ValueError('decode takes one token per sequence of the cache')
        if not 1 <= cache.used < cache.capacity:
            raise ValueError(f'the cache holds {cache.used} of {cache.capacity} tokens: it has to be filled first and '
                             'have room for one more')
        # `used` says nothing of replays of a recorded call, which must not write behind the cache.
        at = cache.lengths.long().clamp_(0, cache.capacity - 1)
        torch.add(at, 1, out=cache.lengths)
        cache.used += 1
        rope = self._rope_for(cache.capacity, tokens.device)
        if rope is not None:
            rope = tuple(t[at] for t in rope)       # each sequence at its own position

        def attend(layer, attention, normed):
            return attention.decode(normed, rope, cache.keys[layer], cache.values[layer], at, cache.lengths)

        x = self.wte(tokens)
        if self.wpe is not None:
            x = x + self.wpe(at)
        x, delta, delta_bias = self._run_blocks(x.unsqueeze(0), attend)
        return self.logits(_add_norm(self.ln_f, x, delta, delta_bias)[1].squeeze(0))

    def generate(self, tokens: torch.Tensor, steps: int, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``steps`` most likely tokens behind each prompt: ``[batch, steps]``."""
        if steps < 1:
            raise ValueError('generate takes at least one step')
        cache = self.new_cache(tokens.shape[0], tokens.shape[1] + steps - 1)           # the last token is not fed back
        out = [self.prefill(tokens, cache, lengths).argmax(dim=-1)]
        for _ in range(steps - 1):
            out.append(self.decode(out[-1], cache).argmax(dim=-1))
        return torch.stack(out, dim=1)

    def num_parameters(self, only_active: bool = False) -> int:
        total = 0
        for name, p in self.named_parameters():
            n = p.numel()
            if only_active and '.moe.experts.mlp.' in name:
                n = n * self.cfg.moe_top_k // max(1, p.shape[0] // self.cfg.ffn_hidden_size)
            total += n
        return total

"""Operators of a mixture-of-experts language model, as measurable cases.

A case is a dict of plain values.  ``listed()`` names those that stand for the operators' main uses;
``draw(rng)`` makes further ones over the same ranges.  Four kinds:

* ``route``    expert selection: softmax or sigmoid scores, a balancing bias, expert groups, top-k,
  renormalised weights (``ops.select_experts``), alone or with its backward pass;
* ``window``   causal attention inside a sliding window with a few first tokens that stay visible
  (``ops.window_attention``), alone or with its backward pass;
* ``decode``   the same attention for one new token per sequence over a key-value cache
  (``ops.window_attention_decode``);
* ``distill``  distillation from a teacher's top logits, loss and gradient (``ops.fused.distillation_loss``).

``run`` computes a pass in its plain form, with elementary torch operations, or, where ``own`` is true,
with the library's kernels.  Head counts, head sizes, vocabularies and expert counts are those of the
presets (``models/transformer.py``) or generic ones.
"""

import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}


def _route(name, tokens, experts, top_k, *, score, bias, groups=1, top_groups=1, norm_p=0, scale=1.0, dtype='bf16',
           train=True, aux=False):
    return dict(name=name, kind='route', tokens=tokens, experts=experts, top_k=top_k, score=score, bias=bias,
                groups=groups, top_groups=top_groups, norm_p=norm_p, scale=scale, dtype=dtype, train=train, aux=aux)


def _window(name, batch, seq, heads, kv_heads, dim, window, sinks, *, dtype='bf16', train=True, ragged=False):
    return dict(name=name, kind='window', batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                window=window, sinks=sinks, dtype=dtype, train=train, ragged=ragged)


def _decode(name, batch, capacity, heads, kv_heads, dim, window, sinks, *, dtype='bf16'):
    return dict(name=name, kind='decode', batch=batch, capacity=capacity, heads=heads, kv_heads=kv_heads, dim=dim,
                window=window, sinks=sinks, dtype=dtype)


def _distill(name, rows, vocab, top, *, temperature, hard, dtype='bf16'):
    return dict(name=name, kind='distill', rows=rows, vocab=vocab, top=top, temperature=temperature, hard=hard,
                dtype=dtype)


def listed():
    return [
        # A decode step of sixteen sequences through a layer with 256 small experts in eight groups: latency.
        _route('route_decode', 16, 256, 8, score='sigmoid', bias=True, groups=8, top_groups=4, norm_p=1, scale=2.5,
               train=False),
        # A micro-batch of 32 x 1024 tokens through the same layer, balanced by its bias alone: the gradient
        # arrives through the weights only.
        _route('route_train_grouped', 32768, 256, 8, score='sigmoid', bias=True, groups=8, top_groups=4, norm_p=1,
               scale=2.5),
        # A ragged batch over an expert count that fills no vector, softmax scores in 32 bits, with the
        # gradient of an auxiliary loss on the scores.
        _route('route_train_odd', 8191, 60, 4, score='softmax', bias=True, norm_p=1, dtype='fp32', aux=True),
        # The layers of the `tiny` preset at batch 4 x 64, with a window: debugging and unit-test sizes.
        _window('window_tiny', 4, 64, 4, 4, 32, 16, 2, dtype='fp16'),
        # A micro-batch of the 125M model (12 heads of 64, 1024 tokens) with a window of a quarter.
        _window('window_train_125m', 8, 1024, 12, 12, 64, 256, 4),
        # A padded fine-tuning batch: ragged lengths, heads of 96, grouped queries.
        _window('window_train_padded', 6, 1999, 16, 4, 96, 512, 4, dtype='fp16', ragged=True),
        # One long document, 32 query heads over 8 key heads of 128: the largest.
        _window('window_train_long', 1, 16384, 32, 8, 128, 4096, 4),
        # Prefill of a prompt of odd length through the same heads.
        _window('window_prefill', 1, 8191, 32, 8, 128, 1024, 4, train=False),
        # One sequence answering far into a long cache: all latency.
        _decode('decode_one', 1, 65536, 32, 8, 128, 4096, 4),
        # A serving batch of ragged lengths, one slot idle.
        _decode('decode_batch', 64, 8192, 32, 8, 128, 4096, 4),
        # A micro-batch of 8 x 1024 tokens over the presets' vocabulary, 64 teacher logits a token.
        _distill('distill_train', 8192, 51200, 64, temperature=2.0, hard=0.0),
        # A ragged fp16 batch with the targets' cross entropy in the same pass.
        _distill('distill_mixed', 1021, 32000, 20, temperature=2.0, hard=0.5, dtype='fp16'),
    ]


# ----------------------------------------------------------------------------
# Drawing
# ----------------------------------------------------------------------------
_MAX_ROUTE = 32768 * 256
_MAX_PAIRS = 16384 * 4096 * 32 * 128                # pairs x heads x dim of the largest window case
_MAX_TOKENS = 16384 * 32 * 128                      # elements of its queries
_MAX_CACHE = 64 * 8192 * 8 * 128                    # elements of one of the largest caches
_MAX_LOGITS = 8192 * 51200


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_route(rng):
    groups = rng.choice((1, 1, 2, 4, 8))
    experts = groups * max(2, _log(rng, 8, 512) // groups)
    top_groups = rng.randint(1, groups)
    top_k = rng.randint(1, min(12, top_groups * (experts // groups)))
    return dict(kind='route', tokens=min(_log(rng, 1, 32768), _MAX_ROUTE // experts), experts=experts, top_k=top_k,
                score=rng.choice(('softmax', 'sigmoid')), bias=groups == 1 and rng.random() < 0.5 or groups > 1,
                groups=groups, top_groups=top_groups, norm_p=rng.choice((0, 1, 1, 2)),
                scale=rng.choice((1.0, 2.5)), dtype=rng.choice(('bf16', 'bf16', 'fp16', 'fp32')),
                train=rng.random() < 0.6, aux=rng.random() < 0.5)


def _draw_heads(rng):
    kv_heads = rng.choice((1, 2, 4, 8, 12))
    heads = min(32, kv_heads * rng.choice((1, 1, 2, 4, 8)))
    return heads - heads % kv_heads, kv_heads, rng.choice((32, 64, 64, 80, 96, 128, 128))


def _draw_window(rng):
    heads, kv_heads, dim = _draw_heads(rng)
    seq = _log(rng, 1, 16384)
    window = min(_log(rng, 8, 4096), seq)
    batch = _log(rng, 1, 8)
    while batch > 1 and (batch * seq * heads * dim > _MAX_TOKENS or batch * seq * window * heads * dim > _MAX_PAIRS):
        batch -= 1
    return dict(kind='window', batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, window=window,
                sinks=rng.choice((0, 1, 4, 16)), dtype=rng.choice(('bf16', 'bf16', 'fp16')),
                train=rng.random() < 0.7, ragged=batch > 1 and rng.random() < 0.5)


def _draw_decode(rng):
    heads, kv_heads, dim = _draw_heads(rng)
    capacity = _log(rng, 16, 65536)
    batch = max(1, min(_log(rng, 1, 64), _MAX_CACHE // (capacity * kv_heads * dim)))
    return dict(kind='decode', batch=batch, capacity=capacity, heads=heads, kv_heads=kv_heads, dim=dim,
                window=min(_log(rng, 8, 4096), capacity), sinks=rng.choice((0, 1, 4, 16)),
                dtype=rng.choice(('bf16', 'bf16', 'fp16')))


def _draw_distill(rng):
    vocab = rng.choice((512, 32000, 51200, 50257, _log(rng, 100, 130000)))
    return dict(kind='distill', rows=max(1, min(_log(rng, 16, 8192), _MAX_LOGITS // vocab)), vocab=vocab,
                top=min(_log(rng, 1, 128), vocab), temperature=rng.choice((1.0, 2.0, 4.0)),
                hard=rng.choice((0.0, 0.0, 0.5)), dtype=rng.choice(('bf16', 'bf16', 'fp16', 'fp32')))


def draw(rng):
    return rng.choice((_draw_route, _draw_window, _draw_window, _draw_decode, _draw_distill))(rng)


# ----------------------------------------------------------------------------
# What a program has in hand before the call
# ----------------------------------------------------------------------------
def _lengths(case):
    """Valid keys of each sequence: between a quarter and all of them, spread by the golden ratio; in a
    serving batch every sixteenth slot is idle."""
    n = case['capacity'] if case['kind'] == 'decode' else case['seq']
    out = []
    for b in range(case['batch']):
        part = (0.6180339887498949 * b) % 1.0
        out.append(max(1, int(round(n * (1.0 - 0.75 * part)))))
        if case['kind'] == 'decode' and b % 16 == 9:
            out[-1] = 0
    return out


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device='cuda', dtype=torch.float32) * scale).to(dtype)


def _prepare_route(case, gen):
    dtype = _DTYPES[case['dtype']]
    tokens, experts, top_k = case['tokens'], case['experts'], case['top_k']
    # Logits of a router under way: some experts are liked by most tokens, and the bias works against it.
    liked = _randn(gen, 1, experts, scale=0.5)
    state = dict(logits=(_randn(gen, tokens, experts) + liked).to(dtype), bias=None)
    if case['bias']:
        state['bias'] = (-0.05 * liked[0] + _randn(gen, experts, scale=0.01)).contiguous()
    if case['train']:
        state['logits'].requires_grad_(True)
        state['dweights'] = _randn(gen, tokens, top_k, dtype=dtype)
        if case['aux']:
            state['dscores'] = _randn(gen, 1, experts, scale=0.1).to(dtype).repeat(tokens, 1)
    return state


def _prepare_window(case, gen):
    """Queries, keys and values as a model has them: views of one projection of the hidden states."""
    dtype = _DTYPES[case['dtype']]
    b, s, hq, hk, d = (case[k] for k in ('batch', 'seq', 'heads', 'kv_heads', 'dim'))
    qkv = _randn(gen, b, s, (hq + 2 * hk) * d, dtype=dtype)
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=-1)
    state = dict(q=q.view(b, s, hq, d), k=k.view(b, s, hk, d), v=v.view(b, s, hk, d), lengths=None)
    if case['ragged']:
        state['lengths'] = torch.tensor(_lengths(case), dtype=torch.int32, device='cuda')
    if case['train']:
        for name in 'qkv':
            state[name].requires_grad_(True)
        state['dout'] = _randn(gen, b, s, hq, d, dtype=dtype)
    return state


def _prepare_decode(case, gen):
    dtype = _DTYPES[case['dtype']]
    b, n, hq, hk, d = (case[k] for k in ('batch', 'capacity', 'heads', 'kv_heads', 'dim'))
    return dict(q=_randn(gen, b, hq, d, dtype=dtype), k=_randn(gen, b, n, hk, d, dtype=dtype),
                v=_randn(gen, b, n, hk, d, dtype=dtype),
                lengths=torch.tensor(_lengths(case), dtype=torch.int32, device='cuda'))


def _prepare_distill(case, gen):
    dtype = _DTYPES[case['dtype']]
    rows, vocab, top = case['rows'], case['vocab'], case['top']
    logits = _randn(gen, rows, vocab, dtype=dtype, scale=2.0)
    # The teacher agrees with the student in part; its best logits are kept, fewer of them in some rows,
    # none in the rows of a padded tail.
    values, ids = [], []
    for part in logits.split(1024):
        best = (part.float() + _randn(gen, *part.shape, scale=2.0)).topk(top, dim=-1)
        values.append(best.values)
        ids.append(best.indices)
    values, ids = torch.cat(values), torch.cat(ids)
    kept = torch.randint(max(1, top // 2), top + 1, (rows, 1), generator=gen, device='cuda')
    kept[rows - rows // 16:] = 0
    ids = ids.masked_fill(torch.arange(top, device='cuda') >= kept, -1)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device='cuda')
    targets[rows - rows // 16:] = -100
    # 16-bit floats train under a loss scale, which is what the gradient of the loss then is.
    dloss = torch.full((), 4096.0 if dtype == torch.float16 else 1.0, device='cuda')
    return dict(logits=logits.requires_grad_(True), values=values, ids=ids, targets=targets, dloss=dloss)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    state = {'route': _prepare_route, 'window': _prepare_window, 'decode': _prepare_decode,
             'distill': _prepare_distill}[case['kind']](case, gen)
    return dict(state, case=case)


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------
def _own_route(state, case):
    from megablocks_b200 import ops
    logits = state['logits']
    scores, weights, experts = ops.select_experts(
        logits, case['top_k'], score=case['score'], bias=state['bias'], groups=case['groups'],
        top_groups=case['top_groups'], norm_p=case['norm_p'] or None, scale=case['scale'])
    out = [scores.detach(), weights.detach(), experts]
    if case['train']:
        if case['aux']:
            out += torch.autograd.grad([scores, weights], [logits], [state['dscores'], state['dweights']])
        else:
            out += torch.autograd.grad([weights], [logits], [state['dweights']])
    return out


def _own_window(state, case):
    from megablocks_b200 import ops
    q, k, v = state['q'], state['k'], state['v']
    out = ops.window_attention(q, k, v, window=case['window'], sinks=case['sinks'], lengths=state['lengths'])
    if not case['train']:
        return [out]
    return [out.detach(), *torch.autograd.grad([out], [q, k, v], [state['dout']])]


def _own_decode(state, case):
    from megablocks_b200 import ops
    return [ops.window_attention_decode(state['q'], state['k'], state['v'], state['lengths'], window=case['window'],
                                        sinks=case['sinks'])]


def _own_distill(state, case):
    from megablocks_b200.ops import fused
    logits = state['logits']
    loss = fused.distillation_loss(logits, state['values'], state['ids'], temperature=case['temperature'],
                                   targets=state['targets'] if case['hard'] else None, hard_weight=case['hard'])
    return [loss.detach(), *torch.autograd.grad([loss], [logits], [state['dloss']])]


# The plain forms.  Everything in 32 bits, but for the choice of experts: two scores that are closer than
# 32 bits tell apart have an order all the same, so the values that are compared have 64.
def _scores(x, kind):
    if kind == 'sigmoid':
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


@torch.no_grad()
def _plain_route(state, case):
    dtype = _DTYPES[case['dtype']]
    tokens, experts, top_k, groups = case['tokens'], case['experts'], case['top_k'], case['groups']
    logits = state['logits'].detach()
    wide = logits.double()
    if groups > 1 or state['bias'] is not None:
        choice = _scores(wide, case['score'])
        if state['bias'] is not None:
            choice = choice + state['bias'].double()
    else:
        choice = wide                       # scores have the order of their logits
    if groups > 1:
        two = choice.view(tokens, groups, -1).sort(dim=-1, descending=True).values[..., :2].sum(dim=-1)
        best = two.sort(dim=-1, descending=True, stable=True).indices[:, :case['top_groups']]
        kept = torch.zeros(tokens, groups, dtype=torch.bool, device=wide.device).scatter_(1, best, True)
        order = wide if state['bias'] is None else choice
        choice = order.masked_fill(~kept.repeat_interleave(experts // groups, dim=1), -math.inf)
    chosen = choice.sort(dim=-1, descending=True, stable=True).indices[:, :top_k].contiguous()
    s = _scores(logits.float(), case['score'])
    picked = s.gather(1, chosen)
    p = case['norm_p']
    norm = 1.0 if p == 0 else picked.sum(1, keepdim=True) if p == 1 else picked.square().sum(1, keepdim=True).sqrt()
    weights = picked / norm * case['scale']
    total = s.sum(dim=-1, keepdim=True)
    out = [(s / total).to(dtype), weights.to(dtype), chosen]
    if case['train']:
        dw = state['dweights'].float() * case['scale']
        if p == 0:
            dpicked = dw
        else:
            dot = (dw * picked).sum(1, keepdim=True)
            dpicked = dw / norm - dot / norm**2 * (1.0 if p == 1 else picked / norm)
        ds = torch.zeros_like(s).scatter_(1, chosen, dpicked)
        if case['aux']:
            g = state['dscores'].float()
            ds += (g - (g * s).sum(1, keepdim=True) / total) / total
        if case['score'] == 'softmax':
            dlogits = s * (ds - (ds * s).sum(1, keepdim=True))
        else:
            dlogits = ds * s / (1.0 + torch.exp(logits.float()))
        out.append(dlogits.to(dtype))
    return out


def _key_blocks(case, i0, i1):
    """Key positions that the queries ``[i0, i1)`` can see: the first tokens, then the window."""
    lo = max(0, i0 - case['window'] + 1)
    sinks = torch.arange(min(case['sinks'], lo), device='cuda')
    return torch.cat([sinks, torch.arange(lo, i1, device='cuda')])


def _visible(case, rows, keys, length):
    gap = rows[:, None] - keys[None, :]
    seen = (gap >= 0) & ((gap < case['window']) | (keys < case['sinks'])[None, :])
    if length is not None:                  # [batch, 1, rows, keys]
        seen = seen & (rows[:, None] < length.view(-1, 1, 1, 1)) & (keys < length.view(-1, 1, 1, 1))
    return seen


@torch.no_grad()
def _plain_window(state, case):
    """Blocks of queries against the keys that they can see; the backward pass takes the probabilities anew."""
    dtype = _DTYPES[case['dtype']]
    b, s, hq, hk, d = (case[k] for k in ('batch', 'seq', 'heads', 'kv_heads', 'dim'))
    q, k, v = (state[n].detach().float().transpose(1, 2) for n in 'qkv')
    k, v = k.repeat_interleave(hq // hk, dim=1), v.repeat_interleave(hq // hk, dim=1)
    length = state['lengths']
    scale = 1.0 / math.sqrt(d)
    out = torch.empty_like(q)
    step = max(64, min(1024, 2**28 // (b * hq * min(s, case['window'] + 1024))))
    if case['train']:
        dout = state['dout'].float().transpose(1, 2)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i0 in range(0, s, step):
        i1 = min(s, i0 + step)
        keys = _key_blocks(case, i0, i1)
        seen = _visible(case, torch.arange(i0, i1, device='cuda'), keys, length)
        kb, vb = k[:, :, keys], v[:, :, keys]
        score = (q[:, :, i0:i1] @ kb.transpose(2, 3) * scale).masked_fill_(~seen, -math.inf)
        top = score.max(dim=-1, keepdim=True).values
        prob = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
        total = prob.sum(dim=-1, keepdim=True)
        prob = prob / total.masked_fill(total == 0, 1.0)
        o = prob @ vb
        out[:, :, i0:i1] = o
        if case['train']:
            do = dout[:, :, i0:i1]
            if length is not None:          # rows behind a sequence have no gradient
                do = do * (total != 0)
            dv.index_add_(2, keys, prob.transpose(2, 3) @ do)
            dscore = prob * (do @ vb.transpose(2, 3) - (do * o).sum(dim=-1, keepdim=True)) * scale
            dq[:, :, i0:i1] = dscore @ kb
            dk.index_add_(2, keys, dscore.transpose(2, 3) @ q[:, :, i0:i1])
    outs = [out.transpose(1, 2).to(dtype)]
    if case['train']:
        dk, dv = (t.view(b, hk, hq // hk, s, d).sum(dim=2) for t in (dk, dv))
        outs += [t.transpose(1, 2).to(dtype) for t in (dq, dk, dv)]
    return [t.contiguous() for t in outs]


@torch.no_grad()
def _plain_decode(state, case):
    """The visible keys of every sequence are picked out of the cache, then it is one softmax."""
    b, n, hq, hk, d = (case[k] for k in ('batch', 'capacity', 'heads', 'kv_heads', 'dim'))
    length = state['lengths'].long().view(-1, 1)
    first = (length - case['window']).clamp_(min=0)
    keys = first + torch.arange(min(n, case['window']), device='cuda')
    seen = keys < length
    if case['sinks']:
        extra = torch.arange(min(n, case['sinks']), device='cuda').expand(b, -1)
        keys, seen = torch.cat([extra, keys], 1), torch.cat([extra < first, seen], 1)
    keys = keys.clamp(max=n - 1)
    rows = torch.arange(b, device='cuda').view(-1, 1)
    kb = state['k'][rows, keys].float().masked_fill_(~seen.view(b, -1, 1, 1), 0.0)
    vb = state['v'][rows, keys].float().masked_fill_(~seen.view(b, -1, 1, 1), 0.0)
    q = state['q'].float().view(b, hk, hq // hk, d)
    score = (q @ kb.permute(0, 2, 3, 1) / math.sqrt(d)).masked_fill_(~seen.view(b, 1, 1, -1), -math.inf)
    top = score.max(dim=-1, keepdim=True).values
    prob = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = prob.sum(dim=-1, keepdim=True)
    out = prob @ vb.transpose(1, 2) / total.masked_fill(total == 0, 1.0)
    return [out.reshape(b, hq, d).to(_DTYPES[case['dtype']])]


@torch.no_grad()
def _plain_distill(state, case):
    rows, temp, hard = case['rows'], case['temperature'], case['hard']
    z = state['logits'].detach().float()
    ids = state['ids']
    used = (ids >= 0) & (ids < case['vocab'])
    slot = ids.masked_fill(~used, 0)

    def log_softmax(x):
        top = x.max(dim=-1, keepdim=True).values
        return x - (torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True)) + top)

    some = used.any(dim=-1, keepdim=True)
    teacher = (state['values'].float() / temp).masked_fill(~used, -math.inf).masked_fill(~some, 0.0)
    logp = log_softmax(teacher)
    p = torch.exp(logp) * used
    logq = log_softmax(z / temp)
    terms = (p * (logp.masked_fill(~used, 0.0) - logq.gather(1, slot))).masked_fill(~used, 0.0)
    loss = temp**2 * terms.sum(dim=-1)
    grad = temp * (torch.exp(logq) * some - torch.zeros_like(z).scatter_add_(1, slot, p))
    if hard:
        targets = state['targets'].view(-1, 1)
        valid = (targets >= 0) & (targets < case['vocab'])
        target = targets.masked_fill(~valid, 0)
        logs = log_softmax(z)
        loss = loss - hard * (logs.gather(1, target) * valid).squeeze(1)
        grad += hard * (torch.exp(logs) * valid - torch.zeros_like(z).scatter_add_(1, target, valid.float()))
    return [loss.sum() / rows, (grad * (state['dloss'] / rows)).to(_DTYPES[case['dtype']])]


def run(state):
    case = state['case']
    if own:
        return {'route': _own_route, 'window': _own_window, 'decode': _own_decode,
                'distill': _own_distill}[case['kind']](state, case)
    return {'route': _plain_route, 'window': _plain_window, 'decode': _plain_decode,
            'distill': _plain_distill}[case['kind']](state, case)


# ----------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    lengths = _lengths(case) if case['kind'] == 'decode' or case['ragged'] else [case['seq']] * case['batch']
    w, sinks, total = case['window'], case['sinks'], 0
    for n in lengths:
        if case['kind'] == 'decode':
            total += min(n, w) + min(sinks, max(0, n - w))
            continue
        m = min(n, w)
        total += m * (m + 1) // 2 + (n - m) * w
        far = max(0, n - w)                 # query w + t sees min(sinks, t + 1) first tokens besides its window
        total += sum(min(sinks, t + 1) for t in range(min(far, sinks))) + max(0, far - sinks) * sinks
    return total


def work(case):
    kind, size = case['kind'], _SIZE[case['dtype']]
    if kind == 'route':
        t, e, k = case['tokens'], case['experts'], case['top_k']
        moved = 2 * t * e * size + t * k * (size + 8) + (4 * e if case['bias'] else 0)
        flops = t * e * 5
        if case['train']:                   # the logits are still wanted by the backward pass
            moved += t * e * size + t * k * size + (t * e * size if case['aux'] else 0)
            flops += t * e * 5
        return dict(bytes=moved, flops=flops)
    if kind == 'window':
        b, s, hq, hk, d = (case[k] for k in ('batch', 'seq', 'heads', 'kv_heads', 'dim'))
        rows = sum(_lengths(case)) if case['ragged'] else b * s
        moved = (rows * (hq + 2 * hk) + b * s * hq) * d * size
        flops = 4 * _pairs(case) * hq * d
        if case['train']:
            moved += (rows * hq + b * s * (hq + 2 * hk)) * d * size
            flops += 10 * _pairs(case) * hq * d
        return dict(bytes=moved, flops=flops)
    if kind == 'decode':
        b, hq, hk, d = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dim'))
        return dict(bytes=(2 * _pairs(case) * hk + 2 * b * hq) * d * size, flops=4 * _pairs(case) * hq * d)
    rows, vocab, top = case['rows'], case['vocab'], case['top']
    return dict(bytes=2 * rows * vocab * size + rows * top * 12 + rows * 8,
                flops=rows * vocab * (12 if case['hard'] else 6))


# ----------------------------------------------------------------------------
# The definition, in 64 bits
# ----------------------------------------------------------------------------
def _exact_route(state, case):
    x = state['logits'].detach().double().requires_grad_(True)
    experts, groups, top_k = case['experts'], case['groups'], case['top_k']
    s = torch.softmax(x, dim=-1) if case['score'] == 'softmax' else torch.sigmoid(x)
    with torch.no_grad():
        plain = state['bias'] is None
        c = s.detach() if plain else s.detach() + state['bias'].double()
        order = x.detach() if plain else c
        allowed = torch.ones_like(order, dtype=torch.bool)
        if groups > 1:
            per = c.view(-1, groups, experts // groups).clone()
            value = torch.zeros_like(per[..., 0])
            for _ in range(min(2, experts // groups)):
                at = per.argmax(dim=-1, keepdim=True)
                value += per.gather(-1, at).squeeze(-1)
                per.scatter_(-1, at, -math.inf)
            # Rank of a group: those with more, and those with as much and a lower number.
            number = torch.arange(groups, device='cuda')
            more = value[:, None, :] > value[:, :, None]
            same = (value[:, None, :] == value[:, :, None]) & (number[None, :] < number[:, None])
            kept = (more | same).sum(dim=-1) < case['top_groups']
            allowed = kept[:, torch.arange(experts, device='cuda') // (experts // groups)]
        left = order.masked_fill(~allowed, -math.inf)
        picks = []
        number = torch.arange(experts, device='cuda')
        for _ in range(top_k):
            best = left.max(dim=-1, keepdim=True).values
            at = torch.where((left == best) & allowed, number, experts).min(dim=-1, keepdim=True).values
            picks.append(at)
            left = left.scatter(1, at, -math.inf)
            allowed = allowed.scatter(1, at, False)
        chosen = torch.cat(picks, dim=1)
    w = s.gather(1, chosen)
    if case['norm_p']:
        w = w / torch.linalg.vector_norm(w, ord=case['norm_p'], dim=-1, keepdim=True)
    w = w * case['scale']
    probs = s / s.sum(dim=-1, keepdim=True)
    out = [probs.detach(), w.detach(), chosen]
    if case['train']:
        loss = (w * state['dweights'].double()).sum()
        if case['aux']:
            loss = loss + (probs * state['dscores'].double()).sum()
        out.append(torch.autograd.grad(loss, x)[0])
    return out


def _exact_window(state, case):
    b, s, hq, hk, d = (case[k] for k in ('batch', 'seq', 'heads', 'kv_heads', 'dim'))
    lengths = _lengths(case) if case['ragged'] else [s] * b
    outs = [torch.zeros(b, s, h, d, dtype=torch.float64, device='cuda') for h in (hq, hq, hk, hk)]
    for i in range(b):
        n = lengths[i]
        pos = torch.arange(n, device='cuda')
        ago = pos[:, None] - pos[None, :]
        hidden = (ago < 0) | ((ago >= case['window']) & (pos >= case['sinks'])[None, :])
        for h in range(hq):
            g = h * hk // hq
            q = state['q'].detach()[i, :n, h].double()
            k, v = (state[x].detach()[i, :n, g].double() for x in 'kv')
            p = (q @ k.t()).mul_(d**-0.5).masked_fill_(hidden, -math.inf).softmax(dim=-1)
            outs[0][i, :n, h] = p @ v
            if case['train']:
                do = state['dout'][i, :n, h].double()
                outs[3][i, :n, g] += p.t() @ do
                dp = do @ v.t()
                dp -= (dp * p).sum(dim=-1, keepdim=True)
                dp.mul_(p).mul_(d**-0.5)
                outs[1][i, :n, h] = dp @ k
                outs[2][i, :n, g] += dp.t() @ q
    return outs if case['train'] else outs[:1]


def _exact_decode(state, case):
    b, hq, hk, d = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dim'))
    out = torch.zeros(b, hq, d, dtype=torch.float64, device='cuda')
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        lo = max(0, n - case['window'])
        parts = [(0, min(case['sinks'], lo)), (lo, n)]
        k, v = (torch.cat([state[x][i, a:z] for a, z in parts]).double() for x in 'kv')
        for h in range(hq):
            p = torch.softmax(k[:, h * hk // hq] @ state['q'][i, h].double() * d**-0.5, dim=0)
            out[i, h] = p @ v[:, h * hk // hq]
    return [out]


def _exact_distill(state, case):
    rows, vocab, temp, hard = case['rows'], case['vocab'], case['temperature'], case['hard']
    total = torch.zeros((), dtype=torch.float64, device='cuda')
    grads = []
    for r0 in range(0, rows, 512):
        z = state['logits'].detach()[r0:r0 + 512].double().requires_grad_(True)
        ids, values = state['ids'][r0:r0 + 512], state['values'][r0:r0 + 512].double()
        dense = torch.full_like(z, -math.inf, requires_grad=False)
        used = (ids >= 0).nonzero(as_tuple=True)
        dense[used[0], ids[used]] = values[used]
        live = (ids >= 0).any(dim=-1)
        p = torch.softmax(dense[live] / temp, dim=-1)
        logq = torch.log_softmax(z[live] / temp, dim=-1)
        loss = temp**2 * (torch.xlogy(p, p).sum() - (p * logq).sum())
        if hard:
            target = state['targets'][r0:r0 + 512]
            loss = loss + hard * torch.nn.functional.cross_entropy(z, target, ignore_index=-100, reduction='sum')
        loss = loss / rows
        grads.append(torch.autograd.grad(loss, z, state['dloss'].double())[0])
        total += loss.detach()
    return [total, torch.cat(grads)]


def exact(case, seed):
    state = prepare(case, seed)
    return {'route': _exact_route, 'window': _exact_window, 'decode': _exact_decode,
            'distill': _exact_distill}[case['kind']](state, case)


if __name__ == '__main__':      # the cases and a few drawn ones, with what they cost
    picked = random.Random(0)
    for entry in listed() + [dict(draw(picked), name='drawn') for _ in range(12)]:
        print(entry['name'], {k: v for k, v in entry.items() if k != 'name'}, work(entry))

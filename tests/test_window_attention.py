"""Windowed attention with first tokens that stay visible, against its definition in 64 bits."""

import math
import os
import subprocess
import sys

import pytest
import torch
from conftest import DEVICES
from oracle import assert_rounded
from torch.autograd import forward_ad

from megablocks_b200 import ops

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def visible(seq, window, sinks, length, device='cpu'):
    i = torch.arange(seq, device=device)
    gap = i[:, None] - i[None, :]
    seen = (gap >= 0) & ((gap < window) | (i < sinks)[None, :])
    return seen & (i < length)[:, None] & (i < length)[None, :]


def plain(q, k, v, window, sinks, lengths=None, scale=None, dout=None):
    """Output and, with ``dout``, gradients, and for each the sum of the absolute terms that it is made of."""
    b, s, hq, d = q.shape
    hk = k.shape[2]
    window = s if window is None else window
    scale = d**-0.5 if scale is None else scale
    lengths = [s] * b if lengths is None else [max(0, min(s, int(n))) for n in lengths]
    q, k, v = (t.detach().double() for t in (q, k, v))
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    mags = [torch.zeros_like(t) for t in (q, k, v)]
    for x in range(b):
        n = lengths[x]
        seen = visible(n, window, sinks, n, q.device)
        for h in range(hq):
            g = h * hk // hq
            qq, kk, vv = q[x, :n, h], k[x, :n, g], v[x, :n, g]
            p = (qq @ kk.t() * scale).masked_fill(~seen, -math.inf).softmax(-1) if n else qq.new_zeros(0, 0)
            out[x, :n, h], mag[x, :n, h] = p @ vv, p @ vv.abs()
            if dout is not None:
                do = dout[x, :n, h].double()
                dp = do @ vv.t()
                delta = (dp * p).sum(-1, keepdim=True)
                ds = p * (dp - delta) * scale
                # dP and delta come from sums of d terms of 16-bit inputs; |dS| is bounded by their sizes.
                size = p * (do.abs() @ vv.abs().t() + (do.abs() * mag[x, :n, h]).sum(-1, keepdim=True)) * scale
                grads[0][x, :n, h] = ds @ kk
                grads[1][x, :n, g] += ds.t() @ qq
                grads[2][x, :n, g] += p.t() @ do
                mags[0][x, :n, h] = size @ kk.abs()
                mags[1][x, :n, g] += size.t() @ qq.abs()
                mags[2][x, :n, g] += p.t() @ do.abs()
    return (out, mag) if dout is None else (out, mag, grads, mags)


# The forward pass rounds each probability once (half a step of its value), the backward pass P and dS, whose
# delta comes from the rounded output (half a step of its terms): a result is off by at most two half steps of
# the terms' absolute sum, besides its own rounding.  Scores in fp32: |s| <= 64 x 2^-24 x 2 from their sums and
# the exponent's argument, the exponential's unit; 2^-16 of a term, doubled for dS.  fp16 probabilities and dS
# below 2^-14 round to 2^-25 each, times at most 2^8 for the lazily followed maximum's room the other way: 2^-25.
def check(actual, exact, mag, dtype, steps, tiny):
    half = torch.finfo(dtype).eps / 2
    low = 0.0 if dtype != FP16 else 2.0**-25 * tiny
    assert_rounded(actual, exact, 0.0, mag * (steps * half + 2.0**-15) + low)


def inputs(b, s, hq, hk, d, dtype, device, fused=True):
    if fused:
        qkv = torch.randn(b, s, (hq + 2 * hk) * d).to(dtype).to(device)
        q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=-1)
        return q.view(b, s, hq, d), k.view(b, s, hk, d), v.view(b, s, hk, d)
    return [torch.randn(b, s, h, d).to(dtype).to(device) for h in (hq, hk, hk)]


def run(q, k, v, window, sinks, lengths=None, scale=None, dtype=BF16):
    device = q.device
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    dout = torch.randn(q.shape, device=device).to(dtype)
    out = ops.window_attention(q, k, v, window, sinks, lengths, scale)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    grads = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        assert torch.equal(ops.window_attention(q, k, v, window, sinks, lengths, scale), out)
    want, mag, exact, mags = plain(q, k, v, window, sinks, lengths, scale, dout)
    s = q.shape[1]
    reach = min(s, (window or s) + sinks)
    # A term of a sum meets an input of at most ~6; up to `reach` of them (all queries for a first token).
    check(out.detach(), want, mag, dtype, 1, 6 * reach)
    ratio = q.shape[2] // k.shape[2]
    for got, e, m, n in zip(grads, exact, mags, (reach, s * ratio, s * ratio)):
        check(got, e, m, dtype, 2, 6 * n)
    return out, grads


SHAPES = [
    # batch, seq, heads, kv heads, dim, window, sinks
    (1, 1, 1, 1, 8, None, 0),
    (2, 1, 4, 2, 64, 1, 1),
    (1, 2, 2, 1, 32, 1, 0),
    (2, 64, 4, 4, 32, 16, 2),
    (1, 127, 2, 2, 64, 30, 0),
    (1, 128, 2, 1, 128, 128, 4),
    (1, 129, 3, 1, 128, 50, 1),
    (2, 200, 4, 2, 96, None, 0),
    (1, 257, 2, 2, 80, 64, 4),
    (1, 300, 2, 1, 40, 1, 0),
    (1, 511, 8, 1, 64, 100, 130),
    (1, 700, 4, 2, 128, 200, 3),
    (1, 1025, 2, 1, 64, 17, 1),
    (2, 1300, 2, 1, 128, 300, 16),
    (1, 1500, 1, 1, 72, 64, 200),
    (1, 2500, 2, 1, 128, 33, 5),
]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, FP16])
@pytest.mark.parametrize('b,s,hq,hk,d,window,sinks', SHAPES)
def test_kernel_forward_and_backward(dtype, b, s, hq, hk, d, window, sinks):
    run(*inputs(b, s, hq, hk, d, dtype, 'cuda'), window, sinks, dtype=dtype)


@pytest.mark.parametrize('b,s,hq,hk,d,window,sinks', SHAPES[:9])
def test_composed_forward_and_backward(b, s, hq, hk, d, window, sinks):
    run(*inputs(b, s, hq, hk, d, BF16, 'cpu'), window, sinks, dtype=BF16)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16])
@pytest.mark.parametrize('window,sinks', [(40, 3), (None, 0), (300, 150)])
def test_padded_batches(device, dtype, window, sinks):
    """Rows behind a sequence's end may hold anything; they come out as zeros and have no gradient."""
    b, s, hq, hk, d = 7, 330, 4, 2, 64
    q, k, v = (t.clone() for t in inputs(b, s, hq, hk, d, dtype, device, fused=False))
    lengths = torch.tensor([330, 0, 1, 128, 129, 257, 1000], dtype=torch.int32, device=device)
    pad = torch.arange(s, device=device) >= lengths.view(-1, 1)
    out, grads = run(q, k, v, window, sinks, lengths, dtype=dtype)
    assert not out.detach()[pad].any() and not any(g[pad].any() for g in grads)
    # The same with NaN and infinities there, in the upstream gradient too.
    for t, junk in zip((q, k, v), (math.nan, math.inf, math.nan)):
        t[pad] = junk
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    again = ops.window_attention(q, k, v, window, sinks, lengths.long())
    assert torch.equal(again.detach(), out.detach())
    dout = torch.randn(q.shape, device=device).to(dtype)
    junk = dout.clone()
    junk[pad] = math.nan
    clean = torch.autograd.grad(again, (q, k, v), dout, retain_graph=True)
    for a, c in zip(torch.autograd.grad(again, (q, k, v), junk), clean):
        assert torch.equal(a, c) and torch.isfinite(a).all()


@pytest.mark.parametrize('device', DEVICES)
def test_strides_and_scales(device):
    b, s, hq, hk, d = 2, 150, 4, 2, 64
    q = torch.randn(b, hq, s, d, device=device).to(BF16).transpose(1, 2)              # heads before rows
    k = torch.randn(s, b, hk, d, device=device).to(BF16).transpose(0, 1)              # rows before batch
    v = torch.randn(b, s, hk, d + 8, device=device).to(BF16)[..., :d]
    run(q, k, v, 60, 2, scale=0.3)
    k1 = torch.randn(1, s, hk, d, device=device).to(BF16).expand(b, s, hk, d)         # broadcast
    v1 = torch.randn(b, s, hk, d * 2, device=device).to(BF16)[..., ::2]               # not dense
    q1 = torch.randn(b * s * hq * d + 3, device=device).to(BF16)[3:].view(b, s, hq, d)      # misaligned
    run(q1, k1, v1, 60, 2)
    base = torch.randn(1, s, 1, d, device=device).to(BF16).requires_grad_(True)
    out = ops.window_attention(*(base.expand(b, s, h, d) for h in (hq, hk, hk)), 60)
    grad, = torch.autograd.grad(out.float().sum(), base)
    assert grad.shape == base.shape and torch.isfinite(grad).all()


@pytest.mark.parametrize('device', DEVICES)
def test_large_scores(device):
    """Scores whose maximum moves from tile to tile, by more and by less than the lazy reference follows."""
    b, s, h, d = 1, 600, 2, 64
    q, k, v = inputs(b, s, h, h, d, BF16, device, fused=False)
    k = (k * torch.linspace(0.1, 4, s, device=device).view(1, s, 1, 1)).to(BF16)
    run(q, k, v, 500, 4)
    k = k.flip(1).contiguous()
    run(q, k, v, None, 0)


@pytest.mark.parametrize('device', DEVICES)
def test_some_inputs_without_gradient(device):
    q, k, v = inputs(1, 140, 2, 1, 64, BF16, device, fused=False)
    full = [t.detach().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(ops.window_attention(*full, 50, 2).float().square().sum(), full)
    for i in range(3):
        some = [t.detach().requires_grad_(n == i) for n, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(ops.window_attention(*some, 50, 2).float().square().sum(), some[i])
        assert torch.equal(got, want[i])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype,dim', [(FP32, 24), (BF16, 20), (BF16, 160), (torch.float64, 8)])
def test_types_and_head_sizes_of_the_composed_form(device, dtype, dim):
    q, k, v = (torch.randn(2, 33, h, dim, device=device).to(dtype).requires_grad_(True) for h in (4, 2, 2))
    out = ops.window_attention(q, k, v, 9, 2)
    want, mag = plain(q, k, v, 9, 2)
    assert_rounded(out.detach(), want, 0.0, mag * 2.0**-18)
    torch.autograd.grad(out.sum(), (q, k, v))
    cache = [t.detach() for t in (k, v)]
    lengths = torch.tensor([33, 20], device=device)
    got = ops.window_attention_decode(q.detach()[:, 5], *cache, lengths, 9, 2)
    for b, n in enumerate(lengths.tolist()):
        qq = torch.zeros(1, n, 4, dim, dtype=dtype, device=device)
        qq[:, -1] = q.detach()[b, 5]
        want, mag = plain(qq, cache[0][b:b + 1, :n], cache[1][b:b + 1, :n], 9, 2)
        assert_rounded(got[b], want[0, -1], 0.0, mag[0, -1] * 2.0**-18)


def test_gradient_against_differences():
    q, k, v = (torch.randn(1, 7, h, 4, dtype=torch.float64, requires_grad=True) for h in (2, 1, 1))
    assert torch.autograd.gradcheck(lambda *x: ops.window_attention(*x, 3, 1), (q, k, v))


@pytest.mark.gpu
def test_kernel_gradient_against_differences():
    """Directional differences of the 64-bit form: the step's truncation and cancellation stay below 1e-6 of the
    terms, the kernel's rounding is bounded as above."""
    q, k, v = (t.requires_grad_(True) for t in inputs(1, 200, 2, 1, 64, BF16, 'cuda', fused=False))
    dout = torch.randn(q.shape, device='cuda').to(BF16)
    grads = torch.autograd.grad(ops.window_attention(q, k, v, 70, 3), (q, k, v), dout)
    _, _, _, mags = plain(q, k, v, 70, 3, dout=dout)
    half = torch.finfo(BF16).eps / 2
    for n in range(3):
        way = torch.randn([q, k, v][n].shape, device='cuda', dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [t.detach().double() for t in (q, k, v)]
            moved[n] = moved[n] + sign * 1e-5 * way
            ends.append((plain(*moved, 70, 3)[0] * dout.double()).sum())
        want = (ends[0] - ends[1]) / 2e-5
        got = (grads[n].double() * way).sum()
        bound = (way.abs() * (mags[n] * (2 * half + 2.0**-15 + 1e-6) + grads[n].double().abs() * half)).sum()
        assert abs(got - want) <= bound


# ---- decode ---------------------------------------------------------------------------------------------
def check_decode(q, k, v, lengths, window, sinks, scale=None):
    got = ops.window_attention_decode(q, k, v, lengths, window, sinks, scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    capacity = k.shape[1]
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(n, capacity))
        if n == 0:
            assert not got[b].any()
            continue
        lo = max(0, n - (window or capacity))
        pick = list(range(min(sinks, lo))) + list(range(lo, n))
        kk, vv = k[b, pick].double(), v[b, pick].double()
        ratio = q.shape[1] // k.shape[2]
        kk, vv = kk.repeat_interleave(ratio, 1), vv.repeat_interleave(ratio, 1)
        p = torch.softmax(torch.einsum('hd,nhd->hn', q[b].double(), kk) * (scale or q.shape[2]**-0.5), -1)
        check(got[b], torch.einsum('hn,nhd->hd', p, vv), torch.einsum('hn,nhd->hd', p, vv.abs()), q.dtype, 1,
              6 * len(pick))


DECODE = [
    # batch, capacity, heads, kv heads, dim, window, sinks
    (1, 1, 1, 1, 8, None, 0),
    (3, 17, 4, 2, 64, 5, 2),
    (2, 100, 32, 1, 128, None, 0),
    (2, 70, 40, 2, 96, 64, 1),
    (1, 5000, 8, 2, 128, 4096, 4),
    (5, 3000, 4, 4, 80, 700, 16),
    (2, 1500, 12, 12, 64, 33, 1000),
    (64, 300, 8, 8, 32, 100, 4),
]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16])
@pytest.mark.parametrize('b,n,hq,hk,d,window,sinks', DECODE)
def test_decode(device, dtype, b, n, hq, hk, d, window, sinks):
    q = torch.randn(b, hq, d).to(dtype).to(device)
    k, v = (torch.randn(b, n, hk, d).to(dtype).to(device) for _ in range(2))
    for lengths in (torch.full((b,), n), torch.randint(0, n + 1, (b,)), torch.randint(-2, n + 9, (b,))):
        check_decode(q, k, v, lengths.to(torch.int32).to(device), window, sinks)


@pytest.mark.parametrize('device', DEVICES)
def test_decode_does_not_look_behind_the_end_or_out_of_the_window(device):
    b, n, hq, hk, d = 4, 900, 8, 2, 128
    q = torch.randn(b, hq, d, device=device).to(BF16)
    k, v = (torch.randn(b, n, hk, d, device=device).to(BF16) for _ in range(2))
    lengths = torch.tensor([900, 450, 65, 0], device=device)
    want = ops.window_attention_decode(q, k, v, lengths, 200, 3)
    for x, size in enumerate(lengths.tolist()):
        k[x, size:], v[x, size:] = math.nan, math.inf
        k[x, 3:max(3, size - 200)], v[x, 3:max(3, size - 200)] = math.inf, math.nan
    assert torch.equal(ops.window_attention_decode(q, k, v, lengths.int(), 200, 3), want)
    assert torch.isfinite(want).all() and not want[3].any()


@pytest.mark.parametrize('device', DEVICES)
def test_decode_strides(device):
    """Caches with heads before rows, layers in one tensor, and rows that do not start on 16 bytes."""
    b, n, hq, hk, d = 2, 130, 4, 2, 64
    q = torch.randn(b, d, hq, device=device).to(BF16).transpose(1, 2)
    k = torch.randn(b, hk, n, d, device=device).to(BF16).transpose(1, 2)
    v = torch.randn(b, n, 3, hk, d, device=device).to(BF16)[:, :, 1]
    lengths = torch.tensor([130, 77], dtype=torch.int32, device=device)
    check_decode(q, k, v, lengths, 50, 2, scale=0.2)
    check_decode(q, torch.randn(b, n, hk, d + 1, device=device).to(BF16)[..., 1:], v, lengths, 50, 2)


@pytest.mark.gpu
def test_decode_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements a tensor; only its last rows and a sequence's first are visible."""
    b, n, hk, d = 2, 1100000, 8, 128
    k = torch.empty(b, n, hk, d, dtype=BF16, device='cuda')
    v = torch.empty(b, n, hk, d, dtype=BF16, device='cuda')
    for t in (k, v):
        t[:, :8] = torch.randn(b, 8, hk, d, device='cuda').to(BF16)
        t[:, -600:] = torch.randn(b, 600, hk, d, device='cuda').to(BF16)
    q = torch.randn(b, 16, d, device='cuda').to(BF16)
    check_decode(q, k, v, torch.tensor([n, n - 100], dtype=torch.int32, device='cuda'), 500, 8)


@pytest.mark.parametrize('device', DEVICES)
def test_decode_is_the_last_row_of_the_sequence(device):
    q, k, v = inputs(3, 333, 8, 2, 64, BF16, device, fused=False)
    lengths = torch.tensor([333, 200, 1], dtype=torch.int32, device=device)
    whole = ops.window_attention(q, k, v, 100, 4, lengths)
    last = (lengths - 1).long()
    rows = torch.arange(3, device=device)
    got = ops.window_attention_decode(q[rows, last], k, v, lengths, 100, 4)
    half = torch.finfo(BF16).eps / 2
    _, mag = plain(q, k, v, 100, 4, lengths)
    assert ((got.double() - whole[rows, last].double()).abs() <= mag[rows, last] * (4 * half + 2.0**-14) + 1e-30).all()


# ---- use ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    q, k, v = (t.clone().requires_grad_(True) for t in inputs(1, 700, 4, 2, 128, BF16, 'cuda'))
    lengths = torch.tensor([650], dtype=torch.int32, device='cuda')
    dout = torch.randn(1, 700, 4, 128, device='cuda').to(BF16)
    cache = [t.detach() for t in (k, v)]

    def step():
        out = ops.window_attention(q, k, v, 40, 3, lengths)
        one = ops.window_attention_decode(q.detach()[:, 5], *cache, lengths, 40, 3)
        return [out.detach(), one, *torch.autograd.grad(out, (q, k, v), dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(on_side, step()):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    with torch.no_grad():
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        lengths.fill_(512)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(recorded, step()):
        assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, FP16])
@pytest.mark.parametrize('s,d,window,sinks', [(1, 64, 8, 4), (70, 128, 1, 0), (200, 64, 1, 0), (130, 32, 9, 2)])
def test_queries_that_see_one_key_have_no_score_gradient(dtype, s, d, window, sinks):
    q, k, v = (t.requires_grad_(True) for t in inputs(2, s, 4, 2, d, dtype, 'cuda', fused=False))
    out = ops.window_attention(q, k, v, window, sinks)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
    assert not dq[:, 0].any() and dv[:, 0].any(-1).all()       # single numbers of two heads may cancel
    if s == 1 or window == 1:
        assert not dq.any() and not dk.any()
    else:
        assert dq[:, 1:].any(-1).all() and dk[:, 0].any(-1).all()


@pytest.mark.gpu
def test_the_same_in_every_run():
    q, k, v = (t.requires_grad_(True) for t in inputs(2, 1000, 8, 2, 64, BF16, 'cuda', fused=False))
    dout = torch.randn(q.shape, device='cuda').to(BF16)
    first = torch.autograd.grad(ops.window_attention(q, k, v, 64, 4), (q, k, v), dout)
    for _ in range(5):
        for a, c in zip(torch.autograd.grad(ops.window_attention(q, k, v, 64, 4), (q, k, v), dout), first):
            assert torch.equal(a, c)


@pytest.mark.parametrize('device', DEVICES)
def test_empty_batches(device):
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        q = torch.randn(shape, device=device).to(BF16).requires_grad_(True)
        out = ops.window_attention(q, q, q, 3, 1)
        assert out.shape == shape
        out.sum().backward()
    none = torch.zeros(2, 0, 2, 64, device=device, dtype=BF16)
    one = torch.randn(2, 4, 64, device=device).to(BF16)
    got = ops.window_attention_decode(one, none, none, torch.zeros(2, dtype=torch.int32, device=device), 4)
    assert got.shape == one.shape and not got.any()


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    q, k, v = inputs(2, 10, 4, 2, 64, BF16, device, fused=False)
    lengths = torch.tensor([10, 5], dtype=torch.int32, device=device)
    for args, kw in (((q, k, v), dict(window=0)), ((q, k, v), dict(sinks=-1)), ((q, k, v), dict(scale=0.0)),
                     ((q, k, v), dict(scale=math.nan)), ((q, k, v), dict(lengths=lengths[:1])),
                     ((q, k, v), dict(lengths=lengths.float())), ((q, k[:, :9], v[:, :9]), {}), ((q, k, v[:, :9]), {}),
                     ((q[:, :, :3], k, v), {}), ((q, k[..., :32], v[..., :32]), {}), ((q, k.half(), v), {}),
                     ((q[0], k[0], v[0]), {}), ((q.int(), k.int(), v.int()), {})):
        with pytest.raises(ValueError):
            ops.window_attention(*args, **kw)
    one = q[:, 0]
    for args, kw in (((q, k, v, lengths), {}), ((one, k, v, None), {}), ((one, k, v, lengths[:1]), {}),
                     ((one, k, v, lengths), dict(window=0)), ((one, k, v[:, :9], lengths), {}),
                     ((one[:, :3], k, v, lengths), {}), ((one.detach().requires_grad_(True), k, v, lengths), {})):
        with pytest.raises(ValueError):
            ops.window_attention_decode(*args, **kw)


@pytest.mark.gpu
def test_more_sequences_times_heads_than_a_grid_dimension():
    """80000 short sequences of heads: as two halves."""
    q, k, v = (t.requires_grad_(True) for t in inputs(5000, 3, 16, 8, 32, BF16, 'cuda', fused=False))
    dout = torch.randn(q.shape, device='cuda').to(BF16)

    def step(rows):
        out = ops.window_attention(q[rows], k[rows], v[rows], 2, 1)
        return [out, *(g[rows] for g in torch.autograd.grad(out, (q, k, v), dout[rows]))]

    for whole, a, b in zip(step(slice(None)), step(slice(0, 2500)), step(slice(2500, None))):
        assert torch.equal(whole, torch.cat([a, b]))


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(65536, 1, 1, 8), (1, 1 << 22, 1, 8), (1, 1, 65536, 8)])
def test_sizes_that_are_refused(shape):
    q = torch.zeros(shape, dtype=BF16, device='cuda')
    with pytest.raises(ValueError):
        ops.window_attention(q, q, q, 4)


@pytest.mark.gpu
@pytest.mark.parametrize('batch,heads', [(65536, 1), (1, 65536)])
def test_decode_sizes_that_are_refused(batch, heads):
    q = torch.zeros(batch, heads, 8, dtype=BF16, device='cuda')
    k = torch.zeros(batch, 1, 1, 8, dtype=BF16, device='cuda')
    with pytest.raises(ValueError):
        ops.window_attention_decode(q, k, k, torch.ones(batch, dtype=torch.int32, device='cuda'), 4)


@pytest.mark.parametrize('device', DEVICES)
def test_lengths_beyond_32_bits_are_clamped(device):
    q, k, v = inputs(3, 20, 4, 2, 64, BF16, device, fused=False)
    far = torch.tensor([1 << 40, -(1 << 40) + 5, (1 << 32) + 7], device=device)
    near = torch.tensor([20, 0, 20], dtype=torch.int32, device=device)
    assert torch.equal(ops.window_attention(q, k, v, 6, 1, far), ops.window_attention(q, k, v, 6, 1, near))
    one = q[:, 0]
    assert torch.equal(ops.window_attention_decode(one, k, v, far, 6), ops.window_attention_decode(one, k, v, near, 6))


@pytest.mark.gpu
def test_differentiable_once():
    q, k, v = (t.requires_grad_(True) for t in inputs(1, 20, 4, 2, 64, BF16, 'cuda', fused=False))
    out = ops.window_attention(q, k, v, 6, 1)
    first = torch.autograd.grad(out.float().square().sum(), (q, k, v), retain_graph=True)
    again = torch.autograd.grad(out.float().square().sum(), (q, k, v), create_graph=True)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match='differentiable once'):
        again[0].float().sum().backward()


_FIRST_IN_A_GRAPH = """
import sys, torch
sys.path.insert(0, {root!r})
from megablocks_b200 import ops
from megablocks_b200.utils.status import read as read_status
q = torch.randn(1, 40, 2, 64, device='cuda').bfloat16()
fill = torch.full((1 << 20,), -1, dtype=torch.int32, device='cuda')
del fill
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.window_attention(q, q, q, 8, 2)
assert read_status(False) == 0
graph.replay()
assert torch.equal(out, ops.window_attention(q, q, q, 8, 2)) and read_status(False) == 0
"""


@pytest.mark.gpu
def test_the_first_call_of_a_process_may_be_recorded():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, '-c', _FIRST_IN_A_GRAPH.format(root=root)], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# Far queries that are split, where the last part's tiles end with the sequence: with windows that end one row into a
# tile, and others.
FAR = [(1400, 8, 128, 129), (1472, 4, 64, 257), (1153, 4, 64, 1), (2300, 2, 64, 65), (1300, 1, 96, 129), (1408, 2, 128, 130),
       (1472, 1, 64, 256), (2178, 1, 32, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize('ratio,lengths', [(1, None), (2, None), (1, [0, 64, 65])])
@pytest.mark.parametrize('seq,hk,d,window', FAR)
def test_every_far_query_has_a_share_in_the_first_tokens(seq, hk, d, window, ratio, lengths):
    """Gradients that arrive at single queries, those at the end of a stream among them: what the first tokens get
    of each is there once."""
    b = 1 if lengths is None else 3
    if lengths is not None:
        lengths = torch.tensor([seq - n for n in lengths], dtype=torch.int32, device='cuda')
    q, k, v = (t.requires_grad_(True) for t in inputs(b, seq, hk * ratio, hk, d, BF16, 'cuda', fused=False))
    out = ops.window_attention(q, k, v, window, 4, lengths)
    half = torch.finfo(BF16).eps / 2
    for at in (range(seq - 130, seq, 64), range(140, seq, 256)):
        dout = torch.zeros_like(out)
        rows = list(at) + [seq - 1]
        dout[:, rows] = torch.randn(b, len(rows), hk * ratio, d, device='cuda').to(BF16)
        grads = torch.autograd.grad(out, (k, v), dout, retain_graph=True)
        _, _, exact, mags = plain(q, k, v, window, 4, lengths, dout=dout)
        for got, want, mag in zip(grads, exact[1:], mags[1:]):
            assert_rounded(got, want, 0.0, mag * (2 * half + 2.0**-15))
            assert got[0, :4].any(-1).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('requires_grad', [False, True])
def test_forward_mode_tangents(device, requires_grad):
    q, k, v = inputs(2, 30, 4, 2, 64, BF16, device, fused=False)
    ways = [torch.randn_like(t) for t in (q, k, v)]
    lengths = torch.tensor([30, 11], dtype=torch.int32, device=device)
    eps = 1e-6
    ends = [plain(*(t.double() + sign * eps * w.double() for t, w in zip((q, k, v), ways)), 9, 2, lengths)[0]
            for sign in (1, -1)]
    want = (ends[0] - ends[1]) / (2 * eps)
    with forward_ad.dual_level():
        duals = [forward_ad.make_dual(t.requires_grad_(requires_grad), w) for t, w in zip((q, k, v), ways)]
        tangent = forward_ad.unpack_dual(ops.window_attention(*duals, 9, 2, lengths)).tangent
        # fp32 throughout, rounded once; terms of up to 30 x 8 x 6 sum to 2^-12 at most.
        assert_rounded(tangent, want, 0.0, torch.full((), 2.0**-12, dtype=torch.float64, device=device))
    with forward_ad.dual_level(), torch.no_grad():
        last = [t.detach() for t in (q, k, v)]
        q1, w1 = last[0][:, 10].contiguous(), ways[0][:, 10].contiguous()
        only = torch.full((2,), 11, dtype=torch.int32, device=device)
        one = ops.window_attention_decode(forward_ad.make_dual(q1, w1), last[1], last[2], only, 9, 2)
        tangent = forward_ad.unpack_dual(one).tangent
        assert tangent is not None and tangent.any()

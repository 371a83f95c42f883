"""Expert selection against its definition in 64 bits."""

import math

import pytest
import torch
from conftest import DEVICES
from oracle import assert_rounded
from torch.autograd import forward_ad

from megablocks_b200 import ops
from megablocks_b200.ops import select

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32

# Scores in fp32: the argument's rounding (|x - max| <= 32 in the tests that compare tiny scores: 32 x 2^-23),
# the exponential's and the division's two units each, the sums: below 2^-17 of the value altogether; the
# weights' norm and the gradients' sums add as much again.
REL = 2.0**-16


def plain(logits, top_k, score='softmax', bias=None, groups=1, top_groups=None, norm_p=None, scale=1.0):
    """``(scores, weights, ids)`` token by token in 64 bits; differentiable in ``logits``."""
    top_groups = top_groups or groups
    x = logits.double()
    s = torch.sigmoid(x) if score == 'sigmoid' else torch.softmax(x, -1)
    c = s.detach() if bias is None else s.detach() + bias.double()
    ids = []
    size = x.shape[1] // groups
    for t in range(x.shape[0]):
        row = c[t].tolist()
        order = x[t].tolist() if bias is None else row
        value = [sum(sorted(row[g * size:(g + 1) * size], reverse=True)[:2]) for g in range(groups)]
        kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
        left = [e for e in range(x.shape[1]) if e // size in kept]
        ids.append(sorted(left, key=lambda e: (-order[e], e))[:top_k])
    ids = torch.tensor(ids, dtype=torch.int64, device=x.device).view(x.shape[0], top_k)
    w = s.gather(1, ids)
    if norm_p:
        w = w / torch.linalg.vector_norm(w, ord=norm_p, dim=-1, keepdim=True)
    return s / s.sum(-1, keepdim=True), w * scale, ids


def both(logits, **how):
    how = {k: v for k, v in how.items() if v is not None}
    cpu = {k: v.cpu() if torch.is_tensor(v) else v for k, v in how.items()}
    return ops.select_experts(logits, **how), plain(logits.detach().cpu(), **cpu)


CASES = [
    # tokens, experts, top_k, score, biased, groups, top_groups, norm_p, scale
    (1, 1, 1, 'softmax', False, 1, 1, 1, 1.0),
    (1, 256, 8, 'sigmoid', True, 8, 4, 1, 2.5),
    (33, 64, 4, 'softmax', False, 1, 1, None, 1.0),
    (130, 60, 4, 'softmax', True, 1, 1, 1, 1.0),
    (65, 37, 37 - 6, 'sigmoid', True, 1, 1, 2, 1.0),
    (64, 96, 6, 'softmax', False, 6, 2, 1, 1.0),
    (50, 72, 3, 'sigmoid', True, 24, 3, 1, 0.5),
    (40, 8, 8, 'softmax', True, 8, 8, 2, 1.0),
    (40, 32, 2, 'sigmoid', False, 32, 2, None, 1.0),
    (70, 300, 12, 'softmax', True, 3, 2, 1, 1.0),
    (20, 512, 8, 'sigmoid', True, 8, 2, 1, 2.5),
    (20, 1024, 32, 'softmax', True, 32, 5, 1, 1.0),
    (20, 1023, 32, 'sigmoid', False, 1, 1, 1, 1.0),
    (9, 32, 32, 'sigmoid', True, 1, 1, 1, 1.0),
    (33, 250, 9, 'softmax', True, 5, 2, 2, 1.0),
    (33, 192, 6, 'sigmoid', True, 12, 3, 1, 1.0),
]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('tokens,experts,top_k,score,biased,groups,top_groups,norm_p,scale', CASES)
def test_forward_and_backward(device, dtype, tokens, experts, top_k, score, biased, groups, top_groups, norm_p, scale):
    logits = (torch.randn(tokens, experts) * 1.5).to(dtype).to(device).requires_grad_(True)
    bias = (torch.randn(experts) * 0.1).to(device) if biased else None
    how = dict(top_k=top_k, score=score, groups=groups, top_groups=top_groups, norm_p=norm_p, scale=scale)
    scores, weights, ids = ops.select_experts(logits, bias=bias, **how)
    assert scores.dtype == weights.dtype == dtype and ids.dtype == torch.int64
    wide = logits.detach().double().cpu().requires_grad_(True)
    want = plain(wide, bias=None if bias is None else bias.cpu(), **how)
    assert torch.equal(ids.cpu(), want[2])
    assert_rounded(scores, want[0], REL)
    assert_rounded(weights, want[1], REL)

    dweights, dscores = torch.randn(tokens, top_k).to(dtype), torch.randn(tokens, experts).to(dtype)
    # A gradient is a sum of terms that cancel: its error is REL of the terms.  None is larger than what the
    # weights' gradients give, |dw| scale (1 / norm + 1 / norm^2 ...) s <= 2 sum|dw| scale (divided or not:
    # s / norm <= 1, s <= 1), and the scores', 2 max|g| s / total <= 2 max|g|.
    unit = 2 * scale * dweights.double().abs().sum(1, keepdim=True)
    for use_w, use_s in ((True, False), (True, True), (False, True)):
        terms, total, bound = [], 0, 0.0
        if use_w:
            terms.append((weights, dweights))
            total = total + (want[1] * dweights.double()).sum()
            bound = bound + unit
        if use_s:
            terms.append((scores, dscores))
            total = total + (want[0] * dscores.double()).sum()
            bound = bound + 2 * dscores.double().abs().amax(1, keepdim=True)
        got, = torch.autograd.grad([a for a, _ in terms], logits, [g.to(device) for _, g in terms], retain_graph=True)
        exact, = torch.autograd.grad(total, wide, retain_graph=True)
        assert_rounded(got, exact, REL, (REL * bound).expand_as(exact).to(device))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('groups,top_groups', [(1, 1), (8, 3)])
def test_order_beyond_32_bits(device, score, groups, top_groups):
    """The bias lifts every score to nearly the same value: only 64 bits tell the experts apart."""
    logits = torch.randn(64, 64, device=device)
    s = torch.sigmoid(logits[0].double()) if score == 'sigmoid' else torch.softmax(logits[0].double(), -1)
    bias = (0.75 - s).float()
    logits = logits[:1].repeat(64, 1)
    logits[1:] += torch.randn(63, 1, device=device) * 1e-6
    got, want = both(logits, top_k=6, score=score, bias=bias, groups=groups, top_groups=top_groups, norm_p=1)
    assert torch.equal(got[2].cpu(), want[2])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('experts,top_k', [(24, 5), (64, 32), (200, 8), (256, 32), (700, 32)])
def test_neighbouring_values(device, experts, top_k):
    """fp32 logits, and scores with a bias, that differ in their last bits or not at all."""
    base = torch.rand(60, 1, device=device) + 0.5
    logits = (base.view(torch.int32) + torch.randint(0, 12, (60, experts), device=device, dtype=torch.int32)).view(FP32)
    for groups, top_groups in ((1, 1), (4, 4), (4, 2)):
        got, want = both(logits, top_k=min(top_k, experts // 2), groups=groups, top_groups=top_groups)
        assert torch.equal(got[2].cpu(), want[2])
    bias = torch.zeros(experts, device=device)
    bias[::3] = 2.0**-24
    got, want = both(logits, top_k=top_k, bias=bias, score='sigmoid')
    assert torch.equal(got[2].cpu(), want[2])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,groups,top_groups', [(256, 8, 4), (60, 5, 2), (700, 1, 1)])
def test_some_close_values_among_others(device, score, experts, groups, top_groups):
    """A few of the chosen experts, of those behind them and of the groups are as good as equal, the others not."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(300, experts, generator=gen)
    order = logits.argsort(dim=-1, descending=True)
    for first, count in ((1, 2), (4, 5)):               # of six: the second and third; the fifth to the ninth
        at = order[:, first:first + count]
        near = logits.gather(1, at[:, :1]).expand(-1, count).contiguous().view(torch.int32)
        logits.scatter_(1, at, (near + torch.randint(0, 3, near.shape, generator=gen, dtype=torch.int32)).view(FP32))
    logits = logits.to(device)
    bias = torch.randint(0, 3, (experts,), generator=gen).to(device) * 2.0**-26
    for b in (None, bias):
        got, want = both(logits, top_k=6, score=score, bias=b, groups=groups, top_groups=top_groups, norm_p=1)
        assert torch.equal(got[2].cpu(), want[2])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('bias', [None, 0.0, 0.25])
@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_ties_go_to_the_lowest_id(device, score, bias, dtype):
    logits = torch.randint(-2, 3, (200, 48)).to(dtype).to(device)
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    b = None if bias is None else torch.full((48,), bias, device=device)
    for groups, top_groups in ((1, 1), (4, 2)):
        got, want = both(logits, top_k=8, score=score, bias=b, groups=groups, top_groups=top_groups, norm_p=1)
        assert torch.equal(got[2].cpu(), want[2])
    assert got[2][0].tolist() == list(range(8))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_masked_experts_and_empty_rows(device, dtype):
    low = torch.finfo(dtype).min
    logits = torch.randn(6, 40).to(dtype).to(device)
    logits[0, 3:] = -math.inf           # three experts left for four places
    logits[1, 5:] = low
    logits[2] = -math.inf               # none
    logits[3] = low                     # all alike
    logits.requires_grad_(True)
    scores, weights, ids = ops.select_experts(logits, 4, norm_p=1)
    assert set(ids[0, :3].tolist()) == {0, 1, 2} and ids[0, 3].item() == 3
    assert weights[0, 3].item() == 0
    assert set(ids[1].tolist()) <= set(range(5))
    assert ids[2].tolist() == [0, 1, 2, 3] and not scores[2].any() and not weights[2].any()
    assert ids[3].tolist() == [0, 1, 2, 3]
    assert_rounded(scores[3], torch.full((40,), 1 / 40, dtype=torch.float64), REL)
    rows = [0, 1, 4, 5]
    want = plain(logits.detach().cpu()[rows], 4, norm_p=1)
    assert_rounded(scores[rows], want[0], REL)
    assert_rounded(weights[rows], want[1], REL)
    grad, = torch.autograd.grad([scores, weights], logits, [torch.ones_like(scores), torch.ones_like(weights)])
    assert torch.isfinite(grad).all() and not grad[2].any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('biased', [False, True])
def test_nan_and_inf_give_valid_distinct_ids(device, score, biased):
    logits = torch.randn(8, 64, device=device)
    logits[0, 5] = math.nan
    logits[1] = math.nan
    logits[2, 7] = math.inf
    logits[3, 9] = -math.inf
    bias = torch.randn(64, device=device) * 0.1 if biased else None
    scores, weights, ids = ops.select_experts(logits, 8, score=score, bias=bias, groups=8, top_groups=4, norm_p=1)
    assert ((ids >= 0) & (ids < 64)).all()
    assert all(len(set(row)) == 8 for row in ids.tolist())
    assert weights[1].isnan().all() and torch.isfinite(weights[3:]).all()
    assert scores[0].isnan().any() and torch.isfinite(scores[3:]).all()


@pytest.mark.parametrize('device', DEVICES)
def test_the_bias_chooses_but_does_not_weigh(device):
    logits = torch.zeros(5, 8, device=device, requires_grad=True)
    bias = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.3, 0.2, 0.1], device=device, requires_grad=True)
    scores, weights, ids = ops.select_experts(logits, 3, score='sigmoid', bias=bias, norm_p=1)
    assert ids.tolist() == [[5, 6, 7]] * 5
    torch.testing.assert_close(weights, torch.full((5, 3), 1 / 3, device=device))
    assert weights.requires_grad and torch.autograd.grad(weights.sum(), bias, allow_unused=True)[0] is None


@pytest.mark.parametrize('device', DEVICES)
def test_broadcast_gradients_strides_and_empty_batches(device):
    wide = torch.randn(40, 128, device=device, dtype=BF16)
    view = wide[:, 1:61].requires_grad_(True)           # rows that are neither dense nor aligned
    dense = view.detach().clone().requires_grad_(True)
    row = torch.randn(1, 60, device=device).to(BF16)
    grads = []
    for x, g in ((view, row.expand(40, 60)), (dense, row.expand(40, 60).contiguous())):
        scores, weights, _ = ops.select_experts(x, 4, score='sigmoid', norm_p=1)
        grads.append(torch.autograd.grad([scores, weights], x, [g, torch.ones_like(weights)])[0])
    assert torch.equal(*grads)
    got = ops.select_experts(torch.empty(0, 16, device=device, requires_grad=True), 2)
    assert [tuple(t.shape) for t in got] == [(0, 16), (0, 2), (0, 2)]
    got[1].sum().backward()


def test_gradient_against_differences():
    logits = torch.randn(5, 12, dtype=torch.float64, requires_grad=True)
    for score in ('softmax', 'sigmoid'):
        for norm_p in (None, 1, 2):
            how = dict(score=score, groups=3, top_groups=2, norm_p=norm_p, scale=2.0)
            assert torch.autograd.gradcheck(lambda x: ops.select_experts(x, 3, **how)[:2], logits)


@pytest.mark.gpu
def test_kernel_gradient_against_differences():
    """Central differences of the 64-bit form, whose truncation (step^2 / 6 of the third derivative, below 6 for
    these sums of bounded functions) and cancellation (2^-52 / step) are below 1e-8 of the terms."""
    logits = torch.randn(4, 24, device='cuda', requires_grad=True)
    probe = torch.randn(4, 5, device='cuda')
    how = dict(top_k=5, score='sigmoid', groups=4, top_groups=2, norm_p=1)
    _, weights, _ = ops.select_experts(logits, **how)
    got, = torch.autograd.grad(weights, logits, probe)
    base = logits.detach().double().cpu()
    want = torch.zeros_like(base)
    for i in range(base.numel()):
        step = torch.zeros(base.numel(), dtype=torch.float64)
        step[i] = 1e-5
        hi, lo = ((plain(base + sign * step.view_as(base), **how)[1] * probe.cpu()).sum() for sign in (1, -1))
        want.view(-1)[i] = (hi - lo) / 2e-5
    unit = 2 * probe.double().abs().sum(1, keepdim=True)
    assert_rounded(got, want, REL, (unit * (REL + 1e-8)).expand_as(want).cuda())


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    logits = torch.randn(100, 256, device='cuda', dtype=BF16, requires_grad=True)
    bias = torch.randn(256, device='cuda') * 0.1
    how = dict(score='sigmoid', groups=8, top_groups=4, norm_p=1, scale=2.5)
    dw = torch.randn(100, 8, device='cuda', dtype=BF16)

    def step():
        scores, weights, ids = ops.select_experts(logits, 8, bias=bias, **how)
        return [scores.detach(), weights.detach(), ids, *torch.autograd.grad(weights, logits, dw)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    with torch.no_grad():
        logits.copy_(torch.randn_like(logits))
        bias.copy_(torch.randn_like(bias) * 0.1)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(recorded, step()):
        assert torch.equal(a, b)
    assert not torch.equal(on_side[2], recorded[2])


@pytest.mark.gpu
def test_many_tokens():
    """More tokens than a grid has blocks in one wave, against the composed form on the same device."""
    logits = (torch.randn(70001, 256, device='cuda') + torch.randn(1, 256, device='cuda')).to(BF16)
    bias = torch.randn(256, device='cuda') * 0.05
    how = dict(score='sigmoid', bias=bias, groups=8, top_groups=4, norm_p=1, scale=2.5)
    got = ops.select_experts(logits, 8, **how)
    want = select._composed(logits.double(), 8, how['score'], bias, 8, 4, 1, 2.5)
    assert torch.equal(got[2], want[2])
    assert_rounded(got[0], want[0], REL)
    assert_rounded(got[1], want[1], REL)


@pytest.mark.parametrize('device', DEVICES)
def test_bias_update(device):
    bias = torch.zeros(6, device=device)
    load = torch.tensor([10, 20, 30, 20, 20, 20], dtype=torch.int32, device=device)
    assert ops.update_expert_bias(bias, load, 0.5) is bias
    assert bias.tolist() == [0.5, 0.0, -0.5, 0.0, 0.0, 0.0]
    bias.zero_()
    ops.update_expert_bias(bias, torch.tensor([1, 1, 2, 1, 1, 1], device=device), 0.25)      # mean 7 / 6
    assert bias.tolist() == [0.25, 0.25, -0.25, 0.25, 0.25, 0.25]
    with pytest.raises(ValueError):
        ops.update_expert_bias(bias, load[:5], 0.5)


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    logits = torch.randn(4, 16, device=device)
    bad = [dict(top_k=0), dict(top_k=17), dict(top_k=2, score='tanh'), dict(top_k=2, groups=3),
           dict(top_k=2, groups=0), dict(top_k=9, groups=4, top_groups=2), dict(top_k=2, groups=4, top_groups=5),
           dict(top_k=2, norm_p=3), dict(top_k=2, bias=torch.zeros(15, device=device)),
           dict(top_k=2, bias=torch.zeros(16, device=device, dtype=BF16))]
    for how in bad:
        with pytest.raises(ValueError):
            ops.select_experts(logits, **how)
    for x, k in ((logits.view(2, 2, 16), 2), (logits.to(torch.int32), 2), (torch.randn(2, 1025, device=device), 2),
                 (torch.randn(2, 64, device=device), 33), (torch.randn(2, 0, device=device), 1)):
        with pytest.raises(ValueError):
            ops.select_experts(x, k)


@pytest.mark.gpu
def test_differentiable_once():
    logits = torch.randn(9, 16, device='cuda', requires_grad=True)
    scores, weights, _ = ops.select_experts(logits, 3, score='sigmoid', norm_p=1)
    loss = scores.square().sum() + weights.square().sum()
    first, = torch.autograd.grad(loss, logits, retain_graph=True)
    again, = torch.autograd.grad(loss, logits, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError, match='differentiable once'):
        again.sum().backward()


def banned(experts, groups, which):
    """Biases that take experts out: single ones, 8 consecutive ones, whole groups, all but one or two of a group."""
    size = experts // groups
    bias = torch.randn(experts, generator=torch.Generator().manual_seed(11)) * 0.05
    if which == 'one':
        bias[size // 2] = bias[-1] = -math.inf
    elif which == 'eight':
        bias[:min(8, size)] = -math.inf
        bias[size * (groups // 2):][:min(8, size)] = -math.inf
    elif which == 'group':
        bias[size:2 * size] = -math.inf
    elif which == 'groups':
        for g in range(0, groups, 3):
            bias[g * size:(g + 1) * size] = -math.inf
    elif which == 'most':
        bias[1:size] = -math.inf                # one is left: the sum of the two largest is -inf
        bias[size + 2:2 * size] = -math.inf     # two
    elif which == 'preferred':
        bias[size * (groups - 1)] = math.inf
    return bias


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,groups,top_groups,top_k', [(256, 8, 4, 8), (256, 8, 1, 4), (64, 8, 3, 6), (128, 4, 2, 8),
                                                             (60, 5, 2, 4), (512, 8, 4, 8), (96, 1, 1, 6)])
@pytest.mark.parametrize('which', ['one', 'eight', 'group', 'groups', 'most', 'preferred'])
def test_banned_and_preferred_experts(device, dtype, score, experts, groups, top_groups, top_k, which):
    if groups == 1 and which != 'one':
        which = 'eight' if which == 'eight' else 'preferred'
    bias = banned(experts, groups, which).to(device)
    logits = torch.randn(120, experts).to(dtype).to(device)
    got, want = both(logits, top_k=top_k, score=score, bias=bias, groups=groups, top_groups=top_groups, norm_p=1)
    assert torch.equal(got[2].cpu(), want[2])
    assert_rounded(got[1], want[1], REL)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('experts,groups,top_groups', [(256, 8, 4), (60, 5, 2), (512, 8, 4)])
@pytest.mark.parametrize('size', [30.0, 1e3, 1e4, 1e6])
def test_large_biases_of_both_signs(device, experts, groups, top_groups, size):
    """A group's two largest values nearly cancel: what a key leaves out of them is more than their sum."""
    bias = torch.full((experts,), -size, device=device)
    bias[::experts // groups] = size
    logits = torch.randn(2000, experts, device=device)
    got, want = both(logits, top_k=4, score='sigmoid', bias=bias, groups=groups, top_groups=top_groups)
    assert torch.equal(got[2].cpu(), want[2])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('experts,groups', [(256, 8), (16, 8), (60, 5), (1024, 32)])
def test_a_preferred_expert_among_banned_ones(device, experts, groups):
    """Its group is worth +inf - inf, which counts as +inf, as often as there is one: the lowest ids stay."""
    size = experts // groups
    logits = torch.randn(50, experts, device=device)
    logits[7] = math.nan
    bias = torch.randn(experts, device=device) * 0.1
    want = []
    for g in range(1, groups, 2):
        bias[g * size:(g + 1) * size] = -math.inf
        bias[(g + 1) * size - 1] = math.inf
        want.append((g + 1) * size - 1)
    for top_groups in range(1, len(want) + 1):
        for score in ('softmax', 'sigmoid'):
            _, _, ids = ops.select_experts(logits, top_groups, score=score, bias=bias, groups=groups, top_groups=top_groups)
            rows = torch.arange(50) != 7
            assert (ids.cpu()[rows] == torch.tensor(want[:top_groups])).all()
            assert len(set(ids[7].tolist())) == top_groups
    bias[0] = math.inf                          # its group's second is finite: worth +inf as well
    ids = ops.select_experts(logits, 2, bias=bias, groups=groups, top_groups=2)[2]
    assert (ids.cpu()[rows] == torch.tensor([0, want[0]])).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_forward_mode_tangents(device, requires_grad, score):
    logits = torch.randn(7, 16, device=device)
    way = torch.randn_like(logits)
    how = dict(top_k=3, score=score, norm_p=1, scale=2.0, bias=torch.randn(16, device=device) * 0.1)
    wide = logits.double()
    eps = 1e-6
    ends = [plain(wide + sign * eps * way, **how) for sign in (1, -1)]
    with forward_ad.dual_level():
        got = ops.select_experts(forward_ad.make_dual(logits.requires_grad_(requires_grad), way), **how)
        for i in range(2):
            tangent = forward_ad.unpack_dual(got[i]).tangent
            # Truncation and cancellation of the differences below 1e-9, sums of fp32 terms below 2.
            torch.testing.assert_close(tangent.double(), (ends[0][i] - ends[1][i]) / (2 * eps), rtol=0, atol=2.0**-18)
    got, tangents = torch.func.jvp(lambda x: ops.select_experts(x, **how)[1], (logits.detach(),), (way,))
    torch.testing.assert_close(tangents.double(), (ends[0][1] - ends[1][1]) / (2 * eps), rtol=0, atol=2.0**-18)

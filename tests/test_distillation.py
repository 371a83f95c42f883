"""Distillation from a teacher's top logits against its definition in 64 bits."""

import math
import threading

import pytest
import torch
from conftest import DEVICES
from oracle import assert_rounded
from torch.autograd import forward_ad

from megablocks_b200.ops import fused

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32

# Probabilities in fp32: differences from the maximum are exact for 16-bit logits and rounded once for fp32
# ones, |z - max| / T <= 48 in these tests, so the exponent is off by 48 x 2^-23, the exponential's unit and
# its square by 2^-21, sums and quotients by less: 2^-17 of the value.  A gradient subtracts such terms.
REL = 2.0**-17


def plain(logits, values, ids, temperature=1.0, targets=None, hard_weight=0.0):
    """Mean loss, row by row in 64 bits; differentiable in ``logits``."""
    z = logits.double()
    total = z.new_zeros(())
    for r in range(z.shape[0]):
        used = [i for i in range(ids.shape[1]) if 0 <= ids[r, i] < z.shape[1]]
        if used:
            p = torch.softmax(values[r, used].double() / temperature, 0)
            logq = torch.log_softmax(z[r] / temperature, 0)[ids[r, used].long()]
            total = total + temperature**2 * torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum()
        if targets is not None and 0 <= targets[r] < z.shape[1]:
            total = total + hard_weight * (torch.logsumexp(z[r], 0) - z[r, targets[r]])
    return total / z.shape[0]


def batch(rows, vocab, top, dtype, device, value_dtype=FP32, id_dtype=torch.int64):
    logits = (torch.randn(rows, vocab) * 2).to(dtype)
    values = (torch.randn(rows, top) * 2 + 4).to(value_dtype)
    ids = torch.stack([torch.randperm(vocab)[:top] for _ in range(rows)])
    for r in range(rows):               # some rows keep fewer, some none
        if r % 3 == 1:
            ids[r, top // 2:] = -1
        if r % 7 == 5:
            ids[r] = -1
    targets = torch.randint(0, vocab, (rows,))
    targets[::4] = -100
    targets[1::4] = ids[1::4, 0]        # also among the teacher's
    return logits.to(device), values.to(device), ids.to(id_dtype).to(device), targets.to(device)


def check(logits, values, ids, temperature, targets, hard_weight, factor=1.0, loss_fn=fused.distillation_loss):
    logits = logits.detach().requires_grad_(True)
    before = logits.detach().clone()
    loss = loss_fn(logits, values, ids, temperature, targets, hard_weight)
    assert loss.dim() == 0
    got, = torch.autograd.grad(loss * factor, logits)
    assert torch.equal(logits, before)
    wide = logits.detach().double().cpu().requires_grad_(True)
    t = None if targets is None else targets.cpu()
    want = plain(wide, values.cpu(), ids.cpu(), temperature, t, hard_weight)
    exact, = torch.autograd.grad(want * factor, wide)
    # The loss is a mean of logs of size <= 32 each, taken to 2^-17 at most, times T^2 + hard.
    torch.testing.assert_close(loss.double().cpu(), want.detach(), rtol=2.0**-17,
                               atol=(temperature**2 + hard_weight) * 32 * 2.0**-17)
    # Terms of a gradient: T p, T q, hard softmax, hard: none larger than (T + hard) factor / rows.  An
    # incoming factor other than one is a second rounding (the gradient is kept unscaled, but for fp16).
    unit = (temperature + hard_weight) * abs(factor) / logits.shape[0]
    again = 0.0 if factor == 1.0 or logits.dtype == FP16 else torch.finfo(logits.dtype).eps / 2
    assert_rounded(got, exact, REL + again, torch.full((), 4 * REL * unit, dtype=torch.float64, device=got.device))
    return got


SIZES = [(1, 1, 1), (3, 7, 3), (9, 130, 5), (17, 1000, 32), (8, 4099, 64), (5, 8192, 1024 // 8), (4, 51200, 64),
         (3, 50257, 20)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('rows,vocab,top', SIZES)
@pytest.mark.parametrize('temperature,hard', [(1.0, 0.0), (2.0, 0.5), (3.0, 1.0)])
def test_loss_and_gradient(device, dtype, rows, vocab, top, temperature, hard):
    logits, values, ids, targets = batch(rows, vocab, top, dtype, device)
    check(logits, values, ids, temperature, targets if hard else None, hard, 1024.0 if dtype == FP16 else 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,vocab', [(BF16, 102400), (BF16, 102401), (BF16, 131072), (FP32, 51200), (FP32, 51203),
                                         (FP16, 131001)])
def test_rows_around_and_beyond_shared_memory(dtype, vocab):
    logits, values, ids, targets = batch(3, vocab, 40, dtype, 'cuda')
    check(logits, values, ids, 4.0, targets, 0.5, 1024.0 if dtype == FP16 else 1.0)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('value_dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('id_dtype', [torch.int32, torch.int64])
def test_types_of_the_teacher(device, value_dtype, id_dtype):
    logits, values, ids, targets = batch(12, 515, 9, BF16, device, value_dtype, id_dtype)
    check(logits, values, ids, 2.0, targets, 0.25)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_incoming_gradient_and_a_second_backward_pass(device, dtype):
    logits, values, ids, targets = batch(10, 300, 6, dtype, device)
    check(logits, values, ids, 2.0, targets, 0.5, factor=-3.5 * (512 if dtype == FP16 else 1))
    logits.requires_grad_(True)
    loss = fused.distillation_loss(logits, values, ids, 2.0) * 512.0
    first, = torch.autograd.grad(loss, logits, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, logits)
    assert torch.equal(first, kept)
    half = torch.finfo(dtype).eps / 2
    assert_rounded(second, first.double(), 2 * half + 4 * REL, 16 * REL * 2.0 * 512 / 10)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_columns_named_twice_and_ids_out_of_range(device, dtype):
    logits, values, ids, targets = batch(8, 100, 12, dtype, device)
    ids[:, 3] = ids[:, 0]
    ids[:, 7] = ids[:, 0]
    ids[2, 5] = 100
    ids[3, 5] = 2**31 - 1
    ids[4, 5] = -2**31
    targets[5] = 100
    check(logits, values, ids, 1.0, targets, 0.5)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_rows_that_teach_nothing(device, dtype):
    """Padding may hold anything: no loss, a gradient of zero."""
    logits, values, ids, targets = batch(6, 200, 4, dtype, device)
    ids[:4] = -1
    targets[:4] = -100
    logits[0] = math.nan
    logits[1] = math.inf
    logits[2] = torch.finfo(dtype).max
    values[0] = math.nan
    values[3] = -math.inf
    logits.requires_grad_(True)
    loss = fused.distillation_loss(logits, values, ids, 2.0, targets, 0.5)
    assert torch.isfinite(loss)
    got, = torch.autograd.grad(loss, logits)
    assert not got[:4].any() and got[4].any() and torch.isfinite(got).all()
    want = plain(logits.detach().cpu()[4:], values.cpu()[4:], ids.cpu()[4:], 2.0, targets.cpu()[4:], 0.5) * 2 / 6
    torch.testing.assert_close(loss.detach().double().cpu(), want, rtol=2.0**-16, atol=4.5 * 32 * 2.0**-17)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_masked_columns_and_masked_teacher_slots(device, dtype):
    logits, values, ids, targets = batch(6, 64, 5, dtype, device)
    for r in range(6):
        free = [c for c in range(64) if c not in ids[r].tolist() and c != int(targets[r])]
        logits[r, free[:20]] = -math.inf            # a padded vocabulary
        logits[r, free[20:30]] = torch.finfo(dtype).min
    values[:, 2] = -math.inf                        # a masked slot whose id is still valid
    values[1, 1] = torch.finfo(FP32).min
    got = check(logits, values, ids, 1.0, targets, 0.5)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('vocab', [40, 3001])
@pytest.mark.parametrize('temperature,hard', [(1.0, 0.0), (1.0, 0.5), (0.5, 0.5), (3.0, 0.0)])
def test_rows_masked_by_the_lowest_value(device, dtype, vocab, temperature, hard):
    """All of a row, all but the columns that are named, and long stretches."""
    logits, values, ids, targets = batch(5, vocab, 5, dtype, device)
    low = torch.finfo(dtype).min
    logits[0] = low
    for r, columns in ((1, range(vocab)), (2, range(vocab // 2)), (3, range(vocab // 3, vocab))):
        logits[r, [c for c in columns if c not in ids[r].tolist() and c != int(targets[r])]] = low
    got = check(logits, values, ids, temperature, targets, hard)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize('device', DEVICES)
def test_logits_far_from_zero(device):
    """A constant on all logits changes nothing, also where it is large."""
    logits, values, ids, targets = batch(6, 500, 8, FP32, device)
    logits = (logits * 64).round() / 64             # exact with the offset on
    near = check(logits, values, ids, 3.0, targets, 0.5)
    far = check(logits + 4096.0, values, ids, 3.0, targets, 0.5)
    torch.testing.assert_close(near, far, rtol=2.0**-18, atol=2.0**-18 / 6)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('offset', [0, 1])
def test_misaligned_and_strided_logits(device, dtype, offset):
    store = torch.randn(9 * 333 + 8, device=device).to(dtype)
    logits = store[offset:offset + 9 * 333].view(9, 333)
    _, values, ids, targets = batch(9, 333, 7, dtype, device)
    check(logits, values, ids, 2.0, targets, 0.5, 64.0 if dtype == FP16 else 1.0)
    wide = torch.randn(9, 400, device=device).to(dtype)
    check(wide[:, 3:336], values, ids, 2.0, targets, 0.5, 64.0 if dtype == FP16 else 1.0)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
def test_linear_head(device, dtype):
    rows, vocab, h = 24, 260, 64
    _, values, ids, targets = batch(rows, vocab, 6, dtype, device)
    hidden = (torch.randn(rows, h) / 4).to(dtype).to(device).requires_grad_(True)
    weight = (torch.randn(vocab, h) / 4).to(dtype).to(device).requires_grad_(True)
    factor = 64.0
    loss = fused.linear_distillation_loss(hidden, weight, values, ids, 2.0, targets, 0.5)
    dh, dw = torch.autograd.grad(loss * factor, (hidden, weight))
    hw, ww = (t.detach().double().cpu().requires_grad_(True) for t in (hidden, weight))
    want = plain(hw @ ww.t(), values.cpu(), ids.cpu(), 2.0, targets.cpu(), 0.5)
    eh, ew = torch.autograd.grad(want * factor, (hw, ww))
    eps = torch.finfo(dtype).eps
    # Logits (|z| < 4) round to half a step (a change of q of as much), their gradient (<= 2.5 factor / rows a term) to
    # another, and the products sum 260 or 24 of them with weights of size ~1/4 (max ~1).
    unit = (2 + 0.5) * factor / rows
    per = unit * (4 * eps + eps) + 2.0**-20 * unit
    torch.testing.assert_close(loss.double().cpu(), want.detach(), rtol=2**-14, atol=(4 + 0.5) * 8 * eps + 2.0**-10 * eps)
    assert_rounded(dh, eh, 2 * eps, 2 * per + 2.0**-18)
    assert_rounded(dw, ew, 2 * eps, rows * per + 2.0**-18)
    with torch.no_grad():
        alone = fused.linear_distillation_loss(hidden, weight, values, ids, 2.0, targets, 0.5)
    torch.testing.assert_close(alone, loss.detach(), rtol=2**-20, atol=2**-20)


@pytest.mark.parametrize('device', DEVICES)
def test_without_gradient_and_without_rows(device):
    logits, values, ids, targets = batch(5, 90, 4, BF16, device)
    want = plain(logits.cpu(), values.cpu(), ids.cpu(), 2.0)
    loss = fused.distillation_loss(logits, values, ids, 2.0)
    assert not loss.requires_grad
    torch.testing.assert_close(loss.double().cpu(), want, rtol=2.0**-16, atol=2.0**-12)
    none = torch.empty(0, 90, device=device, requires_grad=True)
    loss = fused.distillation_loss(none, values[:0], ids[:0])
    loss.backward()
    assert loss.item() == 0 and none.grad.shape == (0, 90)


def test_gradient_against_differences():
    logits = torch.randn(4, 15, dtype=torch.float64, requires_grad=True)
    _, values, ids, targets = batch(4, 15, 5, FP32, 'cpu')
    assert torch.autograd.gradcheck(
        lambda z: fused.distillation_loss(z, values.double(), ids, 2.0, targets, 0.5), logits)


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    logits, values, ids, targets = batch(33, 1000, 16, BF16, 'cuda')
    logits.requires_grad_(True)

    def step():
        loss = fused.distillation_loss(logits, values, ids, 2.0, targets, 0.5)
        return [loss.detach(), *torch.autograd.grad(loss * 2.0, logits)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    with torch.no_grad():
        logits.copy_(torch.randn_like(logits))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(recorded, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    logits, values, ids, targets = batch(4, 50, 3, BF16, device)
    good = dict(logits=logits, teacher_logits=values, teacher_ids=ids)
    fused.distillation_loss(**good)
    bad = [dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(hard_weight=-0.5),
           dict(hard_weight=0.5), dict(hard_weight=0.5, targets=targets[:3]),
           dict(hard_weight=0.5, targets=targets.int()), dict(teacher_ids=ids[:, :2]), dict(teacher_ids=ids.float()),
           dict(teacher_logits=values[:3], teacher_ids=ids[:3]), dict(teacher_logits=ids),
           dict(teacher_logits=values[:, :0], teacher_ids=ids[:, :0]), dict(logits=logits.view(2, 2, 50)),
           dict(logits=logits.int()), dict(teacher_logits=torch.zeros(4, 1025, device=device),
                                           teacher_ids=torch.zeros(4, 1025, device=device, dtype=torch.int64))]
    for change in bad:
        with pytest.raises(ValueError):
            fused.distillation_loss(**{**good, **change})


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16])
def test_differentiable_once(dtype):
    logits = torch.randn(9, 300, device='cuda').to(dtype).requires_grad_(True)
    values, ids = torch.randn(9, 4, device='cuda'), torch.randint(0, 300, (9, 4), device='cuda')
    again, = torch.autograd.grad(fused.distillation_loss(logits, values, ids), logits, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        again.sum().backward()
    hidden = torch.randn(9, 64, device='cuda', requires_grad=True)
    weight = torch.randn(300, 64, device='cuda')
    again, = torch.autograd.grad(fused.linear_distillation_loss(hidden, weight, values, ids), hidden, create_graph=True)
    with pytest.raises(RuntimeError):
        again.sum().backward()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('vocab', [90, 131072])
@pytest.mark.parametrize('value_dtype', [BF16, FP32])
def test_a_teacher_of_nan_shows(device, dtype, vocab, value_dtype):
    """One, some or all values of a row: the loss is NaN, and the row's gradient, and no other row's."""
    logits, values, ids, _ = batch(6, vocab, 3, dtype, device, value_dtype)
    ids[:] = torch.arange(18, device=device).view(6, 3)
    ids[5] = -1
    values[1] = math.nan
    values[2, 1] = math.nan
    values[3] = math.nan
    values[5] = math.nan                            # unused
    ids[3, 1:] = -1                                 # a single slot
    for hard, targets in ((0.0, None), (0.5, torch.full((6,), 5, device=device))):
        logits = logits.detach().requires_grad_(True)
        loss = fused.distillation_loss(logits, values, ids, 2.0, targets, hard)
        assert loss.isnan()
        got, = torch.autograd.grad(loss, logits)
        assert got[1:4].isnan().all() and torch.isfinite(got[[0, 4, 5]]).all()
        with torch.no_grad():
            assert fused.distillation_loss(logits, values, ids, 2.0, targets, hard).isnan()
    one, _, _, _ = batch(1, vocab, 1, dtype, device)
    assert fused.distillation_loss(one, values[1:2, :1], ids[1:2, :1]).isnan()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('value_dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('temperature', [0.25, 0.5, 1.0, 3.0])
def test_teacher_values_at_the_ends_of_their_type(device, value_dtype, temperature):
    """Slots that are masked by the lowest value, all of a row's too, and a row of the largest."""
    logits, values, ids, _ = batch(6, 200, 4, BF16, device, value_dtype)
    ids[:] = torch.arange(24, device=device).view(6, 4)
    values[0] = torch.finfo(value_dtype).min
    values[1, 1:] = torch.finfo(value_dtype).min
    values[2] = torch.finfo(value_dtype).max
    values[3, 2] = torch.finfo(value_dtype).max
    got = check(logits, values, ids, temperature, None, 0.0)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('requires_grad', [False, True])
def test_forward_mode_tangents(device, requires_grad):
    logits, values, ids, targets = batch(6, 50, 4, FP32, device)
    way = torch.randn_like(logits)
    eps = 1e-6
    ends = [plain(logits.double().cpu() + sign * eps * way.double().cpu(), values.cpu(), ids.cpu(), 2.0, targets.cpu(), 0.5)
            for sign in (1, -1)]
    want = (ends[0] - ends[1]) / (2 * eps)
    with forward_ad.dual_level():
        loss = fused.distillation_loss(forward_ad.make_dual(logits.requires_grad_(requires_grad), way), values, ids, 2.0,
                                       targets, 0.5)
        # A mean over six rows of at most (T + hard) 2 max|way|, in fp32.
        torch.testing.assert_close(forward_ad.unpack_dual(loss).tangent.double().cpu(), want, rtol=0, atol=2.0**-16)
    hidden, weight = torch.randn(6, 8, device=device), torch.randn(50, 8, device=device)
    way = torch.randn_like(weight)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(weight.requires_grad_(requires_grad), way)
        got = forward_ad.unpack_dual(fused.linear_distillation_loss(hidden, dual, values, ids, 2.0)).tangent
        logits = forward_ad.make_dual(hidden @ weight.detach().t(), hidden @ way.t())
        want = forward_ad.unpack_dual(fused.distillation_loss(logits, values, ids, 2.0)).tangent
        torch.testing.assert_close(got, want)


@pytest.mark.gpu
def test_long_and_short_rows_in_one_recording_and_in_two_threads():
    """A call with shorter rows, or with fewer slots, leaves the shared memory that one with longer rows has asked for."""
    sizes = [(7, 100000, 40), (7, 30000, 8), (7, 60000, 64), (7, 500, 4)]
    calls = [batch(rows, vocab, top, BF16, 'cuda') for rows, vocab, top in sizes]

    def one(call):
        logits, values, ids, targets = call
        logits = logits.detach().requires_grad_(True)
        loss = fused.distillation_loss(logits, values, ids, 2.0, targets, 0.5)
        return loss.detach(), torch.autograd.grad(loss, logits)[0]

    want = [one(c) for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [one(c) for c in calls]
    one(calls[3])
    graph.replay()
    torch.cuda.synchronize()
    for got, exact in zip(recorded, want):
        assert all(torch.equal(a, b) for a, b in zip(got, exact))

    wrong = []

    def loop(call, exact):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got = one(call)
                torch.cuda.current_stream().synchronize()
                wrong.extend(n for n, (a, b) in enumerate(zip(got, exact)) if not torch.equal(a, b))
        except RuntimeError as e:
            wrong.append(e)

    threads = [threading.Thread(target=loop, args=x) for x in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

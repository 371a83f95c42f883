"""Expert selection, windowed attention, distillation and decoding as a model uses them together."""

import dataclasses
import math
import os
import subprocess
import sys
import weakref

import pytest
import torch
from conftest import DEVICES

from megablocks_b200 import Arguments, MoE, dMoE
from megablocks_b200.layers import router as router_lib
from megablocks_b200.models.transformer import MoETransformer, Teacher, preset
from megablocks_b200.ops import select_experts, update_expert_bias
from megablocks_b200.train import Trainer, TrainerConfig

OPTIONS = dict(moe_router_score='sigmoid', moe_router_bias=True, moe_router_groups=2, moe_router_top_groups=1,
               moe_router_scale=1.5, attention_window=9, attention_sinks=2, moe_num_experts=8, moe_loss_weight=0.0)


def build(device, name='tiny-mixtral', **options):
    dtype = torch.bfloat16 if device == 'cuda' else torch.float32
    torch.manual_seed(7)
    model = MoETransformer(preset(name, device=torch.device(device), dtype=dtype, **{**OPTIONS, **options}))
    return model


def teacher_for(cfg, batch, seq, device, top=5, hard=0.5):
    logits = torch.randn(batch, seq, top, device=device) * 2
    ids = torch.randint(0, cfg.vocab_size, (batch, seq, top), device=device, dtype=torch.int32)
    ids[:, -3:] = -1                    # a padded tail
    return Teacher(logits, ids, temperature=2.0, hard_weight=hard)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('layer', [dMoE, MoE])
@pytest.mark.parametrize('norm', [None, 1])
def test_layer_routes_by_select_experts(device, layer, norm):
    args = Arguments(hidden_size=128, ffn_hidden_size=256, moe_num_experts=16, moe_top_k=3, moe_capacity_factor=8,
                     moe_router_score='sigmoid', moe_router_bias=True, moe_router_groups=4, moe_router_top_groups=2,
                     moe_router_scale=2.5, moe_normalize_expert_weights=norm, moe_loss_weight=0.1, bias=False,
                     fp16=False, bf16=device == 'cuda', device=torch.device(device))
    moe = layer(args).train()
    moe.router.expert_bias.copy_(torch.randn(16) * 0.1)
    x = torch.randn(40, 1, 128, device=device, dtype=moe.router.layer.weight.dtype, requires_grad=True)
    scores, weights, experts = moe.router(x)
    logits = moe.router.layer(x.reshape(-1, 128))
    want = select_experts(logits, 3, score='sigmoid', bias=moe.router.expert_bias, groups=4, top_groups=2,
                          norm_p=norm, scale=2.5)
    for a, b in zip((scores, weights, experts), want):
        assert torch.equal(a, b)
    out = moe(x)
    out = out[0] if isinstance(out, tuple) else out
    assert torch.equal(moe.router.expert_load, moe.experts.last_tokens_per_expert.long())
    assert int(moe.router.expert_load.sum()) == 120
    out.float().square().sum().backward()
    assert torch.isfinite(moe.router.layer.weight.grad).all() and moe.router.layer.weight.grad.any()
    moe.eval()(x)
    assert int(moe.router.expert_load.sum()) == 120        # only training counts


def test_default_router_is_as_it_was():
    args = Arguments(hidden_size=64, moe_num_experts=8, moe_top_k=2, fp16=False, device=torch.device('cpu'))
    router = router_lib.LearnedRouter(args)
    assert list(router.state_dict()) == ['layer.weight'] and not router._selects
    for bad in (dict(moe_router_score='tanh'), dict(moe_router_groups=3), dict(moe_router_groups=0),
                dict(moe_router_groups=2, moe_router_top_groups=3), dict(moe_router_top_groups=0)):
        with pytest.raises(ValueError):
            Arguments(moe_num_experts=8, **bad)


def test_bias_keeps_32_bits_and_is_saved():
    args = Arguments(hidden_size=64, moe_num_experts=8, moe_top_k=2, fp16=False, device=torch.device('cpu'),
                     moe_router_bias=True)
    router = router_lib.LearnedRouter(args).bfloat16()
    assert router.layer.weight.dtype == torch.bfloat16 and router.expert_bias.dtype == torch.float32
    assert sorted(router.state_dict()) == ['expert_bias', 'layer.weight']
    router.count_load(torch.tensor([8, 0, 4, 4, 4, 4, 4, 4], dtype=torch.int32))
    other = router_lib.LearnedRouter(Arguments(hidden_size=64, moe_num_experts=4, moe_top_k=2, fp16=False,
                                               device=torch.device('cpu'), moe_router_bias=True))
    other.count_load(torch.tensor([1, 2, 3, 2]))
    router_lib.balance_routers([router, other], 0.25)
    assert router.expert_bias.tolist() == [-0.25, 0.25, 0, 0, 0, 0, 0, 0]
    assert other.expert_bias.tolist() == [0.25, 0, -0.25, 0]
    assert not router.expert_load.any() and not other.expert_load.any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name', ['tiny', 'tiny-mixtral'])
def test_a_distilled_step(device, name):
    """Forward, backward and update with everything on: gradients arrive everywhere, biases move against the load."""
    model = build(device, name)
    cfg = model.cfg
    trainer = Trainer(model, TrainerConfig(lr=1e-3, total_steps=10, router_bias_rate=0.01, grad_accum_steps=2))
    tokens = torch.randint(0, cfg.vocab_size, (4, 33), device=device)
    teacher = teacher_for(cfg, 4, 32, device)
    before = [r.expert_bias.clone() for r in trainer._routers]
    loss = trainer.step(tokens[:, :-1], tokens[:, 1:], teacher=teacher)
    assert torch.isfinite(loss) and loss.dim() == 0
    for p in model.parameters():
        assert p.grad is None or torch.isfinite(p.grad).all()
    for old, router in zip(before, trainer._routers):
        moved = router.expert_bias - old
        assert moved.any() and not router.expert_load.any()
        assert all(abs(abs(v) - 0.01) < 1e-7 or v == 0 for v in moved.tolist())
    loss = trainer.step(tokens[:, :-1], tokens[:, 1:])          # and an ordinary step
    assert torch.isfinite(loss)


def test_distillation_gradient_of_a_model_against_differences():
    """fp32 on the CPU: the directional derivative of the total loss along the parameters of head, attention and
    norms.  Central differences: cancellation 2^-23 x loss / step, truncation step^2; step 2^-6 of a unit
    direction leaves both below 1e-3 of a gradient of size one."""
    model = build('cpu', moe_router_bias=False)
    with torch.no_grad():       # experts chosen by a wide margin: the choice does not flip within the step
        for block in model.blocks:
            block.moe.router.layer.weight.mul_(0)
    tokens = torch.randint(0, 512, (2, 20))
    teacher = teacher_for(model.cfg, 2, 20, 'cpu')
    params = [p for n, p in model.named_parameters() if 'attn' in n or 'ln' in n or 'lm_head' in n]
    total, _ = model.distillation_loss(tokens, teacher, tokens.roll(-1, 1))
    grads = torch.autograd.grad(total, params)
    way = [torch.randn_like(p) for p in params]
    norm = math.sqrt(sum(float(w.square().sum()) for w in way))
    way = [w / norm for w in way]
    want = sum(float((g * w).double().sum()) for g, w in zip(grads, way))
    size = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    ends = []
    for sign in (1, -1):
        with torch.no_grad():
            for p, w in zip(params, way):
                p.add_(w, alpha=sign * 2.0**-6)
            ends.append(float(model.distillation_loss(tokens, teacher, tokens.roll(-1, 1))[0].double()))
            for p, w in zip(params, way):
                p.sub_(w, alpha=sign * 2.0**-6)
    assert abs((ends[0] - ends[1]) / 2.0**-5 - want) <= 2e-3 * (1 + size)


def fixed_choice(model):
    """Every token takes the same experts, whatever its rounding: decoding and the whole sequence agree."""
    with torch.no_grad():
        for block in model.blocks:
            block.moe.router.layer.weight.zero_()
            block.moe.router.expert_bias.copy_(torch.linspace(0.5, -0.5, model.cfg.moe_num_experts))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name', ['tiny', 'tiny-mixtral'])
@pytest.mark.parametrize('window,sinks', [(9, 2), (None, 0), (1, 0)])
def test_decoding_agrees_with_the_whole_sequence(device, name, window, sinks):
    """Logits of a prompt and of each token decoded behind it against one pass over the whole sequence.

    On the CPU in fp32 the two differ by sums of another order.  In bf16 each of the two layers rounds some ten
    tensors by half a step, which norms pass on at about their size: twice 2 x 10 x 2^-8 of the largest logit.  A
    token in a wrong place, or a key too many or too few, moves logits by their own size."""
    model = build(device, name, attention_window=window, attention_sinks=sinks).eval()
    fixed_choice(model)
    batch, prompt, extra = 3, 21, 8
    tokens = torch.randint(0, 512, (batch, prompt + extra), device=device)
    lengths = torch.tensor([prompt, 13, 1], dtype=torch.int32, device=device)
    cache = model.new_cache(batch, prompt + extra)
    got = [model.prefill(tokens[:, :prompt], cache, lengths)]
    for i in range(extra - 1):
        step = tokens[torch.arange(batch), (lengths + i).long()]
        got.append(model.decode(step, cache))
    assert cache.lengths.tolist() == [n + extra - 1 for n in lengths.tolist()]
    with torch.no_grad():
        for b, n in enumerate(lengths.tolist()):
            whole = model(tokens[b:b + 1, :n + extra - 1])[0].float()
            size = whole.abs().max()
            for i in range(extra):
                bound = size * (2.0**-12 if device == 'cpu' else 40 * 2.0**-8)
                assert (got[i][b].float() - whole[n - 1 + i]).abs().max() <= bound


@pytest.mark.parametrize('device', DEVICES)
def test_generate_and_refusals(device):
    model = build(device, 'tiny').eval()
    tokens = torch.randint(0, 512, (2, 6), device=device)
    out = model.generate(tokens, 5, torch.tensor([6, 2], device=device))
    assert out.shape == (2, 5) and ((out >= 0) & (out < 512)).all()
    with pytest.raises(ValueError):
        model.generate(tokens, 0)
    with pytest.raises(ValueError):
        model.new_cache(2, 65)                  # the model has 64 positions
    cache = model.new_cache(2, 7)
    with pytest.raises(ValueError):
        model.decode(tokens[:, 0], cache)       # nothing in it yet
    with pytest.raises(ValueError):
        model.prefill(tokens.repeat(1, 2), cache)
    with pytest.raises(ValueError):
        model.prefill(tokens[:1], cache)
    model.prefill(tokens, cache)
    model.decode(tokens[:, 0], cache)
    with pytest.raises(ValueError):
        model.decode(tokens[:, 0], cache)       # full
    with pytest.raises(ValueError):
        model.distillation_loss(tokens, Teacher(torch.zeros(2, 5, 3, device=device),
                                                torch.zeros(2, 5, 3, device=device, dtype=torch.int64)))


@pytest.mark.parametrize('device', DEVICES)
def test_answering_leaves_a_training_model_as_it_was(device):
    model = build(device, 'tiny', moe_loss_weight=0.1).train()
    frozen = model.blocks[0].ln1.eval()
    tokens = torch.randint(0, 512, (2, 6), device=device)
    first = model.generate(tokens, 3)
    assert model.training and model.blocks[0].moe.training and not frozen.training
    assert all(not b.moe.router.expert_load.any() for b in model.blocks)
    total, _ = model.loss(tokens, tokens.roll(-1, 1))       # no stale auxiliary losses
    total.backward()
    assert torch.equal(model.eval().generate(tokens, 3), first)


@pytest.mark.gpu
@pytest.mark.parametrize('name', ['tiny', 'tiny-mixtral'])
def test_recorded_decoding(name):
    """Replays go on from where the cache is, and past its end they stay inside it."""
    model = build('cuda', name).eval()
    tokens = torch.randint(0, 512, (3, 6), device='cuda')
    lengths = torch.tensor([6, 2, 4], device='cuda')
    new = torch.randint(0, 512, (4, 3), device='cuda')
    eager = model.new_cache(3, 10)
    model.prefill(tokens, eager, lengths)
    want = [model.decode(t, eager) for t in new]
    cache = model.new_cache(3, 10)
    model.prefill(tokens, cache, lengths)
    got = [model.decode(new[0], cache)]
    static, graph = new[1].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.decode(static, cache)
    for t in new[1:]:
        static.copy_(t)
        graph.replay()
        got.append(out.clone())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert cache.lengths.tolist() == eager.lengths.tolist() == [10, 6, 8]
    for _ in range(6):
        graph.replay()
    assert torch.isfinite(out).all() and cache.lengths.tolist() == [10, 10, 10]


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [False, True])
def test_recorded_step_counts_and_balances_like_the_eager_one(graph, monkeypatch):
    """Every step's loads are that step's tokens, and the biases are the rule's.  (The two runs are not compared with one
    another: a few atomics of the backward pass, whose order varies, move a token to another expert in time.)"""
    model = build('cuda', 'tiny')
    trainer = Trainer(model, TrainerConfig(lr=1e-3, total_steps=20, router_bias_rate=0.01, cuda_graph=graph,
                                           graph_warmup_steps=2))
    loads, balance = [], router_lib.balance_routers

    def listen(routers, *args):
        loads.append(torch.stack([r.expert_load for r in routers]))
        balance(routers, *args)

    monkeypatch.setattr(router_lib, 'balance_routers', listen)
    gen = torch.Generator(device='cuda').manual_seed(3)
    want = torch.zeros_like(torch.stack([r.expert_bias for r in trainer._routers]))
    for i in range(6):
        tokens = torch.randint(0, 512, (4, 65), device='cuda', generator=gen)
        trainer.step(tokens[:, :-1], tokens[:, 1:])
        assert len(loads) == i + 1 and (loads[i].sum(dim=1) == 4 * 64 * model.cfg.moe_top_k).all()
        for bias, load in zip(want, loads[i]):
            update_expert_bias(bias, load, 0.01)
    assert (trainer._graph is not None) == graph
    assert torch.equal(torch.stack([r.expert_bias for r in trainer._routers]), want) and want.any()
    assert not torch.equal(loads[4], loads[5])


@pytest.mark.gpu
def test_recorded_and_distilled_steps_in_turn():
    """A distilled step between recorded ones has its own place in the schedule, and those behind it theirs."""
    runs = []
    for graph in (False, True):
        model = build('cuda', 'tiny')
        trainer = Trainer(model, TrainerConfig(lr=1e-2, total_steps=12, cuda_graph=graph, graph_warmup_steps=2))
        gen = torch.Generator(device='cuda').manual_seed(3)
        torch.manual_seed(5)
        teacher = teacher_for(model.cfg, 4, 64, 'cuda')
        rates = []
        for i in range(10):
            tokens = torch.randint(0, 512, (4, 65), device='cuda', generator=gen)
            trainer.step(tokens[:, :-1], tokens[:, 1:], teacher=teacher if i == 4 else None)
            rates.append(trainer.dense_opt.lr)
        assert (trainer._graph is not None) == graph and trainer.step_count == 10
        if graph:
            assert int(trainer._graph_step) == 10
            assert torch.equal(trainer._hyper, trainer._table[9]) and float(trainer._hyper[0]) == pytest.approx(rates[-1])
        runs.append(rates)
    assert runs[0] == runs[1]


_RANK = '''
import sys, torch, torch.distributed as dist
sys.path.insert(0, {root!r})
from megablocks_b200 import Arguments
from megablocks_b200.layers import router as R
rank = int(sys.argv[1])
dist.init_process_group('gloo', init_method='tcp://127.0.0.1:{port}', rank=rank, world_size=2)
r = R.LearnedRouter(Arguments(hidden_size=8, moe_num_experts=4, moe_top_k=1, fp16=False, moe_router_bias=True,
                              device=torch.device('cpu')))
r.count_load(torch.tensor([[4, 0, 2, 2], [0, 1, 3, 4]][rank]))      # together 4, 1, 5, 6: mean 4
R.balance_routers([r], 0.5, dist.group.WORLD)
assert r.expert_bias.tolist() == [0.0, 0.5, -0.5, -0.5], r.expert_bias
dist.destroy_process_group()
'''


def test_ranks_sum_their_loads():
    import socket
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = _RANK.format(root=root, port=port)
    procs = [subprocess.Popen([sys.executable, '-c', code, str(r)]) for r in range(2)]
    assert [p.wait(timeout=120) for p in procs] == [0, 0]


def test_command_line():
    from megablocks_b200 import train
    if torch.cuda.is_available():
        pytest.skip('the CPU run of the command')
    loss = train.main(['--preset', 'tiny', '--steps', '2', '--micro-batch', '2', '--router-score', 'sigmoid',
                       '--router-groups', '2', '--router-top-groups', '1', '--router-bias-rate', '0.01',
                       '--loss-weight', '0', '--attention-window', '16', '--attention-sinks', '2'])
    assert torch.isfinite(loss)


@pytest.mark.parametrize('cast', [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to(torch.bfloat16).float(), lambda m: torch.nn.Sequential(m).bfloat16()[0]])
def test_a_cast_leaves_the_bias_as_it_was(cast):
    args = Arguments(hidden_size=64, moe_num_experts=4, moe_top_k=2, fp16=False, device=torch.device('cpu'),
                     moe_router_bias=True)
    router = router_lib.LearnedRouter(args)
    bias = torch.tensor([0.1234567, 1.001, -0.3333, 2.0005])
    router.expert_bias.copy_(bias)
    router = cast(router)
    assert router.expert_bias.dtype == torch.float32 and torch.equal(router.expert_bias, bias)
    assert torch.equal(router.state_dict()['expert_bias'], bias)


@pytest.mark.parametrize('device', DEVICES)
def test_rotary_tables_stay_where_they_are(device):
    """Longer sequences and caches bring longer tables; those that a recording may read are not freed or moved."""
    model = build(device, 'tiny-mixtral').eval()
    tokens = torch.randint(0, 512, (1, 300), device=device)
    whole = build(device, 'tiny-mixtral').eval()(tokens)
    want = model(tokens[:, :64])
    first = model._rope_for(64, tokens.device)
    places = [(t.data_ptr(), weakref.ref(t.untyped_storage())) for t in first]
    kept = [t.clone() for t in first]
    del first
    model.new_cache(1, 200)
    ready = sum(map(len, model._ropes.values()))
    for n in (65, 100, 200):                    # what a cache needs is there before the first call on it
        model._rope_for(n, tokens.device)
    assert sum(map(len, model._ropes.values())) == ready
    assert torch.equal(model(tokens), whole)
    for n in range(201, 1200):
        model._rope_for(n, tokens.device)
    assert sum(map(len, model._ropes.values())) <= 6        # they at least double
    storages = [t.untyped_storage() for tables in model._ropes.values() for pair in tables for t in pair]
    for (place, storage), table in zip(places, kept):
        assert storage() is not None and place in [s.data_ptr() for s in storages]
        assert any(torch.equal(t[:64], table) and t.data_ptr() == place
                   for tables in model._ropes.values() for pair in tables for t in pair)
    assert torch.equal(model(tokens[:, :64]), want)


@pytest.mark.gpu
def test_recorded_calls_and_longer_tables():
    """A recorded pass and a recorded decode call give the same after the tables grew and memory was used again; a pass
    whose tables are made while it is recorded leaves none that are not filled."""
    model = build('cuda', 'tiny-mixtral', attention_window=None, attention_sinks=0).eval()
    fixed_choice(model)
    tokens = torch.randint(0, 512, (1, 300), device='cuda')
    cache, spare = model.new_cache(1, 40), model.new_cache(1, 40)
    with torch.no_grad():
        model.prefill(tokens[:, :30], cache)
        model.prefill(tokens[:, :30], spare)
        model.decode(tokens[:, 30], spare)                      # warm
        want = model.decode(tokens[:, 31], spare)
        whole = model(tokens[:, :64])
        decode, forward, late = (torch.cuda.CUDAGraph() for _ in range(3))
        static = tokens[:, 30].clone()
        with torch.cuda.graph(decode):
            out = model.decode(static, cache)
        with torch.cuda.graph(forward):
            logits = model(tokens[:, :64])
        with torch.cuda.graph(late):
            long = model(tokens)                                # longer than any table so far
        assert all(len(pairs) == 1 for pairs in model._ropes.values())
        eager = model(tokens)
        model.new_cache(1, 2000)
        junk = [torch.full((n,), float('nan'), device='cuda') for n in (1024, 4096, 8192, 65536) for _ in range(32)]
        del junk
        decode.replay()
        static.copy_(tokens[:, 31])
        decode.replay()
        forward.replay()
        late.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(logits, whole) and torch.equal(long, eager)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name', ['tiny', 'tiny-mixtral'])
def test_answers_in_inference_mode_and_training_behind_them(device, name):
    model = build(device, name)
    tokens = torch.randint(0, 512, (2, 8), device=device)
    want = model.generate(tokens, 4)
    model = build(device, name)                 # without tables
    with torch.inference_mode():
        assert torch.equal(model.generate(tokens, 4), want)
        cache = model.new_cache(2, 12)
        first = model.prefill(tokens, cache).argmax(dim=-1)
    assert torch.equal(model.decode(first.clone(), cache).argmax(dim=-1), want[:, 1])
    total, _ = model.train().loss(tokens, tokens.roll(-1, 1))
    total.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)


@pytest.mark.parametrize('device', DEVICES)
def test_answers_that_fill_the_positions(device):
    """The last token is not fed back: a prompt and all answers but one need a place."""
    model = build(device, 'tiny').eval()                    # 64 positions
    tokens = torch.randint(0, 512, (2, 60), device=device)
    assert model.generate(tokens, 5).shape == (2, 5)
    assert torch.equal(model.generate(tokens, 5)[:, :3], model.generate(tokens, 3))
    with pytest.raises(ValueError):
        model.generate(tokens, 6)
    full = torch.randint(0, 512, (2, 64), device=device)
    assert model.generate(full, 1).shape == (2, 1)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name', ['tiny', 'tiny-mixtral'])
@pytest.mark.parametrize('window', [9, None])
def test_answering_under_autocast(device, name, window):
    """A model of 32 bits fills its cache from keys of 16 and goes on from it."""
    torch.manual_seed(7)
    model = MoETransformer(preset(name, device=torch.device(device), dtype=torch.float32, mlp_impl='sparse',
                                  **{**OPTIONS, 'attention_window': window}))
    fixed_choice(model)
    tokens = torch.randint(0, 512, (2, 12), device=device)
    with torch.autocast(device, torch.bfloat16):
        cache = model.new_cache(2, 12)
        got = [model.prefill(tokens[:, :8], cache)]
        got += [model.decode(tokens[:, i], cache) for i in range(8, 12)]
        whole = model.eval()(tokens).float()
    for i, logits in enumerate(got):
        assert (logits.float() - whole[:, 7 + i]).abs().max() <= whole.abs().max() * 40 * 2.0**-8


def test_positional_arguments_keep_their_places():
    """What stood before the selection's options is given in the same places as without them."""
    names = [f.name for f in dataclasses.fields(Arguments)]
    old = [n for n in names if not n.startswith('moe_router_')]
    assert names[:len(old)] == old
    values = [getattr(Arguments(moe_num_experts=4), n) for n in old]
    values[old.index('ep_fused_comm')] = False
    values[old.index('ep_inflight_microbatches')] = 3
    args = Arguments(*values)
    assert args.ep_fused_comm is False and args.ep_inflight_microbatches == 3 and args.moe_router_score == 'softmax'


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('change', [dict(moe_router_scale=3.0), dict(moe_router_score='sigmoid'),
                                    dict(moe_router_groups=4, moe_router_top_groups=1)])
def test_options_replaced_on_a_router_are_used(device, change):
    how = dict(hidden_size=64, moe_num_experts=16, moe_top_k=2, fp16=False, device=torch.device(device))
    router = router_lib.LearnedRouter(Arguments(**how))
    x = torch.randn(9, 64, device=device)
    plain = router(x)[1]
    router.args = Arguments(**how, **change)
    logits = router.layer(x)
    want = select_experts(logits, 2, score=router.args.moe_router_score, groups=router.args.moe_router_groups,
                          top_groups=router.args.moe_router_top_groups, scale=router.args.moe_router_scale)
    got = router(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(got[1], plain)
    router.args = Arguments(**how)
    assert torch.equal(router(x)[1], plain)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name,top_k', [('tiny', 1), ('tiny-mixtral', 3)])
@pytest.mark.parametrize('training', [False, True])
def test_answers_of_models_that_drop_tokens(device, name, top_k, training):
    """Nothing is dropped in an answer: it does not depend on padding or on other sequences, and agrees with a pass
    over the whole sequence that drops nothing.  Training drops as before."""
    model = build(device, name, dropless=False, moe_capacity_factor=1, moe_top_k=top_k, moe_router_groups=1,
                  moe_router_top_groups=None).train(training)
    fixed_choice(model)                         # all tokens to the same experts: most would be dropped
    tokens = torch.randint(0, 512, (3, 20), device=device)
    lengths = torch.tensor([12, 5, 1], dtype=torch.int32, device=device)
    cache = model.new_cache(3, 16)
    got = [model.prefill(tokens[:, :12], cache, lengths)]
    for i in range(3):
        got.append(model.decode(tokens[torch.arange(3), (lengths + i).long()], cache))
    assert model.moe_args.moe_capacity_factor == 1 and model.training == training
    with pytest.raises(ValueError):
        model.prefill(tokens, cache)
    assert model.moe_args.moe_capacity_factor == 1
    model.eval()
    dropped = model(tokens[:1, :12])[0, -1].float()
    model.moe_args.moe_capacity_factor = 0
    with torch.no_grad():
        for b, n in enumerate(lengths.tolist()):
            whole = model(tokens[b:b + 1, :n + 3])[0].float()
            size = whole.abs().max()
            for i in range(4):
                bound = size * (2.0**-12 if device == 'cpu' else 40 * 2.0**-8)
                assert (got[i][b].float() - whole[n - 1 + i]).abs().max() <= bound
    assert (got[0][0].float() - dropped).abs().max() > 0


@pytest.mark.gpu
def test_recorded_decoding_of_a_model_that_drops_tokens():
    model = build('cuda', 'tiny', dropless=False, moe_capacity_factor=1).eval()
    tokens = torch.randint(0, 512, (3, 6), device='cuda')
    eager, cache = model.new_cache(3, 10), model.new_cache(3, 10)
    for c in (eager, cache):
        model.prefill(tokens, c)
    want = [model.decode(tokens[:, i], eager) for i in range(3)]
    static, graph = tokens[:, 0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.decode(static, cache)
    for i in range(3):
        static.copy_(tokens[:, i])
        graph.replay()
        assert torch.equal(out, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize('training', [False, True])
def test_bins_made_during_a_recording_are_its_own(training):
    """The first call with a number of tokens may be recorded: calls that follow, before a replay, take bins that are
    filled."""
    model = build('cuda', 'tiny', dropless=False, moe_capacity_factor=1).train(training)
    tokens = torch.randint(0, 512, (3, 6), device='cuda')
    cache, spare = model.new_cache(3, 10), model.new_cache(3, 10)
    for c in (cache, spare):
        model.prefill(tokens, c)
    want = build('cuda', 'tiny', dropless=False, moe_capacity_factor=1).eval()
    exact = want.new_cache(3, 10)
    want.prefill(tokens, exact)
    want = want.decode(tokens[:, 0], exact)
    graph = torch.cuda.CUDAGraph()
    known = [set(b.moe.experts.mlp._bins_cache) for b in model.blocks]
    with torch.cuda.graph(graph):
        out = model.decode(tokens[:, 0], cache)
    assert [set(b.moe.experts.mlp._bins_cache) for b in model.blocks] == known
    assert torch.equal(model.decode(tokens[:, 0], spare), want)
    graph.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize('device', DEVICES)
def test_training_behind_answers_in_inference_mode_of_a_model_that_drops_tokens(device):
    model = build(device, 'tiny', dropless=False, moe_capacity_factor=1)
    tokens = torch.randint(0, 512, (1, 8), device=device)
    with torch.inference_mode():
        model.eval()(tokens)                    # as many tokens as the training step has
        model.generate(tokens, 3)
    total, _ = model.train().loss(tokens, tokens.roll(-1, 1))
    total.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)

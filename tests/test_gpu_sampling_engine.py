"""Sampling and 4-bit weights in the engine: every token against the oracle's draw from the step's own logits, the pipelined
decode against stepping, every 4-bit MLP call against float64.

The MLP's tolerance, relative to its output in the 2-norm: the activations' rounding and the output's, HALF / sqrt(3) of the
value rms each at most (the products themselves add fp32 rounding, 1e-6)."""

import pytest
import torch

from oracle import fp4 as O4
from oracle import sampling as O
from tests.test_gpu_engine import _model, _prompts

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _engine(hf, model, eager=False, max_num_seqs=4, eos=-1, **kw):
    from atma_amd.engine import Config, LLMEngine
    return LLMEngine(Config(kvcache_block_size=16, max_num_seqs=max_num_seqs, max_num_batched_tokens=4096, max_model_len=160,
                            num_kvcache_blocks=64, enforce_eager=eager, hf_config=hf, eos=eos, **kw), model=model)


def _params(limits):
    from atma_amd.engine import SamplingParams
    asks = [dict(temperature=0.9, top_k=20, seed=1), dict(temperature=1.3, top_p=0.9, min_p=0.02, seed=2),
            dict(temperature=0.0), dict(temperature=1.0, seed=2 ** 70 + 3)]
    return [SamplingParams(max_tokens=m, ignore_eos=False, **a) for m, a in zip(limits, asks)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eager", [True, False])
def test_every_token_is_the_oracles_draw(dev, dtype, eager):
    from atma_amd.engine.sequence import uniform
    hf, model, _ = _model(dtype, seed=8)
    engine = _engine(hf, model, eager)
    seqs = [engine.add_request(p, sp) for p, sp in zip(_prompts([17, 40, 33, 5], 1), _params((6, 6, 6, 4)))]
    n = 0
    while not engine.is_finished():
        batch, is_prefill = engine.scheduler.schedule()
        toks = engine.model_runner.run(batch, is_prefill)
        logits = engine.model_runner.last_logits.double().tolist()
        for s, tok, x in zip(batch, toks, logits):
            p = s.params
            u = uniform(p.seed, len(s.completion_token_ids)) if p.seed is not None else 0.0
            f32 = lambda v: torch.tensor(v, dtype=torch.float32).item()   # noqa: E731
            assert tok == O.draw(x, u, f32(p.temperature), p.top_k, f32(p.top_p), f32(p.min_p))
            n += 1
        for s in engine.scheduler.commit(batch, toks):
            engine.model_runner.free_seq_slot(s)
    assert n == 22 and [len(s.completion_token_ids) for s in seqs] == [6, 6, 6, 4]
    engine.exit()


@pytest.mark.parametrize("fp4", [False, True])
def test_pipelined_sampling_equals_stepping(dev, fp4):
    """``generate`` launches sampled steps ahead too; a request that ends, by its limit or the end-of-sequence id, ends a run."""
    hf, _, _ = _model(torch.bfloat16, seed=9)
    prompts, limits = _prompts([23, 50, 9, 31], 4), (9, 5, 12, 12)

    def run(eos, pipelined):
        engine = _engine(hf, _model(torch.bfloat16, seed=9)[1], eos=eos, fp4_weights=fp4)
        if pipelined:
            launched = []
            launch = engine.model_runner.launch_decode
            engine.model_runner.launch_decode = lambda seqs, ahead: (launched.append(ahead), launch(seqs, ahead))[1]
            out = [r["token_ids"] for r in engine.generate(prompts, _params(limits))]
            assert sum(launched) > 0
        else:
            seqs = [engine.add_request(p, sp) for p, sp in zip(prompts, _params(limits))]
            while not engine.is_finished():
                engine.step()
            out = [s.completion_token_ids for s in seqs]
        engine.exit()
        return out

    free = run(-1, False)
    assert run(-1, True) == free and [len(t) for t in free] == list(limits)
    eos = free[2][6]
    stepped = run(eos, False)
    assert run(eos, True) == stepped


def test_rows_that_ask_for_a_temperature_alone(dev):
    """They are drawn by the race from torch's random numbers as before, beside rows that are not."""
    from atma_amd.engine import SamplingParams
    from atma_amd.engine.model import Picks, Sampler
    g = torch.Generator().manual_seed(10)
    logits = (3 * torch.randn(4, 500, generator=g)).to(torch.bfloat16).to(dev)
    t = torch.tensor([0.8, 1.0, 0.0, 1.2], device=dev)
    full = lambda v: torch.full((4,), v, device=dev)   # noqa: E731
    race = torch.tensor([False, True, False, True], device=dev)
    picks = Picks(full(0.3), t, torch.full((4,), 5, dtype=torch.int32, device=dev), full(0.9), full(0.0), race)
    torch.manual_seed(11)
    want = Sampler()(logits, t)
    torch.manual_seed(11)
    got = Sampler()(logits, t, picks=picks)
    assert torch.equal(got[race], want[race]) and torch.equal(got[~race], picks.sample(logits)[~race])
    hf, model, _ = _model(torch.bfloat16, seed=11)
    engine = _engine(hf, model)
    sps = [SamplingParams(temperature=1.0, max_tokens=5), SamplingParams(temperature=1.0, max_tokens=5, top_k=3, seed=4)]
    outs = [engine.generate(_prompts([12, 20], 6), sps)[1]["token_ids"] for _ in range(2)]
    assert outs[0] == outs[1] and len(outs[0]) == 5
    engine.exit()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_4_bit_call_of_the_engine(dev, dtype):
    hf, model, _ = _model(dtype, seed=12)
    head = model.proj.weight.detach().to(dtype)
    engine = _engine(hf, model, eager=True, fp4_weights=True)
    calls = []

    def watch(module, kind):
        forward = module.forward

        def seen(x, **kw):
            y = forward(x, **kw)
            calls.append((kind, module, x.detach().cpu(), y.detach().cpu()))
            return y
        module.forward = seen

    for block in model.blocks:
        watch(block.mlp, "mlp")
    watch(model.proj, "head")
    assert torch.equal(model.proj.fp4_weight.cpu(), O4.pack(O4.quantize(head)[0]))
    engine.generate(_prompts([17, 1, 70], 2), _params((3, 3, 3)))
    engine.exit()
    # one prefill and two decode steps
    assert sorted(k for k, *_ in calls) == ["head"] * 3 + ["mlp"] * 3 * len(model.blocks)
    for kind, m, x, y in calls:
        w = lambda n: O4.values(getattr(m, n + "_weight"), getattr(m, n + "_scale").view(torch.float8_e8m0fnu))   # noqa: E731
        if kind == "head":
            want, rounds = O4.linear(x, w("fp4"), m.fp4_bias.cpu())[0], 1
        else:
            a, gate = O4.linear(x, w("fc"), m.fc_bias.cpu())[0].chunk(2, 1)
            want, rounds = O4.linear(gate * a.clamp_min(0).square(), w("proj"), m.proj_bias.cpu())[0], 2
        err = ((y.double() - want).norm() / want.norm()).item()
        allowed = (rounds / 3) ** 0.5 * HALF[dtype] * 1.05 + 1e-6
        print(kind, tuple(x.shape), f"{err:.2e} of {allowed:.2e}", flush=True)
        assert err <= allowed


def test_a_step_from_head_to_token_in_a_graph(dev):
    """The 4-bit head, the soft cap and the sampler as one captured step, replayed with new inputs."""
    from atma_amd.kernel import linear_fp4, quantize_weight_fp4, sample_tokens, softcap_logits
    g = torch.Generator().manual_seed(13)
    weight = quantize_weight_fp4((0.05 * torch.randn(50304, 1024, generator=g)).to(torch.bfloat16).to(dev))
    bias = torch.randn(50304, generator=g).to(torch.bfloat16).to(dev)
    t, k = torch.tensor([0.0] + [0.7] * 31, device=dev), torch.full((32,), 50, dtype=torch.int32, device=dev)
    hs = [torch.randn(32, 1024, generator=g).to(torch.bfloat16).to(dev) for _ in range(3)]
    us = [torch.rand(32, generator=g).to(dev) for _ in range(3)]

    def step(h, u, out=None):
        return sample_tokens(softcap_logits(linear_fp4(h, *weight, bias)), u, t, top_k=k, top_p=0.9, ids_out=out)

    want = [step(h, u) for h, u in zip(hs, us)]
    h, u, ids = hs[0].clone(), us[0].clone(), torch.empty(32, dtype=torch.int64, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(h, u, ids)
    for i in (1, 2, 0, 2):
        h.copy_(hs[i])
        u.copy_(us[i])
        graph.replay()
        assert torch.equal(ids, want[i])

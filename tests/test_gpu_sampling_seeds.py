"""A request with a seed hands the sampler the same numbers alone and batched, at any position and in any graph's bucket, stepped and
pipelined; where its logits are the same to the bit, its tokens are."""

import pytest
import torch

from tests.test_gpu_engine import _model, _prompts
from tests.test_gpu_sampling_engine import _engine

pytestmark = pytest.mark.gpu

NEW = 7


@pytest.mark.parametrize("dtype,eager", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_alone_and_batched(dev, monkeypatch, dtype, eager):
    from atma_amd.engine import SamplingParams
    from atma_amd.engine import model_runner as MR
    hf, model, _ = _model(dtype, seed=15)
    engine = _engine(hf, model, eager, max_num_seqs=8)
    runner = engine.model_runner
    mine = SamplingParams(temperature=0.9, top_k=30, top_p=0.95, min_p=0.01, seed=77, max_tokens=NEW)
    other = [SamplingParams(temperature=0.0, max_tokens=NEW), SamplingParams(temperature=1.1, top_p=0.8, max_tokens=NEW, seed=5),
             SamplingParams(temperature=1.0, min_p=0.1, max_tokens=NEW)]
    prompt, rest = _prompts([21], 3)[0], _prompts([9, 33, 14, 27, 18], 4)
    handed = []

    class Seen(MR.Picks):
        def sample(self, logits, ids_out=None):
            ids = super().sample(logits, ids_out)
            handed.append([v.clone() for v in (self.uniform, self.temperature, self.top_k, self.top_p, self.min_p, logits, ids)])
            return ids
    monkeypatch.setattr(MR, "Picks", Seen)

    def run(at, others, pipelined):
        prompts, sps = list(rest[:others]), [other[i % 3] for i in range(others)]
        prompts.insert(at, prompt)
        sps.insert(at, mine)
        del handed[:]
        if pipelined:
            toks = engine.generate(prompts, sps)[at]["token_ids"]
        else:
            seqs = [engine.add_request(p, s) for p, s in zip(prompts, sps)]
            while not engine.is_finished():
                engine.step()
            toks = seqs[at].completion_token_ids
        assert len(toks) == NEW and len(handed) == NEW
        rows = [[v[at].cpu() for v in step] for step in handed]
        assert [int(r[6]) for r in rows] == toks
        return rows

    alone = run(0, 0, False)
    assert len({float(r[0]) for r in alone}) == NEW
    for at, others, pipelined in ((0, 0, True), (0, 2, False), (0, 2, True), (2, 2, False), (5, 5, False), (5, 5, True), (1, 3, True)):
        rows, same = run(at, others, pipelined), True
        for a, b in zip(alone, rows):
            for x, y in zip(a[:5], b[:5]):
                assert torch.equal(x, y), (at, others, pipelined)
            if torch.equal(a[5], b[5]):
                assert torch.equal(a[6], b[6])
    assert runner.can_pipeline([]) == (dtype != torch.float32 and not eager)
    engine.exit()


def test_without_a_seed_torchs(dev):
    """The same tokens again after the same torch.manual_seed, others after another; requests by temperature alone beside them too."""
    from atma_amd.engine import SamplingParams
    hf, model, _ = _model(torch.bfloat16, seed=16)
    engine = _engine(hf, model)
    sps = [SamplingParams(temperature=2.0, top_k=200, max_tokens=12), SamplingParams(temperature=2.0, max_tokens=12),
           SamplingParams(temperature=2.0, min_p=1e-4, max_tokens=12)]
    prompts = _prompts([12, 20, 7], 6)

    def run(state):
        torch.manual_seed(state)
        return [r["token_ids"] for r in engine.generate(prompts, sps)]
    a, b, c = run(1), run(1), run(2)
    assert a == b and all(x != y for x, y in zip(a, c))
    engine.exit()

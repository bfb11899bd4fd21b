"""What a decode step's host work asks of its requests, no GPU: whether any of them is sampled is settled once a run of steps."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from atma_amd.engine import ModelRunner, Sequence
from atma_amd.engine import model_runner as MR
from atma_amd.engine.sequence import SamplingParams

ROWS, PAGES, PAGE = 8, 4, 16


class Asked(SamplingParams):
    """Counts how often it is asked whether it samples."""
    count = 0

    @property
    def picks(self):
        Asked.count += 1
        return SamplingParams.picks.fget(self)


def _runner(monkeypatch):
    """A runner whose graph leaves row r token 100 + r, and whose sampler adds 1,000 to them."""
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    monkeypatch.setattr(MR.torch.cuda, "Event", lambda: SimpleNamespace(record=lambda: None, synchronize=lambda: None))
    drawn = []

    class Drawn:
        def __init__(self, *args):
            self.args = [a.clone() for a in args]

        def sample(self, logits, ids_out=None):
            drawn.append(self.args)
            return ids_out.copy_(1000 + 100 + torch.arange(len(ids_out)))
    monkeypatch.setattr(MR, "Picks", Drawn)
    r = ModelRunner.__new__(ModelRunner)
    r.device, r.block_size, r.pad_slot = torch.device("cpu"), PAGE, ROWS
    r.config = SimpleNamespace(max_num_seqs=ROWS, enforce_eager=False)
    r.graph_vars = r._decode_stage(ROWS, PAGES)
    r.graph_bs, r.graph_flip, r.last_logits = [2, ROWS], 0, None
    ids = r.graph_vars["input_ids"]

    def replay():
        ids.copy_(100 + torch.arange(ROWS))
    graph = SimpleNamespace(replay=replay)
    r.graphs = {b: [graph, graph] for b in r.graph_bs}
    r.graph_out = {b: [(torch.zeros(b, 10), ids[:b])] * 2 for b in r.graph_bs}
    return r, drawn


def _seqs(asks):
    seqs = []
    for i, ask in enumerate(asks):
        s = Sequence(list(range(5 + i)), Asked(**ask))
        s.block_table, s.seq_slot = [i], i
        seqs.append(s)
    return seqs


def test_a_greedy_run_is_asked_once(monkeypatch):
    r, drawn = _runner(monkeypatch)
    seqs = _seqs([dict(temperature=0.0)] * 5)
    Asked.count = 0
    for step in range(20):
        assert r.collect(r.launch_decode(seqs, ahead=int(step > 0))) == [100, 101, 102, 103, 104]
    assert Asked.count <= len(seqs) and not drawn


def test_a_greedy_step_is_not_asked(monkeypatch):
    """Nor a greedy batch that the sampler takes without a graph."""
    r, drawn = _runner(monkeypatch)
    r.sampler = lambda logits, temps, all_greedy, picks=None: (all_greedy, picks)
    seqs = _seqs([dict(temperature=0.0)] * 5)
    Asked.count = 0
    r._run_decode_graph(seqs)
    assert r._sample(torch.zeros(5, 10), seqs) == (True, None)
    assert Asked.count == 0 and not drawn


@pytest.mark.parametrize("later", [dict(temperature=0.0), dict(temperature=0.8, top_k=6, min_p=0.25, seed=12)], ids=["greedy", "sampled"])
def test_what_a_run_hands_the_sampler(monkeypatch, later):
    """Each launched step's parameters are its requests' at that step; parameters changed between runs are those of the next."""
    r, drawn = _runner(monkeypatch)
    seqs = _seqs([dict(temperature=0.7, top_k=5, seed=3), dict(temperature=0.0), dict(temperature=1.5, top_p=0.5, seed=4)])
    for n in range(3):
        got = r.collect(r.launch_decode(seqs, ahead=int(n > 0)))
        assert got == [1100, 1101, 1102]
    assert len(drawn) == 3
    for n, (u, t, k, p, m) in enumerate(drawn):
        assert u.tolist() == [s.uniform(int(n > 0)) if s.params.picks else 0.0 for s in seqs]
        assert k.tolist() == [5, 0, 0]
        for v, want in ((t, (0.7, 0.0, 1.5)), (p, (1.0, 1.0, 0.5)), (m, (0.0, 0.0, 0.0))):
            assert np.array_equal(v.numpy(), np.float32(want))
    del drawn[:]
    seqs[0].params, seqs[2].params = Asked(**later), Asked(temperature=0.0)
    ids = r.collect(r.launch_decode(seqs, ahead=0))
    if seqs[0].params.picks:
        assert ids == [1100, 1101, 1102] and drawn[0][2].tolist() == [6, 0, 0] and drawn[0][4].tolist() == [0.25, 0.0, 0.0]
    else:
        assert ids == [100, 101, 102] and not drawn


def test_greedy_steps_send_no_sampler_rows(monkeypatch):
    """What the sampler reads lies behind what the graphs read, and is sent with the steps that it is filled for."""
    r, drawn = _runner(monkeypatch)
    v = r.graph_vars
    greedy, sampled = _seqs([dict(temperature=0.0)] * 3), _seqs([dict(temperature=0.7, top_k=5, seed=3)] * 2)
    v["floats"].fill_(-1.0)
    v["top_k"].fill_(-1)
    for step in (lambda: r.launch_decode(greedy, ahead=0), lambda: r.launch_decode(greedy, ahead=1), lambda: r._run_decode_graph(greedy)):
        v["context_lens"].fill_(-1)
        step()
        assert v["context_lens"][:3].min() > 0 and v["slot_mapping"][:3].tolist()[0] >= 0
        assert (v["floats"] == -1).all() and (v["top_k"] == -1).all()
    r.launch_decode(sampled, ahead=0)
    assert v["top_k"][:2].tolist() == [5, 5] and v["block_tables"][:2, 0].tolist() == [0, 1]
    r.launch_decode(sampled, ahead=1)
    assert drawn[1][0].tolist() == [s.uniform(1) for s in sampled]

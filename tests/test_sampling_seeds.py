"""Where requests get their random numbers from: a seed of their own, or torch's CPU generator."""

import random

import pytest
import torch

from atma_amd.engine import ModelRunner, Sequence
from atma_amd.engine.sequence import SamplingParams, uniform

ASKS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.9, min_p=0.1), dict(seed=3),
        dict(temperature=0.0, top_k=5), dict(top_k=5, seed=4)]


@pytest.mark.parametrize("ask", ASKS, ids=str)
def test_the_callers_random_numbers_stay(ask):
    """Python's generator is the caller's; torch's moves for a request that samples without a seed, as it does for the race."""
    random.seed(1)
    torch.manual_seed(1)
    before, torch_before = random.getstate(), torch.get_rng_state()
    s = Sequence([1, 2, 3], SamplingParams(**ask))
    assert torch.equal(torch.get_rng_state(), torch_before)
    first = ModelRunner._picks([s])[0][0, 0]
    assert ModelRunner._picks([s])[0][0, 0] == first
    assert random.getstate() == before
    draws = s.params.picks and s.params.seed is None
    assert torch.equal(torch.get_rng_state(), torch_before) == (not draws)


def test_requests_without_a_seed_repeat_with_torchs():
    def numbers(state):
        torch.manual_seed(state)
        random.seed(7)   # (changes nothing)
        seqs = [Sequence([1], SamplingParams(top_k=5)) for _ in range(3)]
        return [[s.uniform(n) for n in range(4)] for s in seqs]

    a, b, c = numbers(1), numbers(1), numbers(2)
    assert a == b and a != c
    assert len({tuple(row) for row in a}) == 3
    assert all(0.0 <= v < 1.0 for row in a for v in row)


def test_a_seed_is_the_requests_own():
    for seed in (0, 3, -1, 2 ** 70 + 3):
        s = Sequence([1, 2], SamplingParams(top_k=5, seed=seed))
        assert [s.uniform(n) for n in range(3)] == [uniform(seed, n) for n in range(3)]
        s.token_ids.append(9)
        assert s.uniform() == uniform(seed, 1)

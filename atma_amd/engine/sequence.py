"""One generation request of the engine, and its sampling parameters.

A request is a growing token list (prompt, then the tokens it has sampled) plus the
handles the model runner needs to place it on the device: its KV pages, its row of the
per-sequence state tables, and how much of the list is already in those caches.  The
runner reads exactly these attributes, under the names the reference's runner reads
(``inference/engine/model_runner.py:316-480``): ``token_ids`` (through ``len`` and slicing),
``block_table``, ``num_cached_tokens``, ``num_scheduled_tokens``, ``seq_slot``, ``last_token``
and ``temperature``.  The lifecycle (queued -> active -> done) belongs to the scheduler.

``temperature == 0`` asks for greedy decoding (the reference's sampler divides by the
temperature and has no greedy form, ``inference/layers/sampler.py:7-10``).  ``top_k`` (0: all), ``top_p`` and ``min_p``
narrow the choice (``sample_tokens``); with a ``seed`` a request draws the same random numbers in every batch.  One that
narrows it without a seed takes its seed from torch's CPU generator when it is first sampled, so ``torch.manual_seed`` repeats it, as it does
the requests that ask for a temperature alone; Python's ``random`` is left as it is.
"""

from dataclasses import dataclass
from enum import Enum
from itertools import count
from operator import index
from typing import Optional

import torch


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 1.0
    max_tokens: int = 128
    ignore_eos: bool = False
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: Optional[int] = None

    def __post_init__(self):
        if self.top_k < 0 or not 0 < self.top_p <= 1 or not 0 <= self.min_p <= 1:
            raise ValueError(f"top_k >= 0, 0 < top_p <= 1 and 0 <= min_p <= 1 (got {self.top_k}, {self.top_p}, {self.min_p})")
        for name in ("top_k", "seed"):
            v = getattr(self, name)
            if v is not None:
                object.__setattr__(self, name, index(v))   # a whole number of any integer type, as a Python one

    @property
    def picks(self):
        """Whether the request asks for more than a temperature (and not for the likeliest token)."""
        return self.temperature != 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0 or self.seed is not None)


def uniform(seed, n):
    """The n-th random number of a seed: a multiple of 2^-24 in [0, 1), from the splitmix64 sequence (Steele, Lea and Flood, 2014)."""
    mask = (1 << 64) - 1
    z = (seed + (n + 1) * 0x9E3779B97F4A7C15) & mask
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9 & mask
    z = (z ^ (z >> 27)) * 0x94D049BB133111EB & mask
    return ((z ^ (z >> 31)) >> 40) * 2.0 ** -24


class Phase(Enum):
    QUEUED = "queued"      # waiting for pages and a state-table row
    ACTIVE = "active"      # admitted: prompt being prefilled, then decoding
    DONE = "done"          # finished; pages and row released


_ids = count()


class Sequence:
    """A request's tokens and device handles.  ``len(seq)`` is the number of tokens so far;
    ``seq[a:b]`` slices them."""

    __slots__ = ("seq_id", "token_ids", "prompt_len", "params", "phase", "block_table", "seq_slot",
                 "num_cached_tokens", "num_scheduled_tokens", "seed")

    def __init__(self, token_ids, sampling_params: SamplingParams = None):
        self.seq_id = next(_ids)
        self.token_ids = list(token_ids)
        self.prompt_len = len(self.token_ids)
        self.params = sampling_params if sampling_params is not None else SamplingParams()
        self.phase = Phase.QUEUED
        self.block_table = []          # physical KV page of each logical page, in order
        self.seq_slot = -1             # row of the runner's state tables (-1: none held)
        self.num_cached_tokens = 0     # tokens whose K/V, conv tails and memory state are stored
        self.num_scheduled_tokens = 0  # tokens the current step feeds
        self.seed = self.params.seed  # None: drawn when the first random number is asked for

    def __len__(self):
        return len(self.token_ids)

    def __getitem__(self, key):
        return self.token_ids[key]

    @property
    def temperature(self):
        return self.params.temperature

    def uniform(self, ahead=0):
        """The random number of the token that follows ``ahead`` further ones."""
        if self.seed is None:
            self.seed = int(torch.randint(2 ** 63 - 1, (), device="cpu"))
        return uniform(self.seed, len(self.token_ids) - self.prompt_len + ahead)

    @property
    def last_token(self):
        return self.token_ids[-1]

    @property
    def prompt_done(self):
        """Every prompt token is in the caches: the next step is a decode step."""
        return self.num_cached_tokens >= self.prompt_len

    @property
    def completion_token_ids(self):
        return self.token_ids[self.prompt_len:]

    @property
    def is_finished(self):
        return self.phase is Phase.DONE

    def lifetime_tokens(self):
        """The most tokens this request can ever hold: prompt plus its token limit (the
        last sampled token is never fed back, but its slot is counted to keep this simple)."""
        return self.prompt_len + self.params.max_tokens

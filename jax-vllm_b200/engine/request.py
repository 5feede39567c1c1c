"""Request records, after the reference's (jllm/engine/request.py:5-41), with sampling
temperature, filters and seed added, the log-probabilities of what was sampled, and the
requests that continue the same prompt."""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Optional


@dataclass
class SamplingParams:
    max_new_tokens: int = 64
    eos_id: Optional[int] = None      # generation stops after this token (which is emitted)
    temperature: float = 0.0          # 0: greedy; > 0: a draw from softmax(logits / temperature)
    seed: Optional[int] = None        # None: the request id
    stop_token_ids: tuple = ()        # more tokens that end the generation (emitted, like eos_id)
    ignore_eos: bool = False          # run to max_new_tokens whatever is sampled (for measurements)
    # Filters of a draw (temperature > 0).  With the tokens in order of their logits and p = exp((logit - largest) / temperature):
    top_k: int = 0                    # > 0: only the first top_k tokens
    top_p: float = 1.0                # < 1: of those, only the ones before which less than top_p of their sum of p lies
    min_p: float = 0.0                # > 0: only tokens with p >= min_p
    logprobs: Optional[int] = None    # not None: every event carries its token's log-probability (of the logits as they are,
                                      # without temperature and filters) and the so many likeliest tokens with theirs

    def __post_init__(self):
        if self.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        if self.temperature < 0:
            raise ValueError("temperature must not be negative")
        if self.top_k < 0 or self.top_k >= 1 << 31:
            raise ValueError("top_k must not be negative (0: all tokens)")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_p must lie in (0, 1]")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError("min_p must lie in [0, 1]")
        if self.logprobs is not None and not 0 <= self.logprobs <= 128:
            raise ValueError("logprobs must be None or lie in [0, 128]")
        self.stop_token_ids = tuple(int(t) for t in self.stop_token_ids)

    @property
    def filtered(self) -> bool:
        return self.temperature > 0 and (self.top_k > 0 or self.top_p < 1.0 or self.min_p > 0.0)

    def stops_at(self, token: int) -> bool:
        if self.ignore_eos:
            return False
        return (self.eos_id is not None and token == self.eos_id) or token in self.stop_token_ids


@dataclass
class Request:
    request_id: int
    prompt_ids: list
    sampling: SamplingParams
    output_ids: list = field(default_factory=list)
    finished: bool = False
    slot: Optional[int] = None
    preemptions: int = 0
    arrival: float = 0.0
    first_token_time: Optional[float] = None
    followers: list = field(default_factory=list)   # requests that continue the same prompt once it is computed
    logprobs: list = field(default_factory=list)    # with sampling.logprobs: of every token in output_ids that was sampled here
    top_logprobs: list = field(default_factory=list)

    @property
    def tokens(self) -> list:
        """Everything known of the sequence: the prompt and what was generated so far."""
        return self.prompt_ids + self.output_ids


@dataclass
class StepEvent:
    request_id: int
    token: int
    finished: bool
    logprob: Optional[float] = None          # with SamplingParams.logprobs
    top_logprobs: Optional[list] = None      # the likeliest tokens as (token, logprob), the likeliest first


@dataclass
class EngineStats:
    admissions: int = 0
    scheduler_loops: int = 0
    steps: int = 0                    # batches run on the device
    prefill_tokens: int = 0           # tokens run that were not single decoded tokens
    decode_tokens: int = 0
    emitted_tokens: int = 0
    cache_hit_blocks: int = 0
    cache_hit_tokens: int = 0
    preemptions: int = 0
    forks: int = 0                    # requests that took over what another holds in the cache
    finished: int = 0
    # per step (the reference has no counterpart: its pool is always the worst case and its steps are padded)
    last_step_tokens: int = 0         # tokens that the last step ran
    max_step_tokens: int = 0
    pages_in_use: int = 0             # after the last step, in the fullest pool
    max_pages_in_use: int = 0
    pages_total: int = 0

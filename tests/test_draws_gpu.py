"""Draws against their definition: the token with the largest logit / T - log(-log(u)), u = (n + 1/2) / 2^24 in (0, 1), evaluated
in 64 bits.  What the device may add to it: u is rounded to 32 bits (2^-25 at most, and it stays below 1), and the score is
formed in 32 bits."""

import numpy as np
import pytest
import torch

from jax_vllm_b200 import ops
from jax_vllm_b200.sampling import uniform

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def mix(z):
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def uniforms(seed, counter, n):
    with np.errstate(over="ignore"):
        h = mix(np.uint64(seed) + np.uint64(0x9E3779B97F4A7C15) * np.uint64(counter + 1))
        h = mix(h ^ (np.arange(n, dtype=np.uint64) * np.uint64(0xD1342543DE82EF95) + np.uint64(0x2545F4914F6CDD1D)))
    return ((h >> np.uint64(40)).astype(np.float64) + 0.5) / 16777216.0


def possible(x, t, kept, seed, counter):
    """The tokens that may have the largest score among the kept ones."""
    u = uniforms(seed, counter, x.size)
    y = x / t
    # rounded to 32 bits u is off by half a step of the numbers below 1, and at most the largest of them
    low, high = (y - np.log(-np.log(v)) for v in (np.maximum(u - 2.0 ** -25, 2.0 ** -25), np.minimum(u + 2.0 ** -25, 1 - 2.0 ** -24)))
    # the quotient, both logarithms (the inner one's error is relative) and the difference: six half steps of the terms
    off = 2.0 ** -24 * 6 * (np.abs(y) + np.maximum(np.abs(low - y), np.abs(high - y)) + 1)
    return set(np.where(kept & (high + off >= np.max(np.where(kept, low - off, -INF))))[0].tolist())


def filtered(x, t, k, p, m, seed, counter):
    one = lambda v, d: torch.tensor([v], dtype=d, device=DEV)  # noqa: E731
    return ops.sample_filtered(x[None].to(DEV), one(t, torch.float32), one(k, torch.int32), one(p, torch.float32), one(m, torch.float32),
                               one(seed, torch.int64), one(counter, torch.int64)).item()


def plain(x, t, seed, counter):
    one = lambda v, d: torch.tensor([v], dtype=d, device=DEV)  # noqa: E731
    return ops.sample(x[None].to(DEV), one(t, torch.float32), one(seed, torch.int64), one(counter, torch.int64)).item()


# (seed, token, vocabulary) whose 24 random bits at counter 0 are all ones
TOPMOST = [(925, 3341, 4096), (15, 16852, 151936), (52, 78975, 151936)]


@pytest.mark.parametrize("seed,token,vocab", TOPMOST)
def test_the_topmost_random_number_is_below_one(seed, token, vocab):
    """Its score is 17.3 in 64 bits and 16.6 in 32: 25 below the others in logit / T, its token cannot be drawn (no other's
    score is below -2.9).  Without filters, and under filters of every path that keeps it."""
    assert uniforms(seed, 0, vocab)[token] == uniform(seed, 0, token) == 1 - 2.0 ** -25
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(vocab, generator=gen) * 0.01
    x[token] = -25.0
    kept = np.ones(vocab, bool)
    for t in (1.0, 1.25):
        x[token] = -25.0 * t
        want = possible(x.double().numpy(), t, kept, seed, 0)
        assert token not in want
        assert plain(x, t, seed, 0) in want
        # none, a count that leaves one token out at most, a share and a mass that leave all of them
        for k, p, m in ((0, 1.0, 0.0), (vocab - 1, 1.0, 0.0), (0, 1.0, 1e-12), (vocab - 1, 1.0, 1e-12)):
            assert filtered(x, t, k, p, m, seed, 0) in want, (t, k, p, m)
    # a short list: 30 tokens and this one, the others masked
    few = torch.full((vocab,), -INF)
    at = torch.randperm(vocab, generator=gen)[:30]
    few[at] = 0.0
    few[token] = -25.0
    kept = (few > -INF).numpy()
    want = possible(np.where(kept, few.double().numpy(), 0.0), 1.0, kept, seed, 0)
    assert token not in want
    for k, p, m in ((0, 1.0, 0.0), (40, 1.0, 0.0), (40, 1.0, 1e-12), (0, 1.0, 1e-12)):
        assert filtered(few, 1.0, k, p, m, seed, 0) in want, (k, p, m)


@pytest.mark.parametrize("seed,token,vocab", TOPMOST)
def test_the_topmost_random_number_under_masses(seed, token, vocab):
    """Half of the tokens 10 above the rest, of which top-p keeps about a half too, this token as the first of them."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(vocab, generator=gen) * 0.01
    x[torch.randperm(vocab, generator=gen)[:vocab // 2]] += 10
    x[token] = 0.5
    mass = np.exp(x.double().numpy())
    p = 1 - 0.5 * mass[mass < 2].sum() / mass.sum()
    want = possible(x.double().numpy(), 1.0, np.ones(vocab, bool), seed, 0)
    assert token not in want
    assert filtered(x, 1.0, 0, p, 0.0, seed, 0) in want
    assert filtered(x, 1.0, vocab - 1, p, 1e-9, seed, 0) in want


def test_every_drawn_token_is_the_definition_s():
    """2,000 rows of 4,096 even logits, with and without filters."""
    rows, vocab = 2000, 4096
    x = torch.zeros(rows, vocab, device=DEV)
    seeds, counters = torch.arange(rows, device=DEV), torch.arange(rows, device=DEV) % 7
    f = lambda v, d: torch.full((rows,), v, dtype=d, device=DEV)  # noqa: E731
    a = ops.sample(x, f(0.8, torch.float32), seeds, counters).tolist()
    b = ops.sample_filtered(x, f(0.8, torch.float32), f(0, torch.int32), f(1.0, torch.float32), f(0.0, torch.float32), seeds, counters).tolist()
    c = ops.sample_filtered(x, f(0.8, torch.float32), f(1000, torch.int32), f(1.0, torch.float32), f(0.0, torch.float32), seeds, counters).tolist()
    assert a == b
    everything, first = np.ones(vocab, bool), np.arange(vocab) < 1000
    for r in range(rows):
        assert a[r] in possible(np.zeros(vocab), 0.8, everything, r, r % 7)
        assert c[r] in possible(np.zeros(vocab), 0.8, first, r, r % 7)

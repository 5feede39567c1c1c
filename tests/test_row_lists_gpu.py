"""The lists of a row's first tokens where they are hard to get: many equal logits, masks of a low finite value, rows in ascending
order, long rows that one block reads by itself.  Against the same 64-bit implementations as the operators' other tests."""

import numpy as np
import pytest
import torch

from jax_vllm_b200 import ops
from tests.test_continuations_ops_gpu import DTYPES, check_sample, graph_of, names, near, plain_logprobs, rows_of, sample
from tests.test_draws_gpu import uniforms

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FILTERS = [(1.0, 0, 0.9, 0.0), (1.0, 100, 1.0, 0.0), (1.0, 700, 0.98, 0.0), (0.5, 1900, 1.0, 0.0), (2.0, 0, 0.3, 0.0), (1.0, 0, 0.9999, 0.0)]


def crowded(vocab, kind, dtype):
    gen = torch.Generator(DEV).manual_seed(vocab)
    x = torch.zeros(len(FILTERS), vocab, device=DEV)
    if kind == "one apart":
        x[:, vocab // 3] = 5.0
    if kind == "few far above":
        x[:] = torch.finfo(dtype).min
        x[:, 3:8] = torch.randn(len(FILTERS), 5, device=DEV, generator=gen)
    if kind == "clipped":
        x = torch.randn(len(FILTERS), vocab, device=DEV, generator=gen).clamp(min=-0.5, max=1.0)
        x[:, vocab // 2] = 4.0
    if kind == "coarse":
        x = (torch.randn(len(FILTERS), vocab, device=DEV, generator=gen) * 0.05 + 8).bfloat16()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=names.get)
@pytest.mark.parametrize("kind", ["one apart", "few far above", "clipped", "coarse"])
@pytest.mark.parametrize("vocab", [128, 129, 255, 513, 1024, 1025, 1900, 2048, 2049, 9001])
def test_lists_of_mostly_equal_logits(vocab, kind, dtype):
    x = crowded(vocab, kind, dtype)
    check_sample(x, rows_of(FILTERS, vocab))
    tokens = torch.full((x.shape[0],), vocab // 3, dtype=torch.int32, device=DEV)
    for top in (20, 128):
        got, want = ops.token_logprobs(x, tokens, top), plain_logprobs(x, tokens, top)
        assert torch.equal(got[1], want[1])
        near(got[0], want[0], "token"); near(got[2], want[2], "top")


def microseconds(call):
    graph, _ = graph_of(lambda: [call() for _ in range(20)])
    best = float("inf")
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(); graph.replay(); b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / 20)
    return best


def test_a_crowded_list_takes_no_multiple_of_an_even_one():
    """1,900 tokens: one above equal others, against all of them different.  A comparison of every token with every other one
    took ten times as long, a network takes about twice as long."""
    gen = torch.Generator(DEV).manual_seed(1)
    even, one = torch.randn(64, 1900, device=DEV, generator=gen) * 0.1, crowded(1900, "one apart", torch.float32)[:1].repeat(64, 1)
    params = [torch.full((64,), v, dtype=d, device=DEV) for v, d in ((1.0, torch.float32), (0, torch.int32), (0.9, torch.float32), (0.0, torch.float32),
                                                                     (7, torch.int64), (0, torch.int64))]
    a, b = (microseconds(lambda x=x: ops.sample_filtered(x, *params)) for x in (even, one))
    assert b < 4 * a, (a, b)


# A row that one block reads by itself (more rows than multiprocessors) is read once: the bound of what is listed is taken on the
# way, after the first 3,072 vectors of 16 bytes and after 9,216, and masses are relative to the largest logit so far.
# In a row that ascends every vector of a thread (75 of 151,936 logits, 4 a vector) raises its largest, and the sum so far is
# multiplied by an exponential: two steps of it (2^-22) and the product's half a step (2^-24) each, 75 * 5 * 2^-24 = 2.2e-5 of
# the sum at most.  With a mass's own 40 * 2^-24 and the 75 additions' half steps that is 2.9e-5 for either side of a border.
MASSES = 2 * 2.9e-5


def allowed(x, t, k, p, m, seed, counter):
    """The tokens that a row may give by the definition, with 32-bit masses and scores."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    y = x[order]
    mass = np.exp((y - y[0]) / t)
    keep = (y > -np.inf) & (mass >= m)
    if k > 0:
        keep &= np.arange(x.size) < k
    sure, may = keep.copy(), keep.copy()
    if p < 1:
        before = np.cumsum(np.where(keep, mass, 0.0)) - np.where(keep, mass, 0.0)
        target = p * mass[keep].sum()
        sure &= before < target * (1 - MASSES)
        may &= before < target * (1 + MASSES)
    sure[0] = may[0] = True
    q, u = np.where(keep, y, 0.0) / t, uniforms(seed, counter, x.size)[order]
    low, high = (q - np.log(-np.log(v)) for v in (np.maximum(u - 2.0 ** -25, 2.0 ** -25), np.minimum(u + 2.0 ** -25, 1 - 2.0 ** -24)))
    off = 2.0 ** -24 * 6 * (np.abs(q) + np.maximum(np.abs(low - q), np.abs(high - q)) + 1)
    least = np.max(np.where(sure, low - off, -np.inf))
    return set(order[may & (high + off >= least)].tolist())


LONG = [(1.0, 50, 1.0, 0.0), (0.7, 40, 0.95, 0.02), (0.6, 0, 0.9, 0.0), (1.0, 0, 0.4, 0.0), (0.9, 128, 0.98, 0.0), (1.0, 7, 0.9, 0.0), (0.5, 0, 0.99, 0.01)]


def long_rows(order, vocab, n):
    gen = torch.Generator(DEV).manual_seed(vocab + len(order))
    x = torch.randn(n, vocab, device=DEV, generator=gen) * 2.2
    if order == "ascending":
        x = x.sort(1)[0]
    if order == "descending":
        x = x.sort(1, descending=True)[0]
    if order == "masked, then large":
        x[:, :vocab // 2] = -float("inf")
        x[:, -9:] += 6
    if order == "NaN, then small":
        x[:, :vocab // 5] = float("nan")
        x[:, -vocab // 5:] -= 300
    if order == "peaks at both ends":
        x[:, :20] += 9
        x[:, -20:] += 10
    return x


@pytest.mark.parametrize("order", ["random", "ascending", "descending", "masked, then large", "NaN, then small", "peaks at both ends"])
@pytest.mark.parametrize("vocab,dtype,off", [(151936, torch.float32, 0), (36865, torch.float32, 1), (36871, torch.float32, 3), (60013, torch.float32, 2),
                                             (73729, torch.bfloat16, 1), (151936, torch.bfloat16, 0), (90001, torch.bfloat16, 5)])
def test_long_rows_that_one_block_reads(vocab, dtype, off, order):
    """More rows than two blocks each would find room for; a dozen of them against the definition, at every place in the batch."""
    checked, rows = 14, 160
    x = long_rows(order, vocab, checked).to(dtype)
    wide = torch.full((rows, vocab + 8), 70.0, dtype=dtype, device=DEV)
    batch = wide[:, off:off + vocab]
    batch[:] = x[torch.arange(rows, device=DEV) % checked]
    params = rows_of([LONG[i % len(LONG)] for i in range(rows)], vocab)
    got = sample(batch, params).tolist()
    host = x.double().cpu().numpy()
    for r in list(range(7)) + list(range(rows - 7, rows)):
        t, k, p, m, seed, counter = params[r]
        want = allowed(host[r % checked], float(np.float32(t)), k, float(np.float32(p)), float(np.float32(m)), seed, counter)
        assert got[r] in want, (r, params[r], got[r], sorted(want)[:5])
    tokens = torch.full((rows,), vocab - 1, dtype=torch.int32, device=DEV)
    lp, want = ops.token_logprobs(batch, tokens, 20), plain_logprobs(batch[:checked], tokens[:checked], 20)
    assert torch.equal(lp[1][:checked], want[1])
    near(lp[0][:checked], want[0], "token"); near(lp[2][:checked], want[2], "top")

"""Filtered sampling, log-probabilities of tokens, and copies of cache pages and state rows, against plain implementations in
64 bits.  (Refusals that need no GPU: test_continuations_checks.py.)"""

import math

import numpy as np
import pytest
import torch

from jax_vllm_b200 import ops
from jax_vllm_b200.sampling import uniform

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")
DTYPES = [torch.float32, torch.bfloat16]
names = {torch.float32: "f32", torch.bfloat16: "bf16"}


# ------------------------------------------------------------------------------------------------------ plain sampling
def mix(z):
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def uniforms(seed, counter, n):
    with np.errstate(over="ignore"):
        h = mix(np.uint64(seed) + np.uint64(0x9E3779B97F4A7C15) * np.uint64(counter + 1))
        h = mix(h ^ (np.arange(n, dtype=np.uint64) * np.uint64(0xD1342543DE82EF95) + np.uint64(0x2545F4914F6CDD1D)))
    # the half is added in 32 bits, as on the device: above 1/2 the sum is rounded to a whole number of 2^-24
    return ((h >> np.uint64(40)).astype(np.float32) + np.float32(0.5)).astype(np.float64) / 16777216.0


def test_uniforms_of_this_file_are_the_package_s():
    want = np.array([uniform(12345, 6, v) for v in range(500)])
    assert np.abs(uniforms(12345, 6, 500) - want).max() <= 2.0 ** -25


# A mass exp((x - largest) / T) is formed in 32 bits: the difference, log2(e) / T and their product are each off by half a step
# (2^-24), which in the exponent makes 3 * 2^-24 * d for d = (largest - x) / T, and the exponential adds two steps (2^-22).
# Tokens with d > 30 are below 2^-43 of the largest mass and may be left out.  Weighed by the masses themselves, d is no more than
# log(151936) = 12 on the average, so the masses put sums off by 40 * 2^-24 = 2.4e-6 of themselves.  A thread adds up to 75 vectors'
# sums, half a step each (75 * 2^-24 = 4.5e-6 where one block reads a row), across threads in 64 bits.  Both sides of a border
# are such sums: 2 * (2.4e-6 + 4.5e-6) = 1.4e-5; twice 5.7e-6 is asked for.
def accepted(x, t, k, p, m, seed, counter):
    """The tokens that a row may give: exact but where a border, or two scores, lie nearer than 32 bits tell apart."""
    x = np.where(np.isnan(x), -INF, x) + 0.0
    n = x.size
    if not t > 0:
        return {int(np.argmax(x))}
    order = np.argsort(-x, kind="stable")
    y = x[order]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        mass = np.exp(np.where(y == y[0], 0.0, (y - y[0]) / t))
    keep = np.ones(n, bool)
    if k > 0:
        keep &= np.arange(n) < k
    if m > 0:
        keep &= mass >= min(m, 1.0)
    sure, may = keep.copy(), keep.copy()
    if p < 1:
        mass = np.where(keep, mass, 0.0)
        before = np.cumsum(mass) - mass
        target, off = p * mass.sum(), 2 * 5.7e-6 * mass.sum() * p + n * 2.0 ** -43
        sure &= before < target - off
        may &= before < target + off
    sure[0] = may[0] = True
    u = uniforms(seed, counter, n)[order]
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        q = y / t
        q = np.where(np.abs(q) > 3.4028235e38, np.sign(q) * INF, q)        # as it is in 32 bits
        score = q - np.log(-np.log(u))
        # the quotient, both logarithms (the inner one's error is relative) and the difference: six half steps of the terms
        off = 2.0 ** -24 * 6 * (np.abs(np.where(np.isfinite(q), q, 0)) + np.abs(np.log(-np.log(u))) + 1)
    best = np.max(np.where(sure, score, -INF))
    if np.isinf(best):
        return {int(order[np.where(may & (score == best))[0]].min())}
    low = np.max(np.where(sure, score - off, -INF))
    return set(int(i) for i in order[may & (score + off >= low)])


def sample(logits, rows):
    t, k, p, m, seeds, counters = (list(v) for v in zip(*rows))
    f = lambda v, d: torch.tensor(v, dtype=d, device=DEV)  # noqa: E731
    return ops.sample_filtered(logits, f(t, torch.float32), f(k, torch.int32), f(p, torch.float32), f(m, torch.float32),
                               f(seeds, torch.int64), f(counters, torch.int64))


def check_sample(logits, rows):
    got = sample(logits, rows).tolist()
    x = logits.double().cpu().numpy()
    for r, (row, tok) in enumerate(zip(rows, got)):
        t, k, p, m, seed, counter = row
        want = accepted(x[r], float(np.float32(t)), k, float(np.float32(p)), float(np.float32(m)), seed, counter)
        assert tok in want, f"row {r} {row}: {tok} is none of {sorted(want)[:5]}"
    return got


FILTERS = [(0.0, 5, 0.5, 0.1), (1.0, 0, 1.0, 0.0), (0.8, 1, 1.0, 0.0), (0.8, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 0.3, 0.0),
           (1.1, 0, 1.0, 0.05), (0.7, 40, 0.95, 0.02), (0.9, 700, 0.98, 0.0), (1.0, 3000, 0.999, 0.0), (2.0, 0, 0.99, 1e-4),
           (0.05, 20, 0.9, 0.0), (30.0, 20, 0.9, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1e-9, 0.0),
           (1.0, 100000, 0.9999999, 0.0)]


def rows_of(filters, seed):
    return [(*f, (seed * 7919 + 104729 * i) % (1 << 62), i * 3) for i, f in enumerate(filters)]


@pytest.mark.parametrize("dtype", DTYPES, ids=names.get)
@pytest.mark.parametrize("spread", [0.0, 0.02, 1.0, 4.0])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 271, 1025, 4099, 32003, 151936])
def test_filtered_sampling(vocab, spread, dtype):
    gen = torch.Generator(DEV).manual_seed(vocab + int(100 * spread))
    x = torch.randn(len(FILTERS), vocab, device=DEV, generator=gen) * spread
    if spread == 4.0:                                  # some tokens far above the rest
        x[:, :: max(1, vocab // 9)] += 12
    check_sample(x.to(dtype), rows_of(FILTERS, vocab))


@pytest.mark.parametrize("vocab", [50, 5003, 151936])
def test_filtered_sampling_of_masked_rows(vocab):
    """Rows in which the mask leaves nothing, one token, a few; masks of the lowest value; NaN and infinities."""
    gen = torch.Generator(DEV).manual_seed(vocab)
    base = torch.randn(12, vocab, device=DEV, generator=gen) * 2
    at = torch.randint(0, vocab, (40,), device=DEV, generator=gen)
    base[0] = -INF
    base[1] = -INF; base[1, vocab - 1] = -3.0
    base[2] = torch.finfo(torch.float32).min; base[2, at] = torch.randn(40, device=DEV, generator=gen)
    base[3] = torch.finfo(torch.float32).min
    base[4] = float("nan")
    base[5, at] = float("nan")
    base[6] = -INF; base[6, at] = 1.0
    base[7, at[:3]] = INF
    base[8] = -1e9; base[8, at] = torch.randn(40, device=DEV, generator=gen) * 5
    base[9] = 0.0; base[9, ::2] = -0.0
    base[10, at] = -INF
    base[11] = torch.randn(vocab, device=DEV, generator=gen) * 1e30
    for f in FILTERS:
        got = check_sample(base, rows_of([f] * 12, 31))
        assert got[0] == 0 and got[1] == vocab - 1 and got[4] == 0
        assert got[6] in at.tolist() and got[8] in at.tolist()


@pytest.mark.parametrize("filters", [(1e-30, 40, 0.9, 0.0), (1e-38, 0, 0.9, 0.1), (1e30, 40, 0.9, 0.0), (INF, 0, 0.5, 0.0), (INF, 7, 1.0, 0.0),
                                     (float("nan"), 3, 0.5, 0.0), (-1.0, 3, 0.5, 0.0), (1.0, -5, 1.0, 0.0), (1.0, 1 << 30, 0.9, 0.0),
                                     (1.0, 20, 7.0, -1.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1.0, 9.0), (1e-45, 5, 0.5, 0.5)])
def test_filtered_sampling_outside_the_usual_values(filters):
    gen = torch.Generator(DEV).manual_seed(3)
    x = torch.randn(3, 6007, device=DEV, generator=gen)
    t, k, p, m = filters
    check_sample(x, rows_of([(t if t > 0 else 0.0, max(k, 0), p, m)] * 3, 5))
    same = sample(x, rows_of([filters] * 3, 5)).tolist()
    assert same == sample(x, rows_of([(t if t > 0 else 0.0, max(k, 0), min(max(p, 0.0), 1.0), min(max(m, 0.0), 1.0))] * 3, 5)).tolist()


@pytest.mark.parametrize("vocab", [9, 3001, 151936])
def test_rows_without_filters_get_the_tokens_of_plain_sampling(vocab):
    gen = torch.Generator(DEV).manual_seed(vocab)
    rows = 60
    x = torch.randn(rows, vocab, device=DEV, generator=gen) * 3
    x[3] = -INF
    x[4, ::3] = float("nan")
    t = torch.rand(rows, device=DEV, generator=gen) * 2
    t[::5] = 0
    seeds = torch.randint(0, 1 << 62, (rows,), device=DEV, generator=gen)
    counters = torch.randint(0, 999, (rows,), device=DEV, generator=gen)
    zeros = torch.zeros(rows, device=DEV)
    got = ops.sample_filtered(x, t, zeros.int(), zeros + 1, zeros, seeds, counters)
    assert torch.equal(got, ops.sample(x, t, seeds, counters))


@pytest.mark.parametrize("dtype", DTYPES, ids=names.get)
def test_a_row_s_token_depends_on_the_row_alone(dtype):
    """The same rows in a batch of 300, alone, in another order, in rows that are far apart, and off 16-byte boundaries."""
    gen = torch.Generator(DEV).manual_seed(8)
    n, vocab = 300, 20011
    x = (torch.randn(n, vocab, device=DEV, generator=gen) * 2).to(dtype)
    rows = rows_of([FILTERS[i % len(FILTERS)] for i in range(n)], 77)
    whole = sample(x, rows).tolist()
    assert whole == sample(x, rows).tolist()
    assert whole[::-1] == sample(x.flip(0).contiguous(), rows[::-1]).tolist()
    assert whole[:17] == [sample(x[i:i + 1], rows[i:i + 1]).item() for i in range(17)]
    for off in (1, 3, 5):
        wide = torch.full((n, vocab + 29), 50.0, dtype=dtype, device=DEV)
        wide[:, off:off + vocab] = x
        assert whole == sample(wide[:, off:off + vocab], rows).tolist()


def test_the_largest_vocabulary():
    gen = torch.Generator(DEV).manual_seed(2)
    x = torch.randn(3, ops.MOST_VOCAB, device=DEV, generator=gen)
    check_sample(x, rows_of([(1.0, 0, 0.9, 0.0), (1.0, 500000, 0.5, 0.0), (1.0, 0, 1.0, 0.2)], 4))
    x[:] = 1.0
    check_sample(x, rows_of([(1.0, 0, 0.75, 0.0), (1.0, 500000, 0.5, 0.0), (1.0, 0, 1.0, 0.2)], 4))
    with pytest.raises(ops.KernelError):
        sample(torch.zeros(1, ops.MOST_VOCAB + 1, device=DEV), rows_of(FILTERS[:1], 1))


def test_draws_follow_the_kept_tokens_softmax():
    """20,000 draws from five kept tokens: each count within five standard deviations of its expectation."""
    n = 20000
    x = torch.tensor([0.3, -1.0, 1.2, 0.9, -0.2, -3.0, 0.1, -5.0], device=DEV).repeat(n, 1)
    f = lambda v, d: torch.full((n,), v, dtype=d, device=DEV)  # noqa: E731
    got = ops.sample_filtered(x, f(0.8, torch.float32), f(5, torch.int32), f(1.0, torch.float32), f(0.0, torch.float32),
                              f(99, torch.int64), torch.arange(n, device=DEV))
    p = torch.softmax(x[0].double() / 0.8, 0)
    p[torch.argsort(x[0], descending=True)[5:]] = 0
    p /= p.sum()
    counts = torch.bincount(got.long(), minlength=8).double()
    assert ((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all(), (counts, n * p)


def graph_of(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def test_captured_replayed_and_on_other_streams():
    gen = torch.Generator(DEV).manual_seed(5)
    n, vocab = 33, 9001
    x = torch.randn(n, vocab, device=DEV, generator=gen) * 2
    rows = rows_of([FILTERS[i % len(FILTERS)] for i in range(n)], 13)
    params = [torch.tensor(v, dtype=d, device=DEV) for v, d in zip(zip(*rows), (torch.float32, torch.int32, torch.float32, torch.float32,
                                                                                torch.int64, torch.int64))]
    tokens = torch.randint(0, vocab, (n,), device=DEV, dtype=torch.int32, generator=gen)
    one, a = graph_of(lambda: ops.sample_filtered(x, *params))
    two, b = graph_of(lambda: ops.token_logprobs(x, tokens, 7))
    for seed in (1, 2):
        x.copy_(torch.randn(n, vocab, device=DEV, generator=gen) * 2)
        one.replay(); two.replay(); one.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.sample_filtered(x, *params))
        for got, want in zip(b, ops.token_logprobs(x, tokens, 7)):
            assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.sample_filtered(x, *params)
    side.synchronize()
    assert torch.equal(again, a)


# ------------------------------------------------------------------------------------------------------ log-probabilities
def plain_logprobs(x, tokens, top):
    x = x.double()
    x = torch.where(x.isnan(), -INF, x)
    largest = x.amax(1, keepdim=True)
    e = torch.where(x == largest, 1.0, torch.exp(x - largest))
    e = torch.where(largest == -INF, 0.0, e)
    logs = torch.where(x == -INF, -INF, torch.where(x == largest, 0.0, x - largest) - torch.log(e.sum(1, keepdim=True)))
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    return logs.gather(1, tokens.long()[:, None])[:, 0], order.int(), logs.gather(1, order)


# The sum of exponentials: every term is off by 2^-24 |x - largest| (the difference and its product with log2 e) plus two steps
# of the exponential, weighed by the term itself, so under (2 * 30 + 4) * 2^-24; a thread's additions (at most 1,000, in a row)
# and the joins add half a step each of a sum that grows, under 1,000 * 2^-24 in the worst case; the logarithm keeps that as an
# absolute error, and the final difference adds half a step of the result.
def near(got, want, what):
    got, want = got.double(), want.double()
    fine = want.isfinite()
    assert torch.equal(got[~fine], want[~fine]), what
    off = (got[fine] - want[fine]).abs() - 2.0 ** -23 * want[fine].abs()
    assert off.numel() == 0 or off.max() <= 1064 * 2.0 ** -24, (what, off.max())


@pytest.mark.parametrize("dtype", DTYPES, ids=names.get)
@pytest.mark.parametrize("vocab,top", [(1, 0), (1, 1), (2, 2), (7, 5), (128, 128), (271, 64), (1025, 1), (1025, 128), (4099, 20), (32003, 0),
                                       (50021, 20), (151936, 5), (151936, 128)])
def test_token_logprobs(vocab, top, dtype):
    gen = torch.Generator(DEV).manual_seed(vocab + top)
    x = torch.randn(9, vocab, device=DEV, generator=gen) * torch.tensor([0, 0.01, 0.5, 1, 2, 3, 5, 10, 20], device=DEV)[:, None]
    x = x.to(dtype)
    tokens = torch.randint(0, vocab, (9,), device=DEV, generator=gen, dtype=torch.int32)
    got, want = ops.token_logprobs(x, tokens, top), plain_logprobs(x, tokens, top)
    assert torch.equal(got[1], want[1])
    near(got[0], want[0], "token"); near(got[2], want[2], "top")
    wide = torch.full((9, vocab + 13), 60.0, dtype=dtype, device=DEV)
    wide[:, 3:3 + vocab] = x
    again = ops.token_logprobs(wide[:, 3:3 + vocab], tokens, top)
    assert torch.equal(got[1], again[1])
    near(again[0], want[0], "token"); near(again[2], want[2], "top")


@pytest.mark.parametrize("vocab", [50, 151936])
def test_token_logprobs_of_masked_rows(vocab):
    gen = torch.Generator(DEV).manual_seed(vocab)
    x = torch.randn(9, vocab, device=DEV, generator=gen) * 2
    x[0] = -INF
    x[1] = float("nan")
    x[2] = -INF; x[2, 17] = -4.0
    x[3] = torch.finfo(torch.float32).min
    x[4, ::2] = -INF
    x[5, ::3] = float("nan")
    x[6, 11] = INF; x[6, 3] = INF
    x[7] = torch.finfo(torch.float32).min; x[7, 5] = 2.0
    x[8] = torch.randn(vocab, device=DEV, generator=gen) * 1e30
    for token in (0, 3, 17, vocab - 1):
        tokens = torch.full((9,), token, dtype=torch.int32, device=DEV)
        got, want = ops.token_logprobs(x, tokens, 20), plain_logprobs(x, tokens, 20)
        assert torch.equal(got[1], want[1])
        near(got[0], want[0], "token"); near(got[2], want[2], "top")


def test_a_token_outside_the_vocabulary_is_reported():
    x = torch.randn(3, 100, device=DEV)
    ops.check_status(DEV)
    got = ops.token_logprobs(x, torch.tensor([5, 100, -1], dtype=torch.int32, device=DEV))[0]
    torch.cuda.synchronize()
    assert got.isnan().tolist() == [False, True, True]
    with pytest.raises(ops.KernelError, match="token id"):
        ops.check_status(DEV)
    ops.clear_status(DEV)


# ---------------------------------------------------------------------------------------------------------------- copies
def plain_copy(stores, src, dst, tokens, into):
    for a, b in zip(stores, into):
        new = a[:, src].clone()
        for i, d in enumerate(dst):
            t = a.shape[2] if tokens is None else tokens[i]
            b[:, d, :t] = new[:, i, :t]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8], ids=str)
@pytest.mark.parametrize("layers,pages,page,heads,dim", [(1, 3, 1, 1, 1), (36, 40, 16, 8, 128), (2, 50, 5, 1, 77), (7, 33, 8, 3, 33), (1, 2500, 4, 1, 24),
                                                         (3, 9, 64, 2, 576)])
def test_pages_are_copied(layers, pages, page, heads, dim, dtype):
    gen = np.random.RandomState(pages + dim)
    make = lambda n: [torch.from_numpy(gen.randint(-99, 99, (layers, n, page, heads, dim))).to(dtype).to(DEV) for _ in range(2)]  # noqa: E731
    for n, fan, part, into in ((1, 1, True, False), (pages // 3, 2, True, False), (max(1, pages // 8), 5, False, False), (pages - 1, 1, False, True),
                               (pages // 2, 1, True, True)):
        if not into and n * (1 + fan) > pages:
            continue
        where = gen.permutation(pages).tolist()
        src = [p for p in where[:n] for _ in range(fan)]
        dst = gen.permutation(n * fan + 3)[:n * fan].tolist() if into else where[n:n + n * fan]
        tokens = gen.randint(0, page + 1, n * fan).tolist() if part else None
        stores = make(pages)
        to = make(n * fan + 3) if into else stores
        want_from, want_to = [s.clone() for s in stores], [s.clone() for s in to]
        plain_copy(want_from, src, dst, tokens, want_to if into else want_from)
        ops.copy_pages(stores, src, dst, tokens=tokens, into=to if into else None)
        for got, want in zip(stores + to, want_from + (want_to if into else want_from)):
            assert torch.equal(got, want)


def test_pages_of_strided_stores():
    """Keys and values in one tensor, a slice of the layers, pages before layers, a base off 16-byte boundaries."""
    both = torch.randn(6, 2, 20, 4, 3, 8, device=DEV)
    want = both.clone()
    want[1:5, :, [3, 9]] = want[1:5, :, [7, 7]]
    ops.copy_pages([both[1:5, 0], both[1:5, 1]], [7, 7], torch.tensor([3, 9]))
    assert torch.equal(both, want)
    turned = torch.randn(20, 6, 4, 3, 8, device=DEV)
    want = turned.clone()
    want[[0, 19]] = want[[10, 11]]
    ops.copy_pages([turned.transpose(0, 1)], [10, 11], np.array([0, 19]))
    assert torch.equal(turned, want)
    flat = torch.randn(1 + 2 * 9 * 4 * 5, device=DEV)
    odd = flat[1:].view(2, 9, 4, 5)
    want = odd.clone()
    want[:, 2, :3] = want[:, 8, :3]
    ops.copy_pages([odd], [8], [2], tokens=[3])
    assert torch.equal(odd, want)


def test_pages_behind_four_gigabytes():
    store = torch.zeros((3, 70000, 16, 2, 512), dtype=torch.bfloat16, device=DEV)        # 6.9 GB
    store[:, 69990:69995] = torch.randn(3, 5, 16, 2, 512, device=DEV).bfloat16()
    ops.copy_pages([store], [69990, 69991, 69994], [69999, 0, 41234])
    for a, b in ((69990, 69999), (69991, 0), (69994, 41234)):
        assert torch.equal(store[:, a], store[:, b]) and store[:, b].any()


@pytest.mark.parametrize("n", [1, 5, 48, 130])
def test_slots_are_copied(n):
    """State tensors of many shapes and types, more of them than one launch takes."""
    gen = torch.Generator(DEV).manual_seed(n)
    shapes = [((7,), torch.float32), ((4, 3, 5), torch.bfloat16), ((32, 64, 64), torch.float32), ((1,), torch.bfloat16), ((), torch.float32), ((0, 3), torch.float32)]
    states = []
    for i in range(n):
        shape, dtype = shapes[i % len(shapes)]
        states.append(torch.randn((11, *shape), device=DEV, generator=gen).to(dtype))
    want = [s.clone() for s in states]
    src, dst = [3, 3, 10, 0], [1, 2, 9, 8]
    for s in want:
        s[dst] = s[src]
    ops.copy_slots(states, src, dst)
    for got, w in zip(states, want):
        assert torch.equal(got, w)


def test_copies_are_captured_with_their_pairs():
    store = torch.randn(5, 30, 16, 2, 64, device=DEV)
    state = torch.randn(9, 33, device=DEV)

    def call():
        ops.copy_pages([store], [4, 5], [6, 7], tokens=[16, 3])
        ops.copy_slots([state], [1], [2])

    graph, _ = graph_of(call)
    store.normal_(); state.normal_()
    want, want_state = store.clone(), state.clone()
    want[:, 6], want[:, 7, :3], want_state[2] = want[:, 4], want[:, 5, :3], want_state[1]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(store, want) and torch.equal(state, want_state)


# ---------------------------------------------------------------------------------------------------------- used together
def test_continuations_drawn_scored_and_forked():
    """A prompt's last logits sampled for six continuations, the tokens scored, and its pages and states forked for them, in one
    captured graph: the tokens and scores are the plain implementation's and every fork holds what its source holds."""
    gen = torch.Generator(DEV).manual_seed(21)
    n, vocab = 6, 30011
    logits = (torch.randn(1, vocab, device=DEV, generator=gen) * 3).repeat(n, 1)
    rows = [(0.8, 60, 0.95, 0.01, 1000 + i, 0) for i in range(n)]
    params = [torch.tensor(v, dtype=d, device=DEV) for v, d in zip(zip(*rows), (torch.float32, torch.int32, torch.float32, torch.float32,
                                                                                torch.int64, torch.int64))]
    k, v = (torch.randn(4, 64, 16, 2, 64, device=DEV, generator=gen).bfloat16() for _ in range(2))
    states = [torch.randn(8, 4, 16, 16, device=DEV, generator=gen) for _ in range(3)]

    def call():
        tokens = ops.sample_filtered(logits, *params)
        scores = ops.token_logprobs(logits, tokens, 4)
        ops.copy_pages([k, v], [9] * (n - 1), [20 + i for i in range(n - 1)], tokens=[11] * (n - 1))
        ops.copy_slots(states, [0] * (n - 1), list(range(1, n)))
        return tokens, scores

    graph, (tokens, scores) = graph_of(call)
    graph.replay()
    torch.cuda.synchronize()
    x = logits[0].double().cpu().numpy()
    for i, tok in enumerate(tokens.tolist()):
        t, kk, p, m, seed, counter = rows[i]
        assert tok in accepted(x, float(np.float32(t)), kk, float(np.float32(p)), float(np.float32(m)), seed, counter)
    want = plain_logprobs(logits, tokens, 4)
    assert torch.equal(scores[1], want[1])
    near(scores[0], want[0], "token"); near(scores[2], want[2], "top")
    for i in range(n - 1):
        assert torch.equal(k[:, 20 + i, :11], k[:, 9, :11]) and torch.equal(v[:, 20 + i, :11], v[:, 9, :11])
        assert all(torch.equal(s[1 + i], s[0]) for s in states)
    assert math.isfinite(scores[0].sum().item())

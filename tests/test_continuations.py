"""Continuations of one prompt, forks and pools that change their size, with a stand-in for the device (no GPU): what the
cache manager and the scheduler decide, and what the entry point refuses."""

import random
import threading

import pytest
import torch

from jax_vllm_b200 import registry
from jax_vllm_b200.cache import CacheManager, OutOfPages, PagePool
from jax_vllm_b200.engine import (SamplingParams, add_continuations, add_request, continuations, fork_request, generate, has_work, make_driver,
                                  resize_cache, start, step, stop, stream)
from jax_vllm_b200.parts import BuildContext, FixedStateNeed, Model, PagedKVNeed
from tests.test_scheduler import FakeRunner, next_token
from tests.util import TINY_A

VOCAB = TINY_A["vocab_size"]


class SeededSampler:
    """Token = largest logit + seed: every continuation goes its own way."""

    def sample(self, logits, temperatures, seeds, counters):
        assert len(temperatures) == len(seeds) == len(counters) == logits.shape[0]
        return (logits.argmax(-1) + torch.tensor(seeds)).remainder(VOCAB).to(torch.int32)


def expected(prompt, n, seed, eos=None):
    seq, out = list(prompt), []
    for _ in range(n):
        t = (next_token(seq) + seed) % VOCAB
        out.append(t); seq.append(t)
        if eos is not None and t == eos:
            break
    return out


def driver(**kw):
    model = Model(registry.config_from_dict(TINY_A).to_spec(), BuildContext(torch.float32, torch.device("cpu")))
    runner = FakeRunner()
    return make_driver(model, runner=runner, sampler=SeededSampler(), **kw), runner


# --------------------------------------------------------------------------------------------------- parameters
@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(top_k=1 << 31), dict(top_p=0.0), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=-0.1),
                                 dict(min_p=1.5), dict(min_p=float("nan")), dict(logprobs=-1), dict(logprobs=129)])
def test_parameters_that_are_refused(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)


def test_filters_matter_for_draws_only():
    assert not SamplingParams(top_k=5, top_p=0.5).filtered and not SamplingParams(temperature=1.0).filtered
    assert all(SamplingParams(temperature=1.0, **f).filtered for f in (dict(top_k=5), dict(top_p=0.5), dict(min_p=0.1)))


# --------------------------------------------------------------------------------------------------- cache manager
def manager(pages=20, live=6, prefix=True, **need):
    return CacheManager([PagedKVNeed(1, 4), PagedKVNeed(1, 4, **need) if need else None], 4, pages, live, prefix)


@pytest.mark.parametrize("tokens", [0, 1, 4, 7, 8, 13])
@pytest.mark.parametrize("need", [{}, {"window": 6}, {"chunk": 8}, {"window": 5, "keep_first": 3}])
def test_a_fork_shares_full_pages_and_owns_the_last(tokens, need):
    m = manager(pages=40, **need)
    a = m.admit("a")
    m.grow(a, tokens + 5)                              # pages ahead of its tokens are not the fork's
    m.commit(a, list(range(tokens)))
    kids = m.fork("a", ["b", "c"])
    m.check()
    full = tokens // 4
    for kid in kids:
        assert kid.num_tokens == tokens and kid.tokens == a.tokens and kid.hashes == a.hashes
        for g in range(len(m.groups)):
            assert kid.tables[g][:full] == a.tables[g][:full]
            assert len(kid.tables[g]) == -(-tokens // 4)
            if tokens % 4:
                assert kid.tables[g][full] not in (a.tables[g][full], -1)
    assert len({rc.slot for rc in m.live.values()}) == 3
    # each goes on by itself; pages come back one holder at a time
    for rc in (a, *kids):
        m.grow(rc, tokens + 9)
        m.commit(rc, [100 + rc.slot] * 9)
        m.check()
    for rid in ("a", "c", "b"):
        m.release(rid)
        m.check()
    assert all(g.pool.num_free == 40 for g in m.groups)


def test_a_fork_that_does_not_fit_changes_nothing():
    m = manager(pages=4, live=3)
    a = m.admit("a")
    m.grow(a, 10)
    m.commit(a, list(range(10)))
    before = (list(m.groups[0].pool.ref), m.groups[0].pool.free_pages(), m.slots.num_free)
    with pytest.raises(OutOfPages):
        m.fork("a", ["b", "c"])                       # one page is free
    with pytest.raises(RuntimeError):
        m.fork("a", ["b", "c", "d"])                  # two slots are
    for bad in (["a"], ["b", "b"]):
        with pytest.raises(KeyError):
            m.fork("a", bad)
    with pytest.raises(KeyError):
        m.fork("x", ["b"])
    assert before == (list(m.groups[0].pool.ref), m.groups[0].pool.free_pages(), m.slots.num_free)
    m.fork("a", ["b"])
    m.check()


def test_states_follow_a_fork_without_pages():
    m = CacheManager([FixedStateNeed((3,)), FixedStateNeed((2, 2))], 4, 1, 3, False)
    a = m.admit("a")
    m.commit(a, [1, 2, 3])
    b, = m.fork("a", ["b"])
    assert b.slot != a.slot and b.num_tokens == 3 and b.tables == []
    m.check()


def test_a_pool_of_another_size_keeps_what_is_held_and_what_is_known():
    pool = PagePool(8)
    for i in range(8):
        pool.alloc()
        pool.register(i, bytes([i]))
    pool.release([1, 3, 5, 6])                         # free, contents known; given out again in the order 6, 5, 3, 1
    assert pool.free_pages() == [6, 5, 3, 1]
    small, moved = pool.resized(6)
    small.check()
    assert moved == {0: 0, 2: 1, 4: 2, 7: 3, 3: 4, 1: 5}
    assert small.free_pages() == [4, 5] and [small.lookup(bytes([i])) for i in range(8)] == [0, 5, 1, 4, 2, None, None, 3]
    large, moved = pool.resized(11)
    large.check()
    assert large.num_free == 7 and large.free_pages()[-4:] == [moved[p] for p in (6, 5, 3, 1)] and sorted(moved) == list(range(8))
    assert all(large.lookup(bytes([p])) == moved[p] for p in range(8))
    with pytest.raises(OutOfPages):
        pool.resized(3)
    pool.check()


def test_resizing_moves_tables_and_keeps_prefixes():
    m = manager(pages=12)
    a = m.admit("a"); m.grow(a, 9); m.commit(a, list(range(9)))
    b = m.admit("b"); m.grow(b, 16); m.commit(b, list(range(50, 66)))
    m.release("a")
    content = {h: p for h, p in m.groups[0].pool.page_of_hash.items()}
    table = list(b.tables[0])
    m.resize(6)
    m.check()
    assert m.num_pages == 6 and sorted(b.tables[0]) == [0, 1, 2, 3] and list(b.tables[0]) == [sorted(table).index(p) for p in table]
    c = m.admit("c", list(range(9)) + [7])
    assert c.num_tokens == 8                           # the two full pages of `a` moved along
    m.check()
    with pytest.raises(OutOfPages):
        m.resize(5)
    with pytest.raises(ValueError):
        m.resize(0)
    m.check()
    assert set(m.groups[0].pool.page_of_hash) <= set(content)


# --------------------------------------------------------------------------------------------------- entry point
@pytest.mark.parametrize("n", [1, 2, 5])
@pytest.mark.parametrize("length", [1, 4, 11, 20])
def test_a_prompt_is_computed_once_for_all_its_continuations(length, n):
    d, r = driver(max_num_seqs=5, max_model_len=64, block_size=4, max_tokens_per_step=8)
    prompt = [(7 * i + 3) % VOCAB for i in range(length)]
    reqs = continuations(d, prompt, n, SamplingParams(max_new_tokens=6, seed=10))
    assert [q.output_ids for q in reqs] == [expected(prompt, 6, 10 + i) for i in range(n)]
    assert sum(k for batch in r.batches for _, k, _ in batch) == length + 5 * n       # every token ran once
    assert d.stats.forks == n - 1 and d.stats.finished == n and not has_work(d) and not d.cache.live
    assert d.stats.cache_hit_tokens == 0
    d.cache.check()


def test_continuations_beside_other_requests_with_few_slots_and_pages():
    d, r = driver(max_num_seqs=3, max_model_len=64, block_size=4, max_tokens_per_step=8, num_blocks=16)
    prompts = [[1, 2, 3], [9] * 17, [5]]
    ids = [i for p in prompts for i in add_continuations(d, p, 4, SamplingParams(max_new_tokens=9, seed=3))]
    reqs = [d.requests[i] for i in ids]
    while has_work(d):
        step(d)
        d.cache.check()
    want = [expected(p, 9, 3 + i) for p in prompts for i in range(4)]
    assert [q.output_ids for q in reqs] == want and all(q.finished for q in reqs)
    assert 0 < d.stats.forks < 9                       # some found no slot and were computed by themselves
    assert d.stats.finished == 12 and not d.cache.live


def test_continuations_that_end_with_their_first_token():
    d, _ = driver(max_num_seqs=2, max_model_len=64, block_size=4)
    prompt = [4, 5, 6]
    first = [expected(prompt, 1, s)[0] for s in range(3)]
    reqs = continuations(d, prompt, 3, [SamplingParams(max_new_tokens=1, seed=0), SamplingParams(max_new_tokens=5, seed=1),
                                        SamplingParams(max_new_tokens=5, seed=2, eos_id=first[2])])
    assert [q.output_ids for q in reqs] == [[first[0]], expected(prompt, 5, 1), [first[2]]]
    assert d.stats.finished == 3 and not d.cache.live and not has_work(d)
    d.cache.check()


def test_events_and_streams_of_continuations():
    from jax_vllm_b200 import stream
    d, _ = driver(max_num_seqs=3, max_model_len=64, block_size=4)
    ids = add_continuations(d, [3, 1, 4], 3, SamplingParams(max_new_tokens=4, seed=0))
    got = {i: [ev.token for ev in stream(d, i)] for i in reversed(ids)}
    assert [got[i] for i in ids] == [expected([3, 1, 4], 4, s) for s in range(3)]


def test_a_running_request_is_forked_where_it_stands():
    for steps in (0, 1, 3, 6):
        d, r = driver(max_num_seqs=3, max_model_len=64, block_size=4, max_tokens_per_step=4)
        prompt = [2, 7, 1, 8, 2, 8, 1, 8, 2]
        a = add_request(d, prompt, SamplingParams(max_new_tokens=10, seed=0))
        for _ in range(steps):
            step(d)
        so_far = list(d.requests[a].output_ids)
        b = fork_request(d, a, SamplingParams(max_new_tokens=10, seed=5))
        c = fork_request(d, a)                         # its own seed: its id
        reqs = [d.requests[i] for i in (a, b, c)]
        while has_work(d):
            step(d)
            d.cache.check()

        def after(seed):
            return so_far + expected(prompt + so_far, 10 - len(so_far), seed)
        assert [q.output_ids for q in reqs] == [after(0), after(5), after(c)]
        assert not d.cache.live


def test_what_the_entry_point_refuses():
    d, _ = driver(max_num_seqs=2, max_model_len=32, block_size=4, num_blocks=12)
    with pytest.raises(ValueError):
        add_continuations(d, [1], 0)
    with pytest.raises(ValueError):
        add_continuations(d, [1], 2, [SamplingParams()])
    with pytest.raises(ValueError):
        add_continuations(d, [1], 2, [SamplingParams(max_new_tokens=4), SamplingParams(max_new_tokens=40)])
    with pytest.raises(ValueError):
        add_continuations(d, [VOCAB], 2, SamplingParams(max_new_tokens=4))
    with pytest.raises(KeyError):
        fork_request(d, 99)
    assert not has_work(d) and not d.requests
    ids = add_continuations(d, [1, 2], 2, SamplingParams(max_new_tokens=4))
    with pytest.raises(ValueError):
        fork_request(d, ids[1])                        # waits for its prompt
    step(d)
    with pytest.raises(ValueError):
        fork_request(d, ids[0], SamplingParams(max_new_tokens=1))
    with pytest.raises(ValueError):
        resize_cache(d, 1)                             # an unfinished request may need two pages
    while has_work(d):
        step(d)
    with pytest.raises(KeyError):
        fork_request(d, ids[0])


def test_the_pool_changes_its_size_between_steps():
    d, _ = driver(max_num_seqs=3, max_model_len=64, block_size=4, num_blocks=40)
    prompts = [[1, 2, 3, 4, 5], [9] * 17, [5]]
    ids = [add_request(d, p, SamplingParams(max_new_tokens=12, seed=i)) for i, p in enumerate(prompts)]
    reqs = [d.requests[i] for i in ids]
    sizes = iter((18, 60, 16, 17, 40, 20))
    while has_work(d):
        step(d)
        size = next(sizes, None)
        if size is not None:
            resize_cache(d, size)
            assert d.cache.num_pages == size == d.num_blocks == d.stats.pages_total
        d.cache.check()
    assert [q.output_ids for q in reqs] == [expected(p, 12, i) for i, p in enumerate(prompts)]
    assert generate(d, prompts, SamplingParams(max_new_tokens=3, seed=1)) == [expected(p, 3, 1) for p in prompts]


def test_more_continuations_than_rows_at_a_time():
    d, r = driver(max_num_seqs=3, max_model_len=64, block_size=4)
    rows = []
    sample = d.sampler.sample
    d.sampler.sample = lambda logits, *a: rows.append(logits.shape[0]) or sample(logits, *a)
    reqs = continuations(d, [4, 5, 6], 150, SamplingParams(max_new_tokens=2, seed=0))
    assert [q.output_ids for q in reqs] == [expected([4, 5, 6], 2, i) for i in range(150)]
    assert rows[:3] == [64, 64, 22] and max(rows[3:]) <= 3
    d.cache.check()


def test_filters_and_scores_of_a_vocabulary_that_is_too_large_are_refused(monkeypatch):
    d, _ = driver(max_num_seqs=2, max_model_len=32, block_size=4)
    from jax_vllm_b200.engine import engine
    monkeypatch.setattr(engine, "MOST_VOCAB", VOCAB - 1)
    for sp in (SamplingParams(max_new_tokens=2, temperature=1.0, top_k=3), SamplingParams(max_new_tokens=2, logprobs=0)):
        with pytest.raises(ValueError):
            add_request(d, [1], sp)
        with pytest.raises(ValueError):
            add_continuations(d, [1], 2, sp)
        i = add_request(d, [1], SamplingParams(max_new_tokens=4, seed=0))
        with pytest.raises(ValueError):
            fork_request(d, i, sp)
    assert generate(d, [[1]], SamplingParams(max_new_tokens=2, temperature=1.0, seed=0)) == [expected([1], 2, 0)]


def test_a_pool_that_was_left_half_resized_takes_no_more_steps(monkeypatch):
    d, _ = driver(max_num_seqs=2, max_model_len=32, block_size=4, num_blocks=12)
    i = add_request(d, [1, 2, 3, 4, 5], SamplingParams(max_new_tokens=9, seed=0))
    step(d)
    with pytest.raises(ValueError):
        resize_cache(d, 1)
    assert d.cache.broken is None and step(d)

    def no_memory(*a):
        raise torch.OutOfMemoryError("no memory")
    monkeypatch.setattr(d.cache, "_move", no_memory)
    with pytest.raises(torch.OutOfMemoryError):
        resize_cache(d, 9)
    with pytest.raises(RuntimeError, match="half resized"):
        step(d)
    assert not d.requests[i].finished


def test_continuations_forks_and_sizes_from_several_threads():
    d, _ = driver(max_num_seqs=5, max_model_len=64, block_size=4, max_tokens_per_step=16, num_blocks=60)
    faults = []

    def work(k):
        r = random.Random(k)
        try:
            for _ in range(6):
                prompt = [r.randrange(VOCAB) for _ in range(r.randrange(1, 30))]
                ids = add_continuations(d, prompt, r.randrange(1, 6), SamplingParams(max_new_tokens=12, seed=k))
                for _ in range(2):
                    try:
                        f = fork_request(d, ids[0], SamplingParams(max_new_tokens=20, seed=k))
                        got = [e.token for e in stream(d, f)]
                        assert got == expected(prompt, 20, k)[20 - len(got):]
                    except KeyError:                   # it has finished
                        pass
                    try:
                        resize_cache(d, r.randrange(20, 80))
                    except ValueError:                 # too few pages for what is live
                        pass
                for i, rid in enumerate(ids):
                    assert [e.token for e in stream(d, rid)] == expected(prompt, 12, k + i)
        except BaseException as exc:
            faults.append(exc)

    start(d)
    threads = [threading.Thread(target=work, args=(k,), daemon=True) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not faults and not any(t.is_alive() for t in threads) and d.router.failure is None
    stop(d)
    d.cache.check()
    assert not d.cache.live and not d.requests

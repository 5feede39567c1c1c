"""Steps, forks and sizes on several streams and from several threads on the GPU: the tokens of one stream and one thread."""

import random
import threading

import pytest
import torch

from tests.util import PAGE_SIZE, TINY, make_folder, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    from jax_vllm_b200 import load_from_path
    return load_from_path(make_folder(tmp_path_factory.mktemp("order"), "a", seed=6), dtype="fp32")


P, VOCAB = PAGE_SIZE["a"], TINY["a"]["vocab_size"]


def driver(model, **kw):
    from jax_vllm_b200 import make_driver
    return make_driver(model, **{**dict(max_num_seqs=5, max_model_len=96, block_size=P), **kw})


def params(n, length=12):
    from jax_vllm_b200 import SamplingParams
    return [SamplingParams(max_new_tokens=length, temperature=0.9, top_p=0.95, seed=300 + i) for i in range(n)]


@pytest.mark.parametrize("portions", [False, True], ids=["whole prompt", "in portions"])
def test_steps_on_streams_in_turn(model, portions):
    """Every step on another stream than the last; each stream is busy (20 million clocks, 10 ms) before it gets to the step's
    last work, so that nothing but the engine's own order keeps the next step behind it."""
    from jax_vllm_b200 import add_continuations, continuations, has_work, step
    prompt = random_tokens(2 * P + 3, VOCAB, seed=41)
    kw = dict(max_tokens_per_step=P + 1) if portions else {}
    want = [r.output_ids for r in continuations(driver(model, **kw), prompt, 4, params(4))]
    d = driver(model, **kw)
    fork, run = d.cache.fork, d.runner.step

    def late_fork(*a):
        torch.cuda._sleep(20_000_000)
        return fork(*a)

    def late_step(entries):
        if portions:
            torch.cuda._sleep(20_000_000)
        return run(entries)
    d.cache.fork, d.runner.step = late_fork, late_step
    reqs = [d.requests[i] for i in add_continuations(d, prompt, 4, params(4))]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    k = 0
    while has_work(d):
        with torch.cuda.stream(streams[k % 3]):
            step(d)
        k += 1
    assert d.stats.forks == 3
    assert [r.output_ids for r in reqs] == want


def test_a_fork_waits_for_nothing_but_the_cache(model):
    """A request is forked while a stream that has nothing to do with the engine is busy (a second or so): the call returns
    before that has ended, and the fork's tokens are the ones that it has to give."""
    from jax_vllm_b200 import add_request, fork_request, has_work, step
    prompt = random_tokens(P + 3, VOCAB, seed=43)
    d = driver(model)
    a = add_request(d, prompt, params(1)[0])
    for _ in range(4):
        step(d)
    torch.cuda.synchronize()
    other, side, done = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(other):
        torch.cuda._sleep(1_500_000_000)
        done.record()
    with torch.cuda.stream(side):
        b = fork_request(d, a, params(1)[0])
    assert not done.query()
    reqs = [d.requests[i] for i in (a, b)]
    while has_work(d):
        step(d)
    assert reqs[0].output_ids == reqs[1].output_ids and d.stats.forks == 1


def test_a_refused_size_keeps_the_captured_steps(model):
    from jax_vllm_b200 import generate, resize_cache
    d = driver(model, num_blocks=40)
    prompts = [random_tokens(n, VOCAB, seed=50 + n) for n in (5, 9)]
    want = generate(d, prompts, params(2))
    kept = {n: g for n, g in d.runner.graphs_filtered.items()}
    assert kept
    page = sum(t.nbytes for g in d.cache.groups for t in (g.k, g.v)) // 40
    for size in (0, (1 << 39) // page):                # none, and three times what the device has
        with pytest.raises(ValueError):
            resize_cache(d, size)
    assert d.runner.graphs_filtered == kept
    assert generate(d, prompts, params(2)) == want
    resize_cache(d, 41)
    assert not d.runner.graphs_filtered
    assert generate(d, prompts, params(2)) == want


def test_prewarming_captures_the_steps_with_filters_too(model):
    from jax_vllm_b200 import generate, prewarm
    prompts = [random_tokens(n, VOCAB, seed=60 + n) for n in (5, 19, 2)]
    want = generate(driver(model, max_num_seqs=3), prompts, params(3))
    d = driver(model, max_num_seqs=3)
    prewarm(d)
    assert sorted(d.runner.graphs_sampled) == sorted(d.runner.graphs_filtered) == [1, 2, 3]
    d.cache.check()
    assert not d.cache.live
    kept = dict(d.runner.graphs_filtered)
    assert generate(d, prompts, params(3)) == want
    assert d.runner.graphs_filtered == kept and d.runner.graph_replays > 10


def test_continuations_of_several_lengths_from_several_threads(model):
    """Threads that add continuations with limits of their own, fork them and change the pool's size while the engine's thread
    steps (a size that is too small for what is live is refused).  Every token is that of the request alone."""
    from jax_vllm_b200 import SamplingParams, add_continuations, fork_request, generate, resize_cache, start, stop, stream
    prompts = [random_tokens(n, VOCAB, seed=70 + n) for n in (3, P, 2 * P + 1)]
    limits = (4, 30, 11)
    sp = lambda k, i: SamplingParams(max_new_tokens=limits[(k + i) % 3], temperature=0.9, top_k=30, top_p=0.95, seed=1000 * k + i)  # noqa: E731
    alone = driver(model, max_num_seqs=1)
    want = {(k, i): generate(alone, [prompts[k % 3]], sp(k, i))[0] for k in range(4) for i in range(3)}
    d = driver(model, num_blocks=40)
    faults = []

    def work(k):
        r = random.Random(k)
        try:
            for _ in range(3):
                ids = add_continuations(d, prompts[k % 3], 3, [sp(k, i) for i in range(3)])
                try:
                    f = fork_request(d, ids[0], sp(k, 0))
                    got = [e.token for e in stream(d, f)]
                    assert got == want[k, 0][len(want[k, 0]) - len(got):]
                except (KeyError, ValueError):         # it has finished, or has as many tokens as it may
                    pass
                try:
                    resize_cache(d, r.randrange(5, 60))
                except ValueError:                     # too few pages for what is live
                    pass
                for i, rid in enumerate(ids):
                    assert [e.token for e in stream(d, rid)] == want[k, i]
        except BaseException as exc:
            faults.append(exc)

    start(d)
    threads = [threading.Thread(target=work, args=(k,), daemon=True) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not faults and not any(t.is_alive() for t in threads) and d.router.failure is None
    stop(d)
    d.cache.check()
    assert not d.cache.live and not d.requests

"""Filters, log-probabilities, continuations, forks and pools of another size through the entry point on the GPU: tokens are
the plain implementation's where it decides them, and the same with and without captured steps, beside other requests or
alone, forked or computed by themselves."""

import importlib

import pytest
import torch

from tests.plain.qwen3_plain import PlainModel
from tests.util import PAGE_SIZE, TINY, make_folder, random_tokens

pytestmark = pytest.mark.gpu

# 32-bit logits of the engine lie within 1e-4 of the plain implementation's (the limit of the tests that compare them)
LOGITS = 1e-4


@pytest.fixture(scope="module", params=["a", "b", "d"])
def setup(request, tmp_path_factory):
    from jax_vllm_b200 import load_from_path
    tag = request.param
    folder = make_folder(tmp_path_factory.mktemp(f"cont_{tag}"), tag, seed=6)
    return tag, PlainModel(folder), load_from_path(folder, dtype="fp32")


def driver(model, tag, **kw):
    from jax_vllm_b200 import make_driver
    return make_driver(model, **{**dict(max_num_seqs=4, max_model_len=96, block_size=PAGE_SIZE[tag]), **kw})


def test_filtered_tokens_pass_the_filters_of_the_plain_logits(setup):
    """Every sampled token is one that the plain logits' filters leave, with room for the logits' difference: a probability
    beside the largest is off by a factor of exp(2 * 1e-4 / T), a rank by the tokens within 2e-4."""
    from jax_vllm_b200 import SamplingParams, generate
    tag, plain, model = setup
    prompts = [random_tokens(n, TINY[tag]["vocab_size"], seed=300 + n) for n in (3, 18, 26, 9)]
    params = [SamplingParams(max_new_tokens=20, temperature=0.9, top_k=4, seed=1), SamplingParams(max_new_tokens=20, temperature=1.2, top_p=0.6, seed=2),
              SamplingParams(max_new_tokens=20, temperature=1.0, min_p=0.5, seed=3),
              SamplingParams(max_new_tokens=20, temperature=0.7, top_k=30, top_p=0.8, min_p=0.1, seed=4)]
    got = generate(driver(model, tag), prompts, params)
    some = 0
    for p, sp, out in zip(prompts, params, got):
        logits = plain.logits(p + out[:-1]).double()[len(p) - 1:]
        for x, tok in zip(logits, out):
            rank = int((x > x[tok] + 2 * LOGITS).sum())
            share = torch.exp((x - x.max()) / sp.temperature)
            slack = 2 * LOGITS / sp.temperature * 2
            assert sp.top_k == 0 or rank < sp.top_k
            assert share[tok] >= sp.min_p * (1 - slack)
            kept = share[share >= sp.min_p].sort(descending=True).values[:sp.top_k or None]
            assert sp.top_p == 1 or kept[:rank].sum() < sp.top_p * kept.sum() * (1 + 2 * slack)
            some += rank > 0
    assert some > 10                                   # they are draws, not the largest logit each time


def test_a_filter_that_leaves_one_token_is_greedy(setup):
    from jax_vllm_b200 import SamplingParams, generate
    tag, plain, model = setup
    prompts = [random_tokens(n, TINY[tag]["vocab_size"], seed=20 + n) for n in (5, 17, 33)]
    want = [plain.greedy(p, 8) for p in prompts]
    for f in (dict(top_k=1), dict(top_p=1e-6), dict(min_p=1.0)):
        assert generate(driver(model, tag), prompts, SamplingParams(max_new_tokens=8, temperature=1.5, **f)) == want


def test_the_same_tokens_captured_or_not_alone_or_beside_others(setup):
    from jax_vllm_b200 import SamplingParams, generate
    tag, _, model = setup
    vocab = TINY[tag]["vocab_size"]
    prompts = [random_tokens(n, vocab, seed=400 + n) for n in (7, 1, 30, 12, 5)]
    params = [SamplingParams(max_new_tokens=15, temperature=0.8, top_p=0.9, seed=11), SamplingParams(max_new_tokens=9),
              SamplingParams(max_new_tokens=15, temperature=1.0, seed=12), SamplingParams(max_new_tokens=12, temperature=1.1, top_k=7, seed=13),
              SamplingParams(max_new_tokens=15, temperature=0.6, min_p=0.02, top_k=90, top_p=0.99, seed=14)]
    captured = driver(model, tag, prefix_cache=False)
    together = generate(captured, prompts, params)
    assert captured.runner.graphs_filtered and captured.runner.graph_replays > 10
    assert generate(captured, prompts, params) == together                   # from graphs captured before
    eager = driver(model, tag, cuda_graphs=False)
    assert generate(eager, prompts, params) == together
    alone = driver(model, tag, max_num_seqs=1)
    assert [generate(alone, [p], sp)[0] for p, sp in zip(prompts, params)] == together


def test_log_probabilities_are_the_plain_logits(setup):
    from jax_vllm_b200 import SamplingParams, add_request, step, has_work
    tag, plain, model = setup
    vocab = TINY[tag]["vocab_size"]
    d = driver(model, tag)
    prompts = [random_tokens(n, vocab, seed=500 + n) for n in (4, 21, 11)]
    params = [SamplingParams(max_new_tokens=8, logprobs=5), SamplingParams(max_new_tokens=6, temperature=0.9, top_k=8, seed=2, logprobs=0),
              SamplingParams(max_new_tokens=7)]
    ids = [add_request(d, p, sp) for p, sp in zip(prompts, params)]
    reqs = [d.requests[i] for i in ids]
    events = {i: [] for i in ids}
    while has_work(d):
        for ev in step(d):
            events[ev.request_id].append(ev)
    for i, p, sp, req in zip(ids, prompts, params, reqs):
        logs = torch.log_softmax(plain.logits(p + req.output_ids[:-1]).double(), -1)[len(p) - 1:]
        for ev, row in zip(events[i], logs):
            if sp.logprobs is None:
                assert ev.logprob is None and ev.top_logprobs is None
                continue
            assert abs(ev.logprob - row[ev.token].item()) <= 3 * LOGITS
            assert len(ev.top_logprobs) == sp.logprobs
            best = row.topk(max(sp.logprobs, 1)).values.tolist()
            for (tok, lp), b in zip(ev.top_logprobs, best):
                assert abs(lp - b) <= 3 * LOGITS and abs(lp - row[tok].item()) <= 3 * LOGITS
        assert req.logprobs == [ev.logprob for ev in events[i] if ev.logprob is not None]


def test_continuations_are_the_requests_that_they_would_be_alone(setup):
    from jax_vllm_b200 import SamplingParams, continuations, generate
    tag, _, model = setup
    P, vocab = PAGE_SIZE[tag], TINY[tag]["vocab_size"]
    for length in (1, P - 1, P, 2 * P + 3):
        prompt = random_tokens(length, vocab, seed=600 + length)
        sp = SamplingParams(max_new_tokens=P + 5, temperature=0.9, top_p=0.95, seed=40)
        d = driver(model, tag, prefix_cache=False)
        reqs = continuations(d, prompt, 4, sp)
        d.cache.check()
        assert not d.cache.live and d.stats.forks == 3
        want = [generate(driver(model, tag, max_num_seqs=1), [prompt], SamplingParams(max_new_tokens=P + 5, temperature=0.9, top_p=0.95, seed=40 + i))[0]
                for i in range(4)]
        assert [r.output_ids for r in reqs] == want
        # more continuations than places: the others are computed by themselves, with the same tokens
        small = driver(model, tag, max_num_seqs=2)
        assert [r.output_ids for r in continuations(small, prompt, 4, sp)] == want


def test_the_likeliest_of_several_continuations(setup):
    from jax_vllm_b200 import SamplingParams, continuations
    tag, plain, model = setup
    prompt = random_tokens(10, TINY[tag]["vocab_size"], seed=71)
    reqs = continuations(driver(model, tag), prompt, 4, SamplingParams(max_new_tokens=6, temperature=1.0, top_k=20, seed=5, logprobs=0))
    for r in reqs:
        logs = torch.log_softmax(plain.logits(prompt + r.output_ids[:-1]).double(), -1)[len(prompt) - 1:]
        assert abs(sum(r.logprobs) - sum(logs[k, t].item() for k, t in enumerate(r.output_ids))) <= 6 * 3 * LOGITS


def test_a_forked_request_goes_on_as_the_other_would(setup):
    from jax_vllm_b200 import SamplingParams, add_request, fork_request, has_work, step
    tag, plain, model = setup
    prompt = random_tokens(2 * PAGE_SIZE[tag] + 1, TINY[tag]["vocab_size"], seed=81)
    want = plain.greedy(prompt, 14)
    for steps in (1, 4, 9):
        d = driver(model, tag)
        a = add_request(d, prompt, SamplingParams(max_new_tokens=14))
        for _ in range(steps):
            step(d)
        b = fork_request(d, a)
        reqs = [d.requests[i] for i in (a, b)]
        while has_work(d):
            step(d)
        assert [r.output_ids for r in reqs] == [want, want] and d.stats.forks == 1
        d.cache.check()


def test_a_pool_of_another_size_between_steps(setup):
    from jax_vllm_b200 import SamplingParams, add_request, generate, has_work, resize_cache, step
    tag, plain, model = setup
    P, vocab = PAGE_SIZE[tag], TINY[tag]["vocab_size"]
    prompts = [random_tokens(n, vocab, seed=900 + n) for n in (2 * P + 3, 5, P)]
    want = [plain.greedy(p, 20) for p in prompts]
    most = -(-(2 * P + 23) // P)
    d = driver(model, tag, num_blocks=30)
    reqs = [d.requests[add_request(d, p, SamplingParams(max_new_tokens=20))] for p in prompts]
    sizes = iter((3 * most, 64, 2 * most + 6, 40))
    k = 0
    while has_work(d):
        step(d)
        k += 1
        size = next(sizes, None) if k % 3 == 0 else None
        if size is not None:
            resize_cache(d, size)
            assert all(g.k.shape[1] == size and g.v.shape[1] == size for g in d.cache.groups)
            d.cache.check()
    assert [r.output_ids for r in reqs] == want
    resize_cache(d, 64)
    page = sum(t.nbytes for g in d.cache.groups for t in (g.k, g.v)) // 64
    with pytest.raises(ValueError, match="device memory"):
        resize_cache(d, (1 << 39) // page)             # three times what the device has
    assert d.cache.num_pages == 64
    assert generate(d, prompts, SamplingParams(max_new_tokens=20)) == want    # prefixes that moved along among them
    assert d.stats.cache_hit_tokens > 0


# models with recurrent states, windows, chunks, rows shared by keys and values, layers that read another's cache
@pytest.mark.parametrize("family,tag", [("nufapel", "na"), ("nufapel", "nb"), ("gogivik", "ga"), ("gogivik", "gb"), ("nasedra", "na"), ("nasedra", "nd"),
                                        ("guronex", "ga"), ("tidarax", None), ("loselix", None)])
def test_continuations_and_forks_of_every_kind_of_cache(family, tag, tmp_path):
    from jax_vllm_b200 import SamplingParams, add_request, continuations, fork_request, generate, has_work, load_from_path, make_driver, resize_cache, step
    util = importlib.import_module(f"tests.{family}_util")
    tag = tag or sorted(util.CONFIGS)[0]
    c = util.CONFIGS[tag]
    folder = util.write_folder(tmp_path / "m", c, util.make_weights(c, 3))
    model = load_from_path(folder, dtype="fp32")
    vocab = model.spec.vocab_size
    make = lambda live: make_driver(model, max_num_seqs=live, max_model_len=96, block_size=util.PAGE[tag], prefix_cache=False)  # noqa: E731
    prompt = random_tokens(29, vocab, seed=7)
    sp = [SamplingParams(max_new_tokens=14, temperature=0.8, top_k=25, seed=70 + i) for i in range(3)]
    alone = make(1)
    want = [generate(alone, [prompt], s)[0] for s in sp]
    d = make(3)
    assert [r.output_ids for r in continuations(d, prompt, 3, sp)] == want and d.stats.forks == 2
    a = add_request(d, prompt, sp[0])
    for _ in range(5):
        step(d)
    b = fork_request(d, a, sp[0])
    reqs = [d.requests[i] for i in (a, b)]
    if d.cache.groups:
        resize_cache(d, d.cache.num_pages + 5)
    while has_work(d):
        step(d)
    assert [r.output_ids for r in reqs] == [want[0], want[0]]
    d.cache.check()
    assert not d.cache.live


@pytest.mark.parametrize("family,tag", [("nufapel", "na"), ("gogivik", "ga"), ("nasedra", "na"), ("guronex", "ga"), ("tidarax", None), ("loselix", None)])
def test_more_continuations_than_slots_and_pages(family, tag, tmp_path):
    """Some are forked, some wait, some are preempted and computed again; a request is forked in the middle of its prompt."""
    from jax_vllm_b200 import SamplingParams, add_continuations, add_request, fork_request, generate, has_work, load_from_path, make_driver, step
    util = importlib.import_module(f"tests.{family}_util")
    tag = tag or sorted(util.CONFIGS)[0]
    c = util.CONFIGS[tag]
    folder = util.write_folder(tmp_path / "m", c, util.make_weights(c, 5))
    model = load_from_path(folder, dtype="fp32")
    vocab, P = model.spec.vocab_size, util.PAGE[tag]
    prompt, other = random_tokens(2 * P + 3, vocab, seed=17), random_tokens(3 * P + 1, vocab, seed=18)
    sp = [SamplingParams(max_new_tokens=P + 6, temperature=0.9, top_p=0.95, seed=170 + i) for i in range(7)]
    alone = make_driver(model, max_num_seqs=1, max_model_len=6 * P, block_size=P)
    want = [generate(alone, [prompt], s)[0] for s in sp]
    want_other = generate(alone, [other], sp[0])[0]
    d = make_driver(model, max_num_seqs=4, max_model_len=6 * P, block_size=P, num_blocks=11, max_tokens_per_step=2 * P)
    a = add_request(d, other, sp[0])
    step(d)                                            # a part of its prompt
    b = fork_request(d, a, sp[0])
    ids = add_continuations(d, prompt, 7, sp)
    reqs = [d.requests[i] for i in [a, b] + ids]
    while has_work(d):
        step(d)
        d.cache.check()
    assert [r.output_ids for r in reqs] == [want_other, want_other] + want
    assert d.stats.forks > 1 and not d.cache.live


def test_command_line_and_class(tmp_path):
    """cli.py and LLM as a user calls them: the continuations, their tokens and log-probabilities are the entry point's."""
    import json, os, subprocess, sys
    from pathlib import Path
    from jax_vllm_b200 import LLM, SamplingParams
    folder = make_folder(tmp_path / "m", "a", seed=6)
    root = Path(__file__).resolve().parent.parent
    prompts = [random_tokens(n, TINY["a"]["vocab_size"], seed=1300 + n) for n in (9, 21)]
    cmd = [sys.executable, str(root / "cli.py"), "--model-path", str(folder), "--dtype", "fp32", "--max-tokens", "6", "--max-model-len", "64",
           "--block-size", str(PAGE_SIZE["a"]), "--temperature", "0.7", "--top-k", "30", "--top-p", "0.9", "--min-p", "0.01", "--seed", "5",
           "--n", "3", "--logprobs", "2"]
    for p in prompts:
        cmd += ["--prompt-ids", ",".join(map(str, p))]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=600, cwd=str(root), env=dict(os.environ))
    assert out.returncode == 0, out.stderr[-2000:]
    got = [json.loads(line) for line in out.stdout.splitlines() if line.startswith("{")]
    llm = LLM(folder, dtype="fp32", max_num_seqs=4, max_model_len=64, block_size=PAGE_SIZE["a"])
    want = [r for i, p in enumerate(prompts)
            for r in llm.continuations(p, 3, SamplingParams(max_new_tokens=6, temperature=0.7, top_k=30, top_p=0.9, min_p=0.01, seed=5 + 3 * i, logprobs=2))]
    assert [g["output_ids"] for g in got] == [r.output_ids for r in want]
    for g, r in zip(got, want):
        assert len(g["logprobs"]) == 6 and [[t for t, _ in step] for step in g["top_logprobs"]] == [[t for t, _ in step] for step in r.top_logprobs]
        # log-probabilities of logits that lie within LOGITS of the plain ones differ by twice that at most, those of two runs by four times
        assert max(abs(a - b) for a, b in zip(g["logprobs"], r.logprobs)) <= 4 * LOGITS
    i = llm.add_request(prompts[0], SamplingParams(max_new_tokens=8))
    llm.step()
    j = llm.fork_request(i)
    llm.resize_cache(llm.driver.num_blocks + 1)
    first, second = llm.driver.requests[i], llm.driver.requests[j]
    while llm.has_work():
        llm.step()
    assert first.output_ids == second.output_ids and len(first.output_ids) == 8

"""Continuations, forks and sizes that meet one another, with a stand-in for the device (no GPU)."""

import threading

import pytest
import torch

from jax_vllm_b200.engine import SamplingParams, add_continuations, add_request, fork_request, has_work, prewarm, resize_cache, step
from jax_vllm_b200.engine import engine as eng
from tests.test_continuations import driver, expected


def resized_on_the_way(monkeypatch, d, num_blocks):
    """Another thread asks for a pool of another size at the moment at which the engine makes its next request record.
    Returns the function that ends that thread, and what it was refused with, if it was."""
    refused, made = [], eng._new_request

    def other():
        try:
            resize_cache(d, num_blocks)
        except ValueError as exc:
            refused.append(exc)
    thread = threading.Thread(target=other, daemon=True)

    def new_request(*a, **k):
        if not thread.is_alive() and thread.ident is None:
            thread.start()
            thread.join(0.5)                           # it may have to wait for this request
        return made(*a, **k)
    monkeypatch.setattr(eng, "_new_request", new_request)

    def end():
        thread.join(30)
        assert not thread.is_alive()
        return refused
    return end


@pytest.mark.parametrize("limits", [(4, 40), (40, 4), (4, 4, 40)])
def test_a_smaller_pool_and_continuations_of_several_lengths(monkeypatch, limits):
    """Either the pool is smaller and the continuations are refused, or they are there and the smaller pool is: never both."""
    d, _ = driver(max_num_seqs=4, max_model_len=64, block_size=4, num_blocks=16)
    end = resized_on_the_way(monkeypatch, d, 3)
    params = [SamplingParams(max_new_tokens=n, seed=i) for i, n in enumerate(limits)]
    try:
        ids = add_continuations(d, [1, 2, 3], len(limits), params)
    except ValueError:
        end()
        assert not d.requests and not d.router._queues and not has_work(d)
        return
    reqs = [d.requests[i] for i in ids]
    assert end() and d.cache.num_pages == 16           # the continuations came first
    while has_work(d):
        step(d)
        d.cache.check()
    assert [r.output_ids for r in reqs] == [expected([1, 2, 3], n, i) for i, n in enumerate(limits)]


def test_a_smaller_pool_and_a_request(monkeypatch):
    d, _ = driver(max_num_seqs=2, max_model_len=64, block_size=4, num_blocks=16)
    end = resized_on_the_way(monkeypatch, d, 3)
    try:
        i = add_request(d, [1, 2, 3], SamplingParams(max_new_tokens=40, seed=0))
    except ValueError:
        end()
        assert not d.requests and not d.router._queues and not has_work(d)
        return
    req = d.requests[i]
    assert end()
    while has_work(d):
        step(d)
    assert req.output_ids == expected([1, 2, 3], 40, 0)


def test_what_is_refused_leaves_nothing_behind():
    """A pool that became too small before the request was made."""
    d, _ = driver(max_num_seqs=2, max_model_len=64, block_size=4, num_blocks=16)
    resize_cache(d, 3)
    for call in (lambda: add_request(d, [1], SamplingParams(max_new_tokens=40)),
                 lambda: add_continuations(d, [1], 2, [SamplingParams(max_new_tokens=4), SamplingParams(max_new_tokens=40)])):
        with pytest.raises(ValueError, match="pages"):
            call()
        assert not d.requests and not d.router._queues and not has_work(d)


# ------------------------------------------------------------------------------------------------------ work in flight
@pytest.mark.parametrize("n", [1, 3])
def test_the_next_step_follows_what_a_step_leaves_running(n):
    """A portion of a prompt without logits, and the copies for forks, are not waited for: the runner is told, after them, and
    asked to follow them before anything else is issued."""
    d, r = driver(max_num_seqs=4, max_model_len=64, block_size=4, max_tokens_per_step=8)
    log = []
    r.leave, r.follow = lambda: log.append("leave"), lambda: log.append("follow")
    run, fork, admit = r.step, d.cache.fork, d.cache.admit
    r.step = lambda entries: log.append("step") or run(entries)
    d.cache.fork = lambda *a: log.append("fork") or fork(*a)
    d.cache.admit = lambda *a: log.append("admit") or admit(*a)          # clears state rows on the device
    add_continuations(d, [5] * 13, n, SamplingParams(max_new_tokens=4, seed=0))
    step(d)                                            # eight tokens of the prompt
    assert log == ["follow", "admit", "step", "leave"]
    del log[:]
    step(d)                                            # the rest, and the first tokens
    assert log == ["follow", "step"] + (["fork", "leave"] if n > 1 else [])
    del log[:]
    step(d)
    assert log == ["follow", "step"]


def test_a_fork_between_steps_is_ordered_like_a_step():
    d, r = driver(max_num_seqs=4, max_model_len=64, block_size=4)
    a = add_request(d, [5] * 6, SamplingParams(max_new_tokens=6, seed=0))
    step(d)
    log = []
    r.leave, r.follow = lambda: log.append("leave"), lambda: log.append("follow")
    fork = d.cache.fork
    d.cache.fork = lambda *a: log.append("fork") or fork(*a)
    fork_request(d, a)
    assert log == ["follow", "fork", "leave"]


def test_prewarming_is_ordered_like_a_step():
    d, r = driver(max_num_seqs=2, max_model_len=64, block_size=4)
    log = []
    r.leave, r.follow = lambda: log.append("leave"), lambda: log.append("follow")
    r.warm_up = lambda decode_batches: log.append(("warm", decode_batches))
    prewarm(d)
    assert log == ["follow", ("warm", 2), "leave"]


# --------------------------------------------------------------------------------------------------------------- sizes
def test_a_size_that_is_refused_costs_no_captured_step(monkeypatch):
    """Too small for what is live, too large for the device: both before the runner drops its captured steps."""
    d, r = driver(max_num_seqs=2, max_model_len=64, block_size=4, num_blocks=16)
    forgotten = []
    r.forget_graphs = lambda: forgotten.append(d.cache.num_pages)
    add_request(d, [1, 2, 3], SamplingParams(max_new_tokens=20, seed=0))
    step(d)
    ahead = d.ahead
    with pytest.raises(ValueError):
        resize_cache(d, 3)
    device = torch.device("cuda")
    monkeypatch.setattr(type(d.cache), "_stores", lambda self: [FakeStore(device, 1 << 20, 16)])
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (5 << 20, 9 << 20))
    monkeypatch.setattr(torch.cuda, "memory_reserved", lambda device: 3 << 20)
    monkeypatch.setattr(torch.cuda, "memory_allocated", lambda device: 1 << 20)
    with pytest.raises(ValueError, match="device memory"):
        resize_cache(d, 16 * 8)                        # 8 MB; 5 are free and 2 more without captured steps
    assert not forgotten and d.ahead is ahead and d.cache.num_pages == 16
    with pytest.raises(ValueError, match="device memory"):
        resize_cache(d, 16 * 6)                        # 6 MB: they go, and leave no more than before here
    assert forgotten == [16] and d.cache.num_pages == 16 and d.cache.broken is None


class FakeStore:
    """What the check of the room asks of a store."""

    def __init__(self, device, nbytes, pages):
        self.device, self.nbytes, self.shape = device, nbytes, (1, pages)


def test_what_the_entry_point_issues_goes_to_the_driver_s_device(monkeypatch):
    """A driver of the second GPU, used while the first is the current one (both stand-ins): the runner, the sampler, the copies
    of forks and of a resize all find the driver's device current."""
    d, r = driver(max_num_seqs=4, max_model_len=64, block_size=4)
    current, seen = ["cuda:0"], []

    class Device:
        def __init__(self, device):
            self.device = str(device)

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *a):
            current.pop()
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    object.__setattr__(d.config, "device", "cuda:1")

    def watched(owner, name):
        call = getattr(owner, name)
        setattr(owner, name, lambda *a: seen.append((name, current[-1])) or call(*a))
    for owner, name in ((r, "step"), (d.sampler, "sample"), (d.cache, "fork"), (d.cache, "resize")):
        watched(owner, name)
    add_continuations(d, [5] * 6, 2, SamplingParams(max_new_tokens=6, seed=0))
    step(d)
    fork_request(d, 0)
    resize_cache(d, d.num_blocks + 1)
    step(d)
    assert [name for name, _ in seen] == ["step", "sample", "fork", "fork", "resize", "step", "sample"]
    assert {device for _, device in seen} == {"cuda:1"} and current == ["cuda:0"]

"""The engine's programming entry point, in the manner of the reference's
(jllm/engine/engine.py:63-233): `make_driver`, `add_request`, `step`, `has_work`,
`stream`, `start`, `stop`, `prewarm`, with the same names and meanings of arguments
(max_num_seqs, max_model_len, max_prefill_len, block_size, num_blocks, dtype), token ids
in and out.  `step` admits, runs ONE batch on the device (decoded tokens and prompt
portions together) and returns the events of the tokens it produced.

Beyond the reference's: `add_continuations` continues one prompt in several ways and computes it
once, `fork_request` branches a request where it stands, `resize_cache` gives the pool of pages
another size while requests live.
"""

from __future__ import annotations

import contextlib
import threading
import time
import weakref
from dataclasses import replace
from typing import Iterator, Optional

import torch

from ..cache import CacheManager
from ..config import EngineConfig, parse_dtype
from ..ops import MOST_VOCAB
from ..sampling import Sampler
from .background import EventRouter
from .batch import StepEntry
from .request import EngineStats, Request, SamplingParams, StepEvent
from .runner import Runner
from .scheduler import Scheduler


class Driver:
    def __init__(self, model, config: EngineConfig, runner=None, sampler=None):
        """`runner` and `sampler` default to the device ones; tests of the scheduling pass
        stand-ins with the same `step`/`sample` methods."""
        self.model, self.config = model, config
        self.max_num_seqs, self.max_model_len = config.max_num_seqs, config.max_model_len
        self.max_prefill_len, self.block_size = config.prompt_limit, config.block_size
        self.stats = EngineStats()
        pages = config.pool_pages
        if config.num_blocks is None and config.memory_fraction is not None:
            # the pool is sized from the memory that is free now (the weights are loaded already)
            probe = CacheManager(model.cache_needs(), config.block_size, 1, 1, False)
            itemsize = 4 if config.dtype == torch.float32 else 2
            free_bytes = torch.cuda.mem_get_info(torch.device(config.device))[0]
            pages = config.pages_for_memory(probe.bytes_per_page(itemsize), free_bytes)
        self.num_blocks = pages
        self.cache = CacheManager(model.cache_needs(), config.block_size, pages, config.max_num_seqs,
                                  config.prefix_cache)
        self.runner = runner if runner is not None else Runner(
            model, self.cache, config.device, config.dtype, max_model_len=config.max_model_len,
            cuda_graphs=config.cuda_graphs)
        self.scheduler = Scheduler(self.cache, config.max_tokens_per_step, config.max_model_len, config.prompt_limit,
                                   self.stats)
        self.sampler = sampler if sampler is not None else Sampler(config.device)
        self.requests: dict[int, Request] = {}
        self.id_lock = threading.Lock()
        self.step_lock = threading.Lock()          # the scheduler and the cache are touched under it only
        self.next_id = 0
        # The router reaches the driver through a weak reference: a strong one would close a cycle, and a driver that
        # only the cycle collector frees may be freed at any moment, in the middle of another driver's graph capture
        # (where destroying this driver's captured graphs is an error).  A driver that is dropped stops its thread.
        me = weakref.ref(self)
        self.router = EventRouter(lambda: step(me()) if me() is not None else [],
                                  lambda: me() is not None and has_work(me()))
        weakref.finalize(self, self.router.stop, False)
        self.ahead = None                  # the next step's plan, made while the device ran the last one
        self.host_tokens = None            # pinned memory that the sampled tokens come back to


def make_driver(model, max_num_seqs: int = 4, max_model_len: int = 2048, max_prefill_len: Optional[int] = None,
                block_size: int = 16, num_blocks: Optional[int] = None, dtype=None, runner=None, sampler=None,
                **more) -> Driver:
    """A driver for a loaded model.  `dtype` defaults to the model's compute dtype and must
    equal it.  `more`: max_tokens_per_step, prefix_cache, decode_split_size, cuda_graphs, memory_fraction (with
    num_blocks None the pool takes that share of the free device memory instead of the worst case)."""
    model_dtype = model.ctx.dtype
    dtype = parse_dtype(dtype) if dtype is not None else model_dtype
    if dtype != model_dtype:
        raise ValueError(f"the model was loaded as {model_dtype}, the driver was asked for {dtype}")
    more.setdefault("decode_split_size", model.ctx.decode_split_size)
    if more["decode_split_size"] != model.ctx.decode_split_size:
        raise ValueError("decode_split_size is fixed when the model is loaded")
    cfg = EngineConfig(dtype=dtype, max_num_seqs=max_num_seqs, max_model_len=max_model_len,
                       max_prefill_len=max_prefill_len, block_size=block_size, num_blocks=num_blocks,
                       device=str(model.ctx.device), **more)
    return Driver(model, cfg, runner=runner, sampler=sampler)


def _checked_prompt(driver: Driver, prompt_ids) -> list:
    prompt = [int(t) for t in prompt_ids]
    vocab = driver.model.spec.vocab_size
    if any(t < 0 or t >= vocab for t in prompt):
        raise ValueError(f"prompt holds token ids outside [0, {vocab})")
    return prompt


def _check_sampling(driver: Driver, prompt: list, sampling: SamplingParams) -> None:
    driver.scheduler.validate(prompt, sampling)
    vocab = driver.model.spec.vocab_size
    if vocab > MOST_VOCAB and (sampling.filtered or sampling.logprobs is not None):
        raise ValueError(f"filters and log-probabilities are for at most {MOST_VOCAB} tokens, the vocabulary has {vocab}")


def _new_request(driver: Driver, prompt: list, sampling: SamplingParams, arrival: Optional[float] = None) -> Request:
    with driver.id_lock:
        rid = driver.next_id
        driver.next_id += 1
    driver.router.open(rid)
    return Request(request_id=rid, prompt_ids=prompt, sampling=sampling, arrival=time.perf_counter() if arrival is None else arrival)


def _add(driver: Driver, prompt: list, sampling: list) -> list:
    """Registers requests that continue one prompt, the first of them with the scheduler; returns their ids."""
    arrival = time.perf_counter()
    for sp in sampling:
        _check_sampling(driver, prompt, sp)      # what is refused anyway need not wait for a step
    with driver.step_lock:
        # the pool may have changed its size meanwhile: all are checked before anything of them is registered
        for sp in sampling:
            _check_sampling(driver, prompt, sp)
        reqs = [_new_request(driver, prompt, sp, arrival) for sp in sampling]
        reqs[0].followers = reqs[1:]
        for req in reqs:
            driver.requests[req.request_id] = req
        driver.scheduler.add(reqs[0])
    driver.router.wake()
    return [req.request_id for req in reqs]


def add_request(driver: Driver, prompt_ids, sampling: Optional[SamplingParams] = None) -> int:
    driver.router.raise_if_failed()
    sp = sampling or SamplingParams()
    return _add(driver, _checked_prompt(driver, prompt_ids), [sp])[0]


def add_continuations(driver: Driver, prompt_ids, n: int, sampling=None) -> list:
    """Adds `n` requests that continue the same prompt; returns their ids.  The prompt is computed once: when its last
    token is done, every continuation draws its first token from the same logits, and all but the first take over the
    prompt's pages (full ones shared, the last copied) and states.  One that finds no state slot then waits and is computed
    by itself.  `sampling`: parameters for all (a seed s becomes s, s + 1, ...; without one each has its own) or one per
    continuation."""
    driver.router.raise_if_failed()
    if n < 1:
        raise ValueError("at least one continuation")
    if sampling is None or isinstance(sampling, SamplingParams):
        one = sampling or SamplingParams()
        sampling = [replace(one, seed=None if one.seed is None else one.seed + i) for i in range(n)]
    if len(sampling) != n:
        raise ValueError("one set of sampling parameters for all continuations, or one for each")
    return _add(driver, _checked_prompt(driver, prompt_ids), sampling)


def _on_device(driver: Driver):
    """The driver's device as the current one: launches, events and copies go to the current device's stream."""
    device = torch.device(driver.config.device)
    return torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext()


def _order(driver: Driver) -> tuple:
    """(leave, follow) of the runner: a step that samples ends with the host waiting for its tokens, but what does not (a step
    without logits, copies for forks) may still run when the next one is issued, by another thread or on another stream."""
    nothing = lambda: None  # noqa: E731
    return getattr(driver.runner, "leave", nothing), getattr(driver.runner, "follow", nothing)


@contextlib.contextmanager
def _device_idle(driver: Driver):
    """What is done to the cache between two steps, on whatever stream the caller has, begins after the steps issued so far
    and is done before the next one."""
    device = torch.device(driver.config.device)
    if device.type != "cuda":
        yield
        return
    torch.cuda.synchronize(device)
    yield
    torch.cuda.synchronize(device)


def fork_request(driver: Driver, request_id: int, sampling: Optional[SamplingParams] = None) -> int:
    """Adds a request that goes on from where an unfinished one stands; returns its id.  It shares the full pages that the
    other holds and takes a copy of the last page and of the states; without a free slot or page it waits and is computed
    again.  Its tokens so far are the other's, its events those that it produces itself; `max_new_tokens` counts both.
    `sampling` defaults to the other's parameters, without a seed."""
    driver.router.raise_if_failed()
    with driver.step_lock, _on_device(driver):
        parent = driver.requests.get(request_id)
        if parent is None or parent.finished:
            raise KeyError(f"request {request_id} is not running")
        if any(parent is f for r in list(driver.requests.values()) for f in r.followers):
            raise ValueError(f"request {request_id} waits for the prompt that it continues")
        sp = sampling if sampling is not None else replace(parent.sampling, seed=None)
        if len(parent.output_ids) >= sp.max_new_tokens:
            raise ValueError(f"the request has {len(parent.output_ids)} tokens already, max_new_tokens is {sp.max_new_tokens}")
        _check_sampling(driver, parent.prompt_ids, sp)
        child = _new_request(driver, parent.prompt_ids, sp)
        child.output_ids = list(parent.output_ids)
        driver.requests[child.request_id] = child
        # the copies follow the last step, and the next step follows them: nothing else on the device is waited for
        leave, follow = _order(driver)
        follow()
        driver.scheduler.fork(parent, [child])
        leave()
    driver.router.wake()
    return child.request_id


def resize_cache(driver: Driver, num_blocks: int) -> None:
    """Gives the cache `num_blocks` pages: fewer to return device memory, more to serve more requests.  Live requests go on;
    their pages, and the ones kept for reuse as far as they fit, move to the new pool.  Refused where a request that is not
    finished could need more pages than there would be.  The captured decode steps are dropped and captured again when
    they are next needed."""
    driver.router.raise_if_failed()
    with driver.step_lock, _on_device(driver):
        cache, sched = driver.cache, driver.scheduler
        if not cache.groups:
            raise ValueError("the model keeps no pages")
        for req in list(sched.running) + list(sched.waiting):
            for r in [req] + req.followers:
                need = -(-(len(r.prompt_ids) + r.sampling.max_new_tokens) // cache.page_size)
                if need > num_blocks:
                    raise ValueError(f"request {r.request_id} may need {need} pages, {num_blocks} were asked for")
        held = max(cache.num_pages - g.pool.num_free for g in cache.groups)
        if num_blocks < max(1, held):
            raise ValueError(f"{held} pages are in use, {num_blocks} were asked for")
        cache.check_room(num_blocks, captured=True)      # what is refused costs no captured step
        driver.ahead = None
        if hasattr(driver.runner, "forget_graphs"):
            driver.runner.forget_graphs()
        with _device_idle(driver):
            cache.resize(num_blocks)
        if torch.device(driver.config.device).type == "cuda":
            torch.cuda.empty_cache()             # what the old stores held goes back to the device
        sched.version += 1
        driver.num_blocks = num_blocks
        driver.stats.pages_total = num_blocks


def has_work(driver: Driver) -> bool:
    return driver.scheduler.has_work()


def step(driver: Driver) -> list:
    """One scheduler iteration: at most one batch on the device; returns its StepEvents."""
    driver.router.raise_if_failed()
    with driver.step_lock, _on_device(driver):
        return _step_locked(driver)


def _step_locked(driver: Driver) -> list:
    sched = driver.scheduler
    if driver.cache.broken:
        raise RuntimeError(driver.cache.broken)
    leave, follow = _order(driver)
    follow()
    ahead, driver.ahead = driver.ahead, None
    plan = sched.take_ahead(ahead) or sched.schedule()
    if not plan:
        return []
    entries = [StepEntry(driver.cache.live[s.request.request_id], s.tokens, (len(s.tokens) - 1,) if s.wants_logits else ())
               for s in plan]
    sampled = [s for s in plan if s.wants_logits]
    # one draw for every request whose logits are there, and for every continuation that waits for its prompt
    draws = [(row, req) for row, s in enumerate(sampled) for req in [s.request] + s.request.followers]
    forking = len(draws) > len(sampled)
    params = [req.sampling for _, req in draws]
    temps = [sp.temperature for sp in params]
    seeds = [sp.seed if sp.seed is not None else req.request_id for sp, (_, req) in zip(params, draws)]
    counters = [len(req.output_ids) for _, req in draws]
    filters = [(sp.top_k, sp.top_p, sp.min_p) if sp.filtered else (0, 1.0, 0.0) for sp in params] \
        if any(sp.filtered for sp in params) else None
    top = max([-1] + [sp.logprobs for sp in params if sp.logprobs is not None])      # -1: nobody wants log-probabilities
    # a decode-only step samples inside its replayed graph; any other step hands back logits for the sampler
    fused = getattr(driver.runner, "step_sampled", None)
    more = () if filters is None else (filters,)
    both = fused(entries, temps, seeds, counters, *more) \
        if fused is not None and len(sampled) == len(plan) and not forking and top < 0 else None
    logits = driver.runner.step(entries) if both is None else None
    sched.committed(plan)
    st = driver.stats
    st.steps += 1
    st.last_step_tokens = sum(len(e.tokens) for e in entries)
    st.max_step_tokens = max(st.max_step_tokens, st.last_step_tokens)
    if driver.cache.groups:
        st.pages_total = driver.cache.num_pages
        st.pages_in_use = max(driver.cache.num_pages - g.pool.num_free for g in driver.cache.groups)
        st.max_pages_in_use = max(st.max_pages_in_use, st.pages_in_use)
    events: list = []
    if not sampled:
        leave()
        return events
    if both is None:
        parts = [[], [], [], []]
        # a prompt's continuations need its row once each: of hundreds, no more rows at a time than requests run at a time
        at_once = max(len(sampled), driver.max_num_seqs, 64) if forking else len(draws)
        for i in range(0, len(draws), at_once):
            part = slice(i, i + at_once)
            block = logits
            if forking:
                rows = [row for row, _ in draws[part]]
                block = driver.sampler.repeat_rows(logits, rows) if logits.is_cuda else logits[rows]
            if filters is None:
                tokens = driver.sampler.sample(block, temps[part], seeds[part], counters[part])
            else:
                tokens = driver.sampler.sample_filtered(block, temps[part], seeds[part], counters[part], filters[part])
            parts[0].append(tokens)
            if top >= 0:
                chosen, top_tokens, top_values = driver.sampler.logprobs(block, tokens, top)
                parts[1].append(chosen.view(torch.int32))
                parts[2].append(top_tokens.reshape(-1))
                parts[3].append(top_values.view(torch.int32).reshape(-1))
        if top >= 0:
            top = top_tokens.shape[1]
        both = torch.cat([*parts[0], driver.runner.status_word(), *parts[1], *parts[2], *parts[3]])      # one copy back
    arrived = None
    if both.is_cuda:
        # the copy is on its way while the host plans the next step; waiting for it also synchronises
        if driver.host_tokens is None or driver.host_tokens.numel() < both.numel():
            driver.host_tokens = torch.empty(max(both.numel(), 64), dtype=both.dtype, pin_memory=True)
        back = driver.host_tokens[:both.numel()]
        back.copy_(both, non_blocking=True)
        arrived = torch.cuda.Event()
        arrived.record()
        both = back
    driver.ahead = sched.plan_ahead(plan) if not forking else None
    if driver.ahead is not None and fused is not None and top < 0:
        # its layout goes into the staging buffer now too; only the tokens are missing
        driver.runner.prefill_ahead([StepEntry(driver.cache.live[s.request.request_id], [0], (0,)) for s in driver.ahead[1]],
                                    temps, seeds, [c + 1 for c in counters], *more)
    if arrived is not None:
        arrived.synchronize()
    n = len(draws)
    scores = likely = likely_scores = None
    if top >= 0:
        floats = both.view(torch.float32)
        scores = floats[n + 1:2 * n + 1].tolist()
        likely = both[2 * n + 1:2 * n + 1 + n * top].tolist()
        likely_scores = floats[2 * n + 1 + n * top:].tolist()
    both = both[:n + 1].tolist()
    toks, status = both[:-1], both[-1]
    if status:
        driver.runner.clear_status()
        from ..ops import raise_on_status
        raise_on_status(status)
    now = time.perf_counter()
    by_row = [[] for _ in sampled]
    for k, ((row, req), tok) in enumerate(zip(draws, toks)):
        event = StepEvent(req.request_id, int(tok), False)
        if req.sampling.logprobs is not None:
            m = min(req.sampling.logprobs, top)
            event.logprob = scores[k]
            event.top_logprobs = list(zip(likely[k * top:k * top + m], likely_scores[k * top:k * top + m]))
            req.logprobs.append(event.logprob)
            req.top_logprobs.append(event.top_logprobs)
        req.output_ids.append(event.token)
        if req.first_token_time is None:
            req.first_token_time = now
        driver.stats.emitted_tokens += 1
        event.finished = len(req.output_ids) >= req.sampling.max_new_tokens or req.sampling.stops_at(event.token)
        by_row[row].append((req, event))
        events.append(event)
    for s, made in zip(sampled, by_row):
        # continuations go on from what the first of them holds, before it may be given back
        go_on = [req for req, event in made[1:] if not event.finished]
        for req, event in made[1:]:
            if event.finished:
                sched.finish_unstarted(req)
        s.request.followers = []
        if go_on:
            sched.fork(s.request, go_on)
        if made[0][1].finished:
            sched.finish(s.request)
    if forking:
        leave()
    return events


def _run_to_end(driver: Driver, ids: list) -> list:
    reqs = [driver.requests[i] for i in ids]
    while any(not r.finished for r in reqs):
        if not step(driver) and not has_work(driver):
            break
    for i in ids:
        driver.router.close(i)
        driver.requests.pop(i, None)
    return reqs


def continuations(driver: Driver, prompt_ids, n: int, sampling=None) -> list:
    """Runs `n` continuations of a prompt to completion (see `add_continuations`); returns their Request records, with
    `output_ids` and, where they were asked for, `logprobs`: the likeliest one is max(..., key=lambda r: sum(r.logprobs))."""
    return _run_to_end(driver, add_continuations(driver, prompt_ids, n, sampling))


def generate(driver: Driver, prompts, sampling=None) -> list:
    """Runs the prompts (lists of token ids) to completion; returns the generated token ids of
    each, in order.  `sampling`: one SamplingParams for all, or one per prompt."""
    if sampling is None or isinstance(sampling, SamplingParams):
        sampling = [sampling] * len(prompts)
    ids = [add_request(driver, p, sp) for p, sp in zip(prompts, sampling)]
    return [list(r.output_ids) for r in _run_to_end(driver, ids)]


# --------------------------------------------------------------- streams and thread
def stream(driver: Driver, request_id: int) -> Iterator[StepEvent]:
    """The events of one request, until the one that finishes it.  With the background thread running they come
    from the thread; without one, the reader steps the engine itself (see engine/background.py)."""
    driver.router.raise_if_failed()
    for ev in driver.router.events(request_id):
        yield ev
    driver.requests.pop(request_id, None)


def start(driver: Driver) -> None:
    """Starts the background thread that steps the engine whenever there is work."""
    driver.router.start()


def stop(driver: Driver, join: bool = True) -> None:
    driver.router.stop(join)


def prewarm(driver: Driver) -> float:
    """Compiles what the model needs, runs one tiny batch and captures the decode graphs of every batch size up
    to `max_num_seqs`, without filters and with them, so that no request pays for it (the reference compiles its
    shape buckets here, jllm/engine/engine.py:112-150); steps that give log-probabilities are captured when they
    are first needed.  Returns the seconds it took."""
    t0 = time.perf_counter()
    with driver.step_lock, _on_device(driver):
        driver.ahead = None
        leave, follow = _order(driver)
        follow()
        driver.runner.warm_up(decode_batches=driver.max_num_seqs)
        leave()
    return time.perf_counter() - t0

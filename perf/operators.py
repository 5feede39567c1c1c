"""Operators for several continuations of one prompt, as cases that can be timed and checked: drawing tokens under filters, scoring
them, and copying the pages and state rows of the cache that a request leaves to its forks or takes into a pool of another size.

    kind     sample     one token a row from softmax(logits / temperature) under top-k, top-p and min-p
             logprobs   the log-probability of a given token a row, and the `top` likeliest tokens with theirs
             pages      pages of key and value stores copied, in place (a fork) or into other stores (a pool of another size)
             slots      rows of fixed-size recurrent states copied to other slots of the same tensors (a fork)

With `own` false, `run` computes them in elementary torch operations; with `own` true it calls the engine's operators.

A row's tokens are in order of their logits, the lowest index first among equals, and count p = exp((logit - largest) / temperature).
Kept are the first top_k of them (0: all) that have p >= min_p (0: all), and of these the ones before which less than top_p of their
sum lies (1: all).  The token is the kept one with the largest logit / temperature - log(-log(u)), where u in (0, 1) is a hash of
(seed, counter, token id): a draw from the kept tokens' softmax.  A temperature of 0 takes the largest logit.  Masked tokens have
logits of minus infinity.
"""

from __future__ import annotations

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
MODES = ("top_k", "top_p", "min_p", "all", "mixed")
MOST_LOGITS = 256 * 151936             # of a drawn case of `sample`
MOST_SCORED = 1024 * 151936            # of a drawn case of `logprobs`
MOST_BYTES = 2 << 30                   # what a drawn case of `pages` or `slots` writes


# ------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request, every filter on: a chat, where only latency counts
        {"name": "sample 1 all", "kind": "sample", "rows": 1, "vocab": 151936, "mode": "all", "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "f32"},
        # a small batch of requests that each have filters of their own (greedy and unfiltered ones among them), 16-bit logits, an odd vocabulary
        {"name": "sample 24 mixed bf16", "kind": "sample", "rows": 24, "vocab": 32003, "mode": "mixed", "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "bf16"},
        # nearly even logits, as of a model that is hardly trained: the kept tokens are most of the vocabulary
        {"name": "sample 64 top_p even", "kind": "sample", "rows": 64, "vocab": 151936, "mode": "top_p", "spread": 1.0, "peaks": 0, "masked": 0.0, "dtype": "f32"},
        # a grammar that leaves a third of the vocabulary
        {"name": "sample 96 top_k masked", "kind": "sample", "rows": 96, "vocab": 100003, "mode": "top_k", "spread": 2.2, "peaks": 40, "masked": 0.67, "dtype": "f32"},
        # the largest batch of a captured decode step
        {"name": "sample 256 all", "kind": "sample", "rows": 256, "vocab": 151936, "mode": "all", "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "f32"},
        # a small decode step whose continuations are compared by their scores
        {"name": "logprobs 8", "kind": "logprobs", "rows": 8, "vocab": 151936, "top": 0, "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "f32"},
        # the likeliest alternatives beside every token, 16-bit logits (equal ones among them), an odd vocabulary
        {"name": "logprobs 64 top 20 bf16", "kind": "logprobs", "rows": 64, "vocab": 50021, "top": 20, "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "bf16"},
        # every place of a prompt scored
        {"name": "logprobs 1024", "kind": "logprobs", "rows": 1024, "vocab": 151936, "top": 0, "spread": 2.2, "peaks": 40, "masked": 0.0, "dtype": "f32"},
        # one request forked into four: its last, partly filled page to three others in every layer
        {"name": "pages fork 1 to 3", "kind": "pages", "layers": 36, "pages": 256, "page": 16, "heads": 8, "dim": 128, "stores": 2,
         "sources": 1, "fan": 3, "part": True, "into": False, "dtype": "bf16"},
        # rows of an odd size in 32 bits (one store: the values are part of the keys), pages of five tokens
        {"name": "pages fork 7 to 14 odd", "kind": "pages", "layers": 9, "pages": 300, "page": 5, "heads": 1, "dim": 77, "stores": 1,
         "sources": 7, "fan": 2, "part": True, "into": False, "dtype": "f32"},
        # a pool made smaller: the pages in use, scattered, to the first pages of new stores
        {"name": "pages into 1500", "kind": "pages", "layers": 28, "pages": 2048, "page": 16, "heads": 8, "dim": 128, "stores": 2,
         "sources": 1500, "fan": 1, "part": False, "into": True, "dtype": "bf16"},
        # eight requests of a model with recurrent layers, each forked into four: a matrix per head in every layer
        {"name": "slots fork 8 to 24", "kind": "slots", "layers": 24, "slots": 64, "heads": 32, "dim": 64, "columns": 64,
         "sources": 8, "fan": 3, "dtype": "f32"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(("sample", "sample", "logprobs", "pages", "slots"))
    if kind in ("sample", "logprobs"):
        rows = _spread(rng, 1, 256 if kind == "sample" else 1024)
        most = (MOST_LOGITS if kind == "sample" else MOST_SCORED) // rows
        case = {"kind": kind, "rows": rows, "vocab": _spread(rng, 300, min(262144, most)),
                "spread": round(0.5 + 3.5 * rng.random(), 2), "peaks": rng.choice((0, 3, 40, 200)), "masked": rng.choice((0.0, 0.0, 0.3, 0.9)),
                "dtype": rng.choice(("f32", "f32", "bf16"))}
        return {**case, "mode": rng.choice(MODES)} if kind == "sample" else {**case, "top": rng.choice((0, 0, 1, 5, 20, 64))}
    if kind == "pages":
        case = {"kind": kind, "layers": _spread(rng, 1, 64), "page": rng.choice((1, 5, 8, 16, 32, 64)), "heads": rng.choice((1, 2, 3, 4, 8, 16)),
                "dim": rng.choice((33, 64, 80, 96, 128, 192, 256)), "stores": rng.choice((1, 2)), "dtype": rng.choice(("f32", "bf16")),
                "into": rng.random() < 0.4}
        row = case["heads"] * case["dim"] * case["page"] * case["layers"] * case["stores"] * DTYPES[case["dtype"]].itemsize
        fan = 1 if case["into"] else _spread(rng, 1, 8)
        sources = _spread(rng, 1, max(1, min(1024, MOST_BYTES // (row * fan))))
        return {**case, "fan": fan, "sources": sources, "part": not case["into"] and rng.random() < 0.7,
                "pages": sources * (1 + fan) + rng.randrange(1, 9)}
    case = {"kind": kind, "layers": _spread(rng, 1, 48), "heads": _spread(rng, 1, 64), "dim": rng.choice((1, 16, 64, 96, 128)),
            "columns": rng.choice((1, 3, 64, 128)), "dtype": rng.choice(("f32", "f32", "bf16"))}
    row = case["heads"] * case["dim"] * case["columns"] * case["layers"] * DTYPES[case["dtype"]].itemsize
    fan = _spread(rng, 1, 8)
    sources = _spread(rng, 1, max(1, min(32, MOST_BYTES // (row * fan))))
    return {**case, "fan": fan, "sources": sources, "slots": sources * (1 + fan) + rng.randrange(1, 9)}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _logits(case, gen):
    """A bulk of logits with some tokens that stand out of it, as far as a model is sure of itself; masked ones at minus infinity."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device=DEVICE) * case["spread"]
    peaks = min(case["peaks"], vocab)
    if peaks:
        at = torch.randint(0, vocab, (rows, peaks), generator=gen, device=DEVICE)
        x.scatter_reduce_(1, at, 4 + 10 * torch.rand(rows, peaks, generator=gen, device=DEVICE), "amax")
    if case["masked"]:
        x.masked_fill_(torch.rand(rows, vocab, generator=gen, device=DEVICE) < case["masked"], -float("inf"))
    return x.to(DTYPES[case["dtype"]])


def _filters(mode, rows):
    """(temperature, top_k, top_p, min_p) a row: as chats, programs and stories ask for them."""
    one = {"top_k": (0.8, 50, 1.0, 0.0), "top_p": (1.0, 0, 0.9, 0.0), "min_p": (1.1, 0, 1.0, 0.05), "all": (0.7, 40, 0.95, 0.02),
           "greedy": (0.0, 0, 1.0, 0.0), "none": (1.0, 0, 1.0, 0.0), "many": (0.9, 700, 0.98, 0.0)}
    names = ("greedy", "none", "top_k", "top_p", "min_p", "all", "many") if mode == "mixed" else (mode,)
    return [one[names[r % len(names)]] for r in range(rows)]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 32))
    s = {"case": case}
    if case["kind"] in ("sample", "logprobs"):
        rows = case["rows"]
        s["logits"] = _logits(case, gen)
        if case["kind"] == "sample":
            t, k, p, m = zip(*_filters(case["mode"], rows))
            s.update(temperature=torch.tensor(t, dtype=torch.float32, device=DEVICE), top_k=torch.tensor(k, dtype=torch.int32, device=DEVICE),
                     top_p=torch.tensor(p, dtype=torch.float32, device=DEVICE), min_p=torch.tensor(m, dtype=torch.float32, device=DEVICE),
                     seeds=torch.randint(0, 1 << 62, (rows,), generator=gen, device=DEVICE),
                     counters=torch.randint(0, 4096, (rows,), generator=gen, device=DEVICE))
        else:
            # tokens as they are sampled: mostly likely ones
            any_token = torch.randint(0, case["vocab"], (rows,), generator=gen, device=DEVICE)
            likely = torch.rand(rows, generator=gen, device=DEVICE) < 0.8
            s["tokens"] = torch.where(likely, s["logits"].argmax(1), any_token).to(torch.int32)
        return s
    dtype, fan, n = DTYPES[case["dtype"]], case["fan"], case["sources"]
    where = host.permutation(case["pages" if case["kind"] == "pages" else "slots"])
    s["src"] = [int(x) for x in where[:n] for _ in range(fan)]
    if case["kind"] == "pages":
        shape = (case["layers"], case["pages"], case["page"], case["heads"], case["dim"])
        s["stores"] = [torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype) for _ in range(case["stores"])]
        s["dst"] = list(range(n)) if case["into"] else [int(x) for x in where[n:n + n * fan]]
        s["into"] = [torch.zeros((case["layers"], n, *shape[2:]), dtype=dtype, device=DEVICE) for _ in range(case["stores"])] if case["into"] else None
        s["held"] = [int(x) for x in np.repeat(host.randint(1, case["page"] + 1, n), fan)] if case["part"] else None
    else:
        shape = (case["slots"], case["heads"], case["dim"], case["columns"])
        s["states"] = [torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype) for _ in range(case["layers"])]
        s["dst"] = [int(x) for x in where[n:n + n * fan]]
    return s


# --------------------------------------------------------------------------------------------------------------- plain forms
def _shift(z, by):
    """z >> by of an unsigned 64-bit number that is held in a signed one."""
    return (z >> by) & ((1 << (64 - by)) - 1)


def _signed(z):
    return z - (1 << 64) if z >= 1 << 63 else z


def _mix(z):
    z = (z ^ _shift(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shift(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ _shift(z, 31)


def _uniform(seeds, counters, ids):
    """In (0, 1), 24 random bits, for every row's seed and counter and every token id."""
    h = _mix(seeds + (counters + 1) * _signed(0x9E3779B97F4A7C15))
    h = _mix(h[:, None] ^ (ids * _signed(0xD1342543DE82EF95) + 0x2545F4914F6CDD1D)[None])
    return (_shift(h, 40).float() + 0.5) * (1.0 / 16777216.0)


def _plain_sample(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    temperature = s["temperature"][:, None]
    hot = temperature > 0
    t = torch.where(hot, temperature, torch.ones_like(temperature))
    ids = torch.arange(vocab, device=x.device)
    score = torch.where(hot, x / t - torch.log(-torch.log(_uniform(s["seeds"], s["counters"], ids))), x)
    best, order = torch.sort(x, dim=1, descending=True, stable=True)       # equals stay in the order of their indices
    mass = torch.exp(torch.where(best == best[:, :1], 0.0, (best.double() - best[:, :1].double()) / t.double()))
    k = s["top_k"][:, None]
    kept = (k <= 0) | (ids[None] < k)
    kept &= (s["min_p"][:, None] <= 0) | (mass >= s["min_p"][:, None].double())
    mass = torch.where(kept, mass, 0.0)
    before = mass.cumsum(1) - mass
    p = s["top_p"][:, None].double()
    kept &= (p >= 1) | (before < p * mass.sum(1, keepdim=True))
    kept |= ids[None] == 0                                                 # the first is always kept
    score = torch.where(kept | ~hot, score.gather(1, order), -float("inf"))
    winners = torch.where(score == score.amax(1, keepdim=True), order, vocab)
    return winners.amin(1).to(torch.int32)


def _plain_logprobs(s):
    x = s["logits"].float()
    top = s["case"]["top"]
    largest = x.amax(1, keepdim=True)
    norm = largest + torch.log(torch.exp(x - largest).sum(1, keepdim=True))
    chosen = (x.gather(1, s["tokens"].long()[:, None]) - norm)[:, 0]
    best, order = torch.sort(x, dim=1, descending=True, stable=True) if top else (x, torch.zeros_like(x[:, :0]))
    return chosen, order[:, :top].to(torch.int32), best[:, :top] - norm


def _plain_pages(s):
    src, dst = torch.tensor(s["src"], device=DEVICE), torch.tensor(s["dst"], device=DEVICE)
    into = s["into"] or s["stores"]
    for store, to in zip(s["stores"], into):
        new = store[:, src]
        if s["held"] is not None:
            first = torch.arange(store.shape[2], device=DEVICE)[None] < torch.tensor(s["held"], device=DEVICE)[:, None]
            new = torch.where(first[None, :, :, None, None], new, to[:, dst])
        to[:, dst] = new
    return into


def _plain_slots(s):
    src, dst = torch.tensor(s["src"], device=DEVICE), torch.tensor(s["dst"], device=DEVICE)
    for state in s["states"]:
        state[dst] = state[src]
    return s["states"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        from jax_vllm_b200 import ops
        if kind == "sample":
            return ops.sample_filtered(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["seeds"],
                                       state["counters"])
        if kind == "logprobs":
            return ops.token_logprobs(state["logits"], state["tokens"], state["case"]["top"])
        if kind == "pages":
            ops.copy_pages(state["stores"], state["src"], state["dst"], tokens=state["held"], into=state["into"])
            return state["into"] or state["stores"]
        ops.copy_slots(state["states"], state["src"], state["dst"])
        return state["states"]
    return {"sample": _plain_sample, "logprobs": _plain_logprobs, "pages": _plain_pages, "slots": _plain_slots}[kind](state)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] in ("sample", "logprobs"):
        n = case["rows"] * case["vocab"]
        back = 4 * case["rows"] * (1 if case["kind"] == "sample" else 2 + 2 * case["top"])
        # a difference, a product, an exponential and a sum for every logit
        return {"bytes": n * size + back + (32 * case["rows"] if case["kind"] == "sample" else 0), "flops": 4 * n}
    if case["kind"] == "pages":
        row = case["layers"] * case["page"] * case["heads"] * case["dim"] * case["stores"] * size
        if case["part"]:
            row = row * (case["page"] + 1) / (2 * case["page"])            # any number of a page's tokens, as often as any other
    else:
        row = case["layers"] * case["heads"] * case["dim"] * case["columns"] * size
    return {"bytes": row * case["sources"] * (1 + case["fan"]), "flops": 0}


# ----------------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_uniform(seed, counter, ids):
    mask = (1 << 64) - 1

    def mix(z):
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9 & mask
        z = (z ^ (z >> 27)) * 0x94D049BB133111EB & mask
        return z ^ (z >> 31)

    h = np.uint64(mix((seed + 0x9E3779B97F4A7C15 * (counter + 1)) & mask))
    with np.errstate(over="ignore"):
        z = h ^ (ids.astype(np.uint64) * np.uint64(0xD1342543DE82EF95) + np.uint64(0x2545F4914F6CDD1D))
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    return ((z >> np.uint64(40)).astype(np.float64) + 0.5) / 16777216.0


def _exact_token(x, t, k, p, m, seed, counter):
    """The token of one row, from its logits in 64 bits."""
    if not t > 0:
        return int(np.argmax(x))
    ids = np.argsort(-x, kind="stable")
    if k > 0:
        ids = ids[:k]
    mass = np.exp(np.where(x[ids] == x[ids[0]], 0.0, x[ids] - x[ids[0]]) / t)
    if m > 0:
        ids, mass = ids[mass >= m], mass[mass >= m]
    if p < 1:
        before = np.concatenate(([0.0], np.cumsum(mass)[:-1]))
        ids = ids[(before < p * mass.sum()) | (np.arange(ids.size) == 0)]
    ids = np.sort(ids)
    return int(ids[np.argmax(x[ids] / t - np.log(-np.log(_exact_uniform(seed, counter, ids))))])


def exact(case, seed):
    if case["kind"] in ("pages", "slots"):
        return None                                                        # copies: no value is computed
    s = prepare(case, seed)
    rows = range(case["rows"])
    if case["kind"] == "sample":
        t, k, p, m, seeds, counters = (s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "seeds", "counters"))
        host = s["logits"].cpu()
        tokens = [_exact_token(host[r].double().numpy(), t[r], k[r], p[r], m[r], seeds[r], counters[r]) for r in rows]
        return torch.tensor(tokens, dtype=torch.int32)
    top, chosen, ids, best = case["top"], [], [], []
    tokens = s["tokens"].tolist()
    host = s["logits"].cpu()
    for r in rows:
        x = host[r].double().numpy()
        norm = x.max() + np.log(np.exp(x - x.max()).sum())
        first = np.argsort(-x, kind="stable")[:top] if top else np.zeros(0, dtype=np.int64)
        chosen.append(x[tokens[r]] - norm)
        ids.append(first.astype(np.int32))
        best.append(x[first] - norm)
    return np.array(chosen), np.stack(ids), np.stack(best)

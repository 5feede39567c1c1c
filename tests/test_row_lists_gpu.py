"""The lists of a row's first tokens where they are hard to get: many equal logits, masks of a low finite value, rows in ascending
order, long rows that one block reads by itself.  Against the same 64-bit implementations as the operators' other tests."""

import pytest
import torch

from jax_vllm_b200 import ops
from tests.test_continuations_ops_gpu import DTYPES, check_sample, graph_of, names, near, plain_logprobs, rows_of

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

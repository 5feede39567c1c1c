"""Stores to copy into that share memory are refused, before anything reaches a device."""

import itertools

import pytest
import torch

from jax_vllm_b200 import ops


def refused(stores, into):
    with pytest.raises(ops.KernelError) as e:
        ops.copy_pages(stores, [0, 1], [1, 0], into=into)
    return "apart" in str(e.value)


def test_two_stores_into_one():
    a, b = torch.zeros(2, 4, 2, 3), torch.zeros(2, 4, 2, 3)
    into = torch.zeros(2, 9, 2, 3)
    assert refused([a, b], [into, into])
    assert refused([a, b], [into[:, :5], into[:, 4:]])
    assert refused([a, b], [into[:, :5], into[:, 3:8]])
    assert not refused([a, b], [into[:, :4], into[:, 4:8]])          # (no CUDA tensors: that is what these are refused for)
    assert refused([a, b], [a, torch.zeros(2, 4, 2, 3)])
    assert refused([a, b], [torch.zeros(2, 4, 2, 3), a])


def test_parts_of_one_tensor():
    """Keys beside values by layers, by pages and by tokens' rows, and one page of them shared: against the bytes themselves."""
    whole = torch.arange(4 * 6 * 5 * 3).view(4, 6, 5, 3)
    views = [whole[a:b, c:d] for a, b, c, d in itertools.product((0, 1), (2, 4), (0, 2, 3), (4, 6))]
    turned = torch.arange(6 * 4 * 5 * 3).view(6, 4, 5, 3).transpose(0, 1)
    views += [turned[a:b, c:d] for a, b, c, d in itertools.product((0, 1), (2, 4), (0, 2, 3), (4, 6))]
    both = torch.arange(4 * 2 * 6 * 5 * 3).view(4, 2, 6, 5, 3)
    views += [both[:, 0], both[:, 1], both[1:, 0], both[:2, 1, 2:]]
    seen = set()
    for x, y in itertools.product(views, views):
        if x.untyped_storage().data_ptr() != y.untyped_storage().data_ptr():
            continue
        want = bool(set(x.reshape(-1).tolist()) & set(y.reshape(-1).tolist()))
        assert ops._meet(x, y) == want
        seen.add(want)
    assert seen == {True, False}

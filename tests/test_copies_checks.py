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


def test_parts_of_one_tensor_with_rows_of_several_lengths_and_types():
    """Keys longer than values, side by side in one row or shared by a byte: the places that each covers, one by one."""
    whole = torch.zeros(4 * 6 * 20, dtype=torch.int32)
    first = whole.data_ptr()

    def part(dtype, row, at, pages=6, layers=4):
        size = torch.empty((), dtype=dtype).element_size()
        return whole.view(dtype).as_strided((layers, pages, 1, row), (6 * 80 // size, 80 // size, row, 1), at)

    def places(t):
        size = t.element_size()
        return {t.data_ptr() - first + size * (l * t.stride(0) + p * t.stride(1) + i) + k for l in range(t.shape[0]) for p in range(t.shape[1])
                for i in range(t.shape[3]) for k in range(size)}
    parts = [part(torch.int32, 12, 0), part(torch.int32, 8, 12), part(torch.int32, 9, 11), part(torch.int16, 16, 24), part(torch.int16, 17, 23),
             part(torch.int8, 32, 48), part(torch.int8, 33, 47), part(torch.int32, 20, 20, pages=5), part(torch.int32, 5, 60, pages=2, layers=3)]
    seen = set()
    for x, y in itertools.product(parts, parts):
        want = bool(places(x) & places(y))
        assert ops._meet(x, y) == want, (x.shape, y.shape)
        seen.add(want)
    assert seen == {True, False}

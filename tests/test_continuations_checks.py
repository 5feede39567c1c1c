"""What the operators for several continuations refuse, before anything reaches a device."""

import numpy as np
import pytest
import torch

from jax_vllm_b200 import ops


@pytest.mark.parametrize("src,dst,apart,tokens", [
    ([0, 1], [2], False, None), ([0], [10], False, None), ([10], [0], False, None), ([-1], [0], False, None), ([0], [-1], False, None),
    ([0, 1], [5, 5], False, None), ([0, 1], [5, 5], True, None), ([0, 1], [1, 2], False, None), ([3], [3], False, None), ([0.5], [1], False, None),
    (["a"], [1], False, None), ([1 << 40], [1], False, None), ([None], [1], False, None), ([0], [1], False, [17]), ([0], [1], False, [-1]), ([0], [1], False, [1, 2]), (torch.tensor([0.0]), [1], False, None),
    (torch.tensor([[0]]), [1], False, None)])
def test_copies_that_are_refused(src, dst, apart, tokens):
    with pytest.raises(ops.KernelError):
        ops.check_copies("copy", src, dst, 10, 10, apart, tokens, 16)


def test_indices_of_any_integer_kind():
    for src in ([1, 1], (1, 1), torch.tensor([1, 1]), torch.tensor([1, 1], dtype=torch.int32), np.array([1, 1]), iter([1, 1])):
        got = ops.check_copies("copy", src, [5, 6], 10, 10, False, [16, 0], 16)
        assert [list(a) for a in got] == [[1, 1], [5, 6], [16, 0]]
    many = list(range(100))
    got = ops.check_copies("copy", many, [i + 100 for i in many], 100, 200, True)
    assert list(got[0]) == many and list(got[1]) == list(range(100, 200)) and got[2] is None
    assert [len(a) for a in ops.check_copies("copy", [], [], 0, 0, False)[:2]] == [0, 0]


@pytest.mark.parametrize("change", [dict(src=100), dict(src=-1), dict(dst=200), dict(dst=-1), dict(dst=150), dict(tokens=17), dict(tokens=-1)])
def test_one_bad_number_among_many_is_refused(change):
    lists = dict(src=list(range(100)), dst=list(range(100, 200)), tokens=[3] * 100)
    for name, value in change.items():
        lists[name][41] = value
    with pytest.raises(ops.KernelError):
        ops.check_copies("copy", lists["src"], lists["dst"], 100, 200, True, lists["tokens"], 16)


def test_tensors_on_the_host_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_pages([torch.zeros(1, 4, 2, 3)], [0], [1])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_slots([torch.zeros(4, 3)], [0], [1])
    one = torch.zeros(1)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.sample_filtered(torch.zeros(1, 5), one, one.int(), one, one, one.long(), one.long())
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.token_logprobs(torch.zeros(1, 5), one.int())


@pytest.mark.parametrize("stores,into", [
    ([], None), ([torch.zeros(2, 4)], None), ([torch.zeros(1, 4, 2, 3), torch.zeros(1, 5, 2, 3)], None), ([torch.zeros(1, 4, 2, 3)], []),
    ([torch.zeros(1, 4, 2, 3)], [torch.zeros(1, 4, 2, 4)]), ([torch.zeros(1, 4, 2, 3)], [torch.zeros(1, 4, 2, 3).bfloat16()]), ([3], None)])
def test_stores_that_are_refused(stores, into):
    with pytest.raises(ops.KernelError):
        ops.copy_pages(stores, [0], [1], into=into)


@pytest.mark.parametrize("states", [[], [torch.zeros(())], [torch.zeros(4, 2), torch.zeros(5, 2)], [1]])
def test_states_that_are_refused(states):
    with pytest.raises(ops.KernelError):
        ops.copy_slots(states, [0], [1])


@pytest.mark.parametrize("change", ["1d", "half", "turned", "expanded", "short", "type", "scalar", "none"])
def test_logits_that_are_refused(change):
    x, per_row = torch.zeros(4, 6), torch.zeros(4)
    k = per_row.int()
    if change == "1d": x = x[0]
    if change == "half": x = x.half()
    if change == "turned": x = torch.zeros(6, 4).t()
    if change == "expanded": x = torch.zeros(1, 6).expand(4, 6)
    if change == "short": per_row = torch.zeros(3)
    if change == "type": k = per_row
    if change == "scalar": k = torch.tensor(3, dtype=torch.int32)
    if change == "none": x = torch.zeros(4, 0)
    with pytest.raises(ops.KernelError) as e:
        ops.sample_filtered(x, per_row, k, per_row, per_row, per_row.long(), per_row.long())
    assert "CUDA" not in str(e.value)


def test_numbers_of_likely_tokens_that_are_refused():
    # the check of the device comes first on the host; what it would refuse there is refused in test_continuations_ops_gpu.py's place too
    for top in (-1, 7, 129):
        with pytest.raises(ops.KernelError):
            ops.token_logprobs(torch.zeros(1, 6), torch.zeros(1, dtype=torch.int32), top)

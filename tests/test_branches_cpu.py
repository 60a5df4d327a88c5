"""Host side of branches of sequences of a paged cache."""

import gc

import pytest
import torch

from scaling_amd import ops
from scaling_amd.nn import BranchStep, PagedBranches
from tests.test_paged_modules_cpu import _attention, _cache


def _ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _tensors(branches, tokens):
    long = lambda n: torch.zeros(n, dtype=torch.int64)
    return ops.StepTensors(_ints([0] * (branches.total + 1)), long(tokens), long(tokens), long(tokens), long(branches.total))


def _plan(branches, tokens):
    """A step, without a GPU to plan it on."""
    return BranchStep(branches, _tensors(branches, tokens), tokens, 1)


def test_closed_branches_take_no_steps():
    """Their pages are others' then, and nothing that was captured before finds any: no free ones, no keys, no page in the table."""
    cache = _cache(num_pages=20)
    cache.step([20, 5, 1])
    free = sorted(cache._free)
    branches = PagedBranches(cache, [0, 1], 2, 30)
    branches.ctx_len.fill_(3)
    plan = _plan(branches, 4)
    branches.close()
    branches.close()
    assert sorted(cache._free) == free
    assert branches.state.tolist() == [0, 0] and branches.ctx_len.tolist() == [0] * 4 and bool((branches.page_table == -1).all())
    with pytest.raises(RuntimeError, match="closed"):
        branches.step(_ints([1] * 4), 4, 1)
    with pytest.raises(RuntimeError, match="closed"):
        _attention().paged_forward(torch.zeros(1, 4, 256, dtype=torch.bfloat16), cache, 0, plan)


@pytest.mark.parametrize("inference", [False, True])
def test_close_of_branches_made_in_inference_mode(inference):
    cache = _cache()
    cache.step([3, 1])
    with torch.inference_mode(inference):
        branches = PagedBranches(cache, [0], 1, 16)
    branches.close()
    assert cache.free_pages == 3 and branches.state.tolist() == [0, 0]


def test_a_prefix_stays_while_branches_read_it():
    """A sequence is not released under branches that are open, of which there may be several; branches that nobody has any more hold nothing."""
    cache = _cache(num_pages=20)
    cache.step([20, 5, 1])
    first, second = PagedBranches(cache, [0, 1], 2, 30), PagedBranches(cache, [1], 1, 30)
    for sequence in (0, 1):
        with pytest.raises(RuntimeError, match=f"sequence {sequence}.*branches"):
            cache.release(sequence)
    assert cache.lengths == [20, 5, 1] and len(cache._pages[0]) == 2
    cache.release(2)
    cache.step([1, 0, 0])                                        # (more keys of a sequence are behind the prefix)
    first.close()
    cache.release(0)
    with pytest.raises(RuntimeError, match="sequence 1"):
        cache.release(1)
    del second
    cache.release(1)
    assert cache.lengths == [0, 0, 0]


def test_scratch_of_steps_of_many_sizes(monkeypatch):
    """Drafts bring another number of tokens in every step: they share one scratch, not one for every number, but for those that captured steps have, which stay."""
    cache = _cache(num_pages=20)
    cache.step([20, 5, 1])
    branches, capturing = PagedBranches(cache, [0, 1], 4, 30), False
    monkeypatch.setattr(PagedBranches, "_capturing", lambda self: capturing, raising=False)
    need = lambda tokens: ops.paged_prefix_workspace(8, 2, tokens, 4, 2, 64, "cpu").numel()
    held = lambda: {x.data_ptr(): x.numel() for x in gc.get_objects() if type(x) is torch.Tensor and x.dtype == torch.float32 and x.numel() >= need(1)}
    most = 0
    for tokens in (8, 9, 5, 17, 40, 11, 39, 41, 8, 100, 64, 240, 101, 33):
        assert branches.workspace(tokens).numel() >= need(tokens)
        most = max(most, tokens)
        assert len(held()) == 1 and sum(held().values()) <= need(2 * most)
    capturing = True
    graphs = branches.workspace(100).data_ptr()                  # the one that there is
    assert graphs in held() and branches.workspace(3).data_ptr() == graphs
    own = branches.workspace(1000)                               # made in the capture: the graph's alone
    assert own.numel() >= need(1000) and set(held()) == {graphs, own.data_ptr()}
    del own
    capturing = False
    assert branches.workspace(64).data_ptr() == graphs and set(held()) == {graphs}
    eager = branches.workspace(5000).data_ptr()
    assert set(held()) == {graphs, eager}
    branches.close()
    assert set(held()) == {graphs}
    del branches
    assert not held()


def test_a_step_is_for_the_layers_in_front_of_the_next_one(monkeypatch):
    """Lengths and pages lie on the device and are the last planned step's: an earlier one is refused from then on."""
    cache = _cache(num_pages=20)
    cache.step([20, 5, 1])
    branches = PagedBranches(cache, [0], 2, 10)
    monkeypatch.setattr(ops, "paged_step", lambda *a, **kw: _tensors(branches, 2))
    attention, x = _attention(), torch.zeros(1, 2, 256, dtype=torch.bfloat16)
    first = branches.step(_ints([1, 1]), 2, 1)
    monkeypatch.setattr(ops, "paged_append", lambda k, *a, q=None, **kw: q)
    monkeypatch.setattr(ops, "paged_prefix_attention", lambda q, *a, **kw: q)
    assert attention.paged_forward(x, cache, 0, first).shape == x.shape
    second = branches.step(_ints([1, 1]), 2, 1)
    with pytest.raises(RuntimeError, match="later step"):
        attention.paged_forward(x, cache, 0, first)
    assert attention.paged_forward(x, cache, 1, second).shape == x.shape

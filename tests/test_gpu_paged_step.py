"""Steps of a paged cache planned on the GPU, against the definition."""

import random

import pytest
import torch

from scaling_amd import ops
from tests import paged_step_oracle as oracle
from tests.kernels import launched

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class _Cache:
    """Lists and their copies on the GPU."""

    def __init__(self, batch, width, n_pages, page, seed):
        rng = random.Random(seed)
        self.page, self.lengths, self.table = page, [0] * batch, [[rng.randrange(-9, 9) for _ in range(width)] for _ in range(batch)]
        self.free, self.count, self.status = rng.sample(range(n_pages), n_pages), n_pages, 0
        self.on_gpu = [_ints(self.lengths), _ints(self.table), _ints(self.free), _ints([n_pages, 0])]

    def step(self, new, tokens, max_ctx=None, offset=None, in_place=True):
        lengths, table, free, state = self.on_gpu
        ctx_len, state_out = (lengths, state) if in_place else (torch.empty_like(lengths), torch.empty_like(state))
        got = ops.paged_step(_ints(new), lengths, table, free, state, self.page, tokens, max_ctx, None if offset is None else _ints(offset),
                             **({} if in_place else dict(ctx_len=ctx_len, state_out=state_out)))
        want = oracle.step(new, self.lengths, self.table, self.free, self.count, self.status, self.page, tokens, max_ctx, offset)
        if not in_place:                                   # left alone; then counted
            assert lengths.tolist() == self.lengths and state.tolist() == [self.count, self.status]
            lengths.copy_(ctx_len)
            state.copy_(state_out)
        self.lengths, self.table, self.free, self.count, self.status, cu, positions, slots, sequences, last = want
        assert got.cu_seqlens.tolist() == cu and got.last.tolist() == last
        assert lengths.tolist() == self.lengths and state.tolist() == [self.count, self.status]
        assert table.tolist() == self.table and free.tolist() == self.free
        assert got.position_ids.tolist() == positions and got.slots.tolist() == slots and got.sequences.tolist() == sequences
        assert got.cu_seqlens.dtype == torch.int32 and all(t.dtype == torch.int64 and t.is_contiguous() for t in got[1:])
        return got


@pytest.mark.parametrize("batch,page,most", [(1, 16, 40), (7, 16, 30), (33, 48, 100), (64, 64, 200), (65, 16, 3), (1000, 16, 5), (1024, 32, 2), (1025, 16, 4), (2500, 16, 6)])
def test_steps(batch, page, most):
    """Sequences that grow, wait, end and start again."""
    rng = random.Random(batch)
    cache = _Cache(batch, 9, 4 * batch + 3, page, seed=batch)
    refused = 0
    for i in range(14):
        new = [rng.choice((0, 1, 1, rng.randint(1, most), -1 if i > 2 else 1)) for _ in range(batch)]
        tokens = max(1, sum(max(n, 0) for n in new) + rng.choice((0, 0, 5)) - (7 if i == 9 else 0))
        print(f"step {i}: {tokens} tokens of {batch} sequences", flush=True)
        cache.step(new, tokens, None if i % 3 else 8 * page + 3, [rng.randrange(1000) for _ in range(batch)] if i % 2 else None, in_place=i % 4 != 3)
        refused += cache.status != 0
        cache.status = 0
        cache.on_gpu[3][1] = 0
    assert refused > 0 or batch == 1


@pytest.mark.parametrize("batch,page,rows", [(1, 16, 0), (2, 16, 1), (63, 32, 0), (65, 16, 9), (130, 48, 0), (1000, 16, 30), (1024, 16, 0), (1024, 16, 4000), (1025, 16, 0)])
def test_single_tokens(batch, page, rows):
    """Steps of a token or none of each sequence, of which some end: pages of those go to others in the same step."""
    rng = random.Random(batch + rows)
    cache = _Cache(batch, 3, 2 * batch, page, seed=batch + 1)
    refused = taken = 0
    for i in range(3 * page + 20):
        ends = 0.3 if i % 7 == 6 else 0.02
        new = [-1 if rng.random() < ends else int(rng.random() < 0.95) for _ in range(batch)]
        tokens = max(1, new.count(1) + rows - (1 if i % 11 == 10 else 0))
        if i % 16 == 0:
            print(f"step {i}: {tokens} tokens of {batch} sequences", flush=True)
        before = cache.count
        cache.step(new, tokens, None if i % 3 else 2 * page + 3, [rng.randrange(1000) for _ in range(batch)] if i % 2 else None, in_place=i % 4 != 3)
        taken += cache.count < before
        refused += cache.status != 0
        cache.status = 0
        cache.on_gpu[3][1] = 0
    assert taken > 0 and (refused > 0 or batch <= 2)


def test_results_are_tensors_like_any():
    """One allocation holds them; they are written to, kept and used in products as others are, also where no gradients are ever wanted."""
    for mode in (torch.inference_mode, torch.no_grad, torch.enable_grad):
        with mode():
            cache = _Cache(3, 4, 12, 16, seed=9)
            got = cache.step([2, 0, 5], 9)
            kept = [t.clone() for t in got]
            for i, t in enumerate(got):
                t.add_(1 + i)
                assert all(torch.equal(x, k + (1 + j if j <= i else 0)) for j, (x, k) in enumerate(zip(got, kept)))
            assert torch.equal(got.position_ids.view(3, 3).t().contiguous().float().sum(), (kept[1] + 2).float().sum())
            assert not any(t.requires_grad for t in got) and got.last.device == got.cu_seqlens.device and got.slots[2:].storage_offset() == 2 + got.slots.storage_offset()


@pytest.mark.parametrize("new,tokens", [([4000, 96, 1], 4097), ([5000, 0, 3000], 9000), ([1, 1, 1], 6000)])
def test_many_rows(new, tokens):
    cache = _Cache(3, 400, 900, 16, seed=1)
    cache.step([17, 16, 1], 34)
    cache.step(new, tokens)
    cache.step([-1, 2000, 5000], 8192)
    cache.step([2000, -1, 1], 2001)


def test_statuses_add_up_and_stay():
    cache = _Cache(3, 4, 5, 16, seed=2)
    cache.step([16, 17, 1], 40)                            # four pages of five
    cache.step([33, 0, 0], 33)                             # three more
    assert cache.status == 1
    cache.step([0, 50, 0], 50)
    assert cache.status == 3
    cache.step([0, 0, 3], 2)
    assert cache.status == 7
    cache.step([0, -1, 15], 15)                            # goes on meanwhile, and stays
    assert cache.status == 7 and cache.lengths == [16, 0, 16]
    cache.step([49, 0, 60], 3)
    cache.status = 0
    cache.on_gpu[3][1] = 0
    cache.step([48, 64, 0], 2)                             # too many rows, and pages for more than those
    assert cache.status == 5
    cache.step([0, 0, 0], 0)
    cache.step([2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], 10)
    cache.step([-2 ** 31, 1, -5], 10)


def test_lengths_and_counts_from_nowhere():
    """Nothing outside the arrays is read or written whatever they hold."""
    cache = _Cache(4, 3, 10, 16, seed=3)
    cache.lengths, cache.count = [-7, 2 ** 31 - 1, 49, 48], 2 ** 31 - 1
    cache.on_gpu[0], cache.on_gpu[3] = _ints(cache.lengths), _ints([cache.count, 0])
    cache.step([1, -1, 0, -1], 5)                          # ten pages are on the stack already
    cache.lengths = cache.on_gpu[0].tolist()
    cache.count = -5
    cache.on_gpu[3][0] = -5
    cache.step([0, 0, 1, 0], 5)


def test_launches_streams_and_replays():
    cache = _Cache(8, 20, 100, 16, seed=4)
    lengths, table, free, state = cache.on_gpu
    new = _ints([1] * 8)
    assert len(launched(lambda: ops.paged_step(new, lengths, table, free, state, 16, 8, ctx_len=torch.empty_like(lengths), state_out=torch.empty_like(state)))) == 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step([3] * 8, 24)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_step(new, lengths, table, free, state, 16, 30)
    rng = random.Random(6)
    for _ in range(12):
        counts = [rng.choice((-1, 0, 1, 4)) for _ in range(8)]
        new.copy_(_ints(counts))
        graph.replay()
        want = oracle.step(counts, cache.lengths, cache.table, cache.free, cache.count, cache.status, 16, 30)
        cache.lengths, cache.table, cache.free, cache.count, cache.status = want[:5]
        torch.cuda.synchronize()
        assert [t.tolist() for t in out] == list(want[5:]) and lengths.tolist() == cache.lengths and table.tolist() == cache.table
        assert free.tolist() == cache.free and state.tolist() == [cache.count, cache.status]


def test_part_of_a_table():
    """Some sequences of a larger cache: rows of its table, entries of its lengths, and the stack of all."""
    cache = _Cache(6, 5, 20, 16, seed=7)
    lengths, table, free, state = cache.on_gpu
    ops.paged_step(_ints([20, 3]), lengths[2:4], table[2:4], free, state, 16, 23)
    want = oracle.step([20, 3], [0, 0], cache.table[2:4], cache.free, cache.count, 0, 16, 23)
    assert lengths.tolist() == [0, 0, 20, 3, 0, 0] and table[2:4].tolist() == want[1] and state.tolist() == [want[3], 0]
    assert table[:2].tolist() == cache.table[:2] and table[4:].tolist() == cache.table[4:]


def test_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    good = dict(new=i(3), lengths=i(3), page_table=i(3, 4), free_pages=i(12), state=i(2), page_size=16, tokens=5)
    ops.paged_step(**good)
    for bad in (dict(new=i(2)), dict(new=i(3).long()), dict(lengths=i(4)), dict(lengths=i(6)[::2]), dict(page_table=i(2, 4)), dict(page_table=i(4, 3).t()), dict(page_table=i(3, 4).long()),
                dict(page_table=i(1, 4).expand(3, 4)), dict(free_pages=i(3, 4)), dict(state=i(1)), dict(page_size=0), dict(page_size=17), dict(tokens=-1), dict(tokens=2 ** 24 + 1),
                dict(max_ctx=65), dict(max_ctx=0), dict(position_offset=i(2)), dict(ctx_len=i(2)), dict(state_out=i(3)), dict(new=torch.zeros(3, dtype=torch.int32)),
                dict(new=i(0), lengths=i(0), page_table=i(0, 4)), dict(page_table=i(3, 0))):
        with pytest.raises((RuntimeError, ValueError)):
            ops.paged_step(**{**good, **bad})
    x = i(3)
    with pytest.raises(RuntimeError, match="memory"):
        ops.paged_step(**{**good, "new": x, "lengths": x})   # lengths are written

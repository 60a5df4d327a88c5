"""The oracle of `ops.paged_step` against the paged cache whose steps the host plans, and the refusals of the C entry."""

import ctypes
import random

import pytest
import torch

from scaling_amd import _lib
from scaling_amd.nn import PagedKVCache
from tests import paged_step_oracle as oracle


def test_oracle_is_the_host_cache():
    """The same pages for the same sequences, and the same refusals."""
    rng = random.Random(5)
    page, n_pages, batch, max_ctx = 16, 40, 6, 150
    cache = PagedKVCache(1, n_pages, batch, max_ctx, 2, 1, 32, torch.bfloat16, "cpu", page)
    lengths, table, free, count = [0] * batch, cache._table.tolist(), list(cache._free), n_pages
    refused = 0
    for _ in range(300):
        new = [rng.choice((0, 1, 1, rng.randint(2, 40), -1)) for _ in range(batch)]
        for b, n in enumerate(new):
            if n < 0:
                cache.release(b)
        got = oracle.step(new, lengths, table, free, count, 0, page, 400, max_ctx)
        lengths, table, free, count, status, cu, positions, slots, sequences, last = got
        new = [max(n, 0) for n in new]
        try:
            step = cache.step(new)
        except (RuntimeError, ValueError):
            assert status != 0 or sum(new) == 0
            refused += status != 0
            assert cu[-1] == 0 and lengths == cache.lengths
            continue
        assert status == 0 and lengths == cache.lengths and count == cache.free_pages and free[:count] == cache._free
        assert all(table[b][:len(p)] == p for b, p in enumerate(cache._pages))
        assert cu == step.cu_seqlens.tolist() and positions[:cu[-1]] == step.position_ids.tolist() and lengths == step.ctx_len.tolist()
        assert [l for l, n in zip(last, new) if n] == step.last.tolist()
        assert [table[b][p // page] * page + p % page for b, p in zip(sequences, positions)][:cu[-1]] == slots[:cu[-1]]
    assert refused > 5


def test_entry_refuses():
    lib = _lib.load()
    assert lib.mi_paged_step(None) == -1
    a = _lib.MiPagedStepArgs()
    buf = (ctypes.c_char * 64)()
    base = ctypes.addressof(buf)
    a.batch, a.max_pages, a.page_size, a.n_free, a.tokens, a.max_ctx = 2, 4, 16, 8, 5, 0
    assert lib.mi_paged_step(ctypes.byref(a)) == -1
    for name, kind in _lib.MiPagedStepArgs._fields_:
        if kind is ctypes.c_void_p and name not in ("stream", "position_offset"):
            setattr(a, name, base)
    for name, value in (("batch", 0), ("batch", (1 << 24) + 1), ("max_pages", 0), ("page_size", 0), ("page_size", 1 << 29), ("n_free", -1), ("tokens", -1),
                        ("tokens", (1 << 24) + 1), ("max_ctx", 65), ("max_ctx", -1), ("page_table_stride", -1)):
        before = getattr(a, name)
        setattr(a, name, value)
        assert lib.mi_paged_step(ctypes.byref(a)) == -3, name
        setattr(a, name, before)
    a.batch, a.max_pages = 1 << 10, 1 << 21                                                  # sums of pages are kept in 32 bits
    assert lib.mi_paged_step(ctypes.byref(a)) == -3
    a.batch, a.max_pages = 2, 4
    for name in ("new_tokens", "lengths", "state", "ctx_len", "state_out", "page_table", "free_pages", "cu_seqlens", "last", "position_ids", "slots", "sequences"):
        setattr(a, name, None)
        assert lib.mi_paged_step(ctypes.byref(a)) == -1, name
        setattr(a, name, base)


def test_ops_refuse_without_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from scaling_amd import ops
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.paged_step(i(2), i(2), i(2, 3), i(6), i(2), 16, 2)

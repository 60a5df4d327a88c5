"""Attention with shared prefixes: the refusals of the C entry, and the size of its workspace."""

import ctypes

import pytest
import torch

from scaling_amd import _lib


def _arguments(base):
    a = _lib.MiPagedPrefixAttnArgs()
    t = a.attn
    for name in ("q", "k_pages", "v_pages", "o", "page_table", "cu_seqlens", "ctx_len"):
        setattr(t, name, base)
    a.prefix_table = a.prefix_len = a.group_seqs = base
    t.total_q, t.batch, t.n_pages, t.page_size, t.max_pages = 4, 2, 8, 16, 4
    t.n_q_heads, t.n_kv_heads, t.head_dim, t.dtype, t.causal, t.softmax_scale = 4, 2, 64, _lib.MI_BF16, 1, 0.125
    t.q_stride_token = t.o_stride_token = 256
    t.q_stride_head = t.o_stride_head = 64
    t.page_stride, t.page_stride_token, t.page_stride_head, t.page_table_stride = 2048, 64, 1024, 4
    a.n_groups, a.max_prefix_pages, a.prefix_table_stride = 1, 4, 4
    return a


def test_entry_refuses():
    lib = _lib.load()
    assert lib.mi_paged_prefix_attn(None) == -1
    buf = (ctypes.c_char * 64)()
    base = ctypes.addressof(buf)
    base += -base % 16
    a = _arguments(base)
    assert lib.mi_paged_prefix_attn(ctypes.byref(a)) == -5 and b"workspace needs" in lib.mi_last_error()
    for where, name, value, status in ((a, "n_groups", -1, -3), (a, "max_prefix_pages", 0, -3), (a, "max_prefix_pages", 1 << 27, -3), (a, "prefix_table", None, -1),
                                       (a, "prefix_len", None, -1), (a, "group_seqs", None, -1), (a.attn, "dtype", 2, -2), (a.attn, "q", None, -1),
                                       (a.attn, "head_dim", 80, -3), (a.attn, "page_size", 24, -3), (a.attn, "n_q_heads", 3, -3), (a.attn, "batch", 0, -3),
                                       (a.attn, "o", base + 2, -4), (a.attn, "q_stride_head", 60, -4), (a.attn, "softmax_scale", -1.0, -3)):
        before = getattr(where, name)
        setattr(where, name, value)
        assert lib.mi_paged_prefix_attn(ctypes.byref(a)) == status, (name, lib.mi_last_error())
        setattr(where, name, before)
    a.attn.total_q = 0
    a.attn.q = None
    assert lib.mi_paged_prefix_attn(ctypes.byref(a)) == 0


def test_workspace_suffices_for_every_bound_of_the_tokens():
    """What a call needs, which the entry says when it refuses, is no more than what the size asks for, nor does a larger size ask for less."""
    lib = _lib.load()
    buf = (ctypes.c_char * 64)()
    base = ctypes.addressof(buf)
    base += -base % 16
    size = lib.mi_paged_prefix_attn_workspace_bytes
    for nq, nkv, d in ((4, 4, 64), (32, 8, 128), (32, 1, 32), (20, 4, 96)):
        least = 0
        for tokens in (1, 3, 17, 40, 100, 300, 2000, 20000):
            for batch in (1, 7, 64, 500):
                for groups in (1, 5, 200):
                    have = size(tokens, batch, groups, nq, nkv, d)
                    assert have <= size(tokens + 1, batch, groups, nq, nkv, d) and have <= size(tokens, batch + 1, groups, nq, nkv, d) <= size(tokens, batch + 1, groups + 1, nq, nkv, d)
                    for longest in (0, 1, 2, 5, 40, tokens):
                        for pages in (1, 20, 1 << 20):
                            a = _arguments(base)
                            a.attn.total_q, a.attn.batch, a.n_groups, a.attn.max_q_len = tokens, batch, groups, longest
                            a.attn.n_q_heads, a.attn.n_kv_heads, a.attn.head_dim = nq, nkv, d
                            a.attn.max_pages = a.max_prefix_pages = pages
                            rc = lib.mi_paged_prefix_attn(ctypes.byref(a))
                            message = lib.mi_last_error().decode()
                            assert rc in (-5, -3), message
                            if rc == -5:
                                assert int(message.split("needs ")[1].split()[0]) <= have, (tokens, batch, groups, longest, pages, nq)
            assert size(tokens, 500, 200, nq, nkv, d) >= least
            least = size(tokens, 500, 200, nq, nkv, d)


def test_ops_refuse_without_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from scaling_amd import ops
    x, i = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.paged_prefix_attention(x, x, x, i, i, i, i, i, i)

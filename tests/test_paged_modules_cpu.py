"""Host side of the paged cache and of the modules' calls over it."""

import pytest
import torch

from scaling_amd import config as C
from scaling_amd.inference import TransformerInferenceModule
from scaling_amd.nn import PagedKVCache, PagedStep, ParallelSelfAttention
from tests.test_modules_cpu import _arch


def _cache(**kw):
    d = dict(num_layers=2, num_pages=5, max_sequences=3, max_ctx=70, n_q=4, n_kv=2, head_dim=64, dtype=torch.bfloat16, device="cpu", page_size=16)
    d.update(kw)
    return PagedKVCache(**d)


def _consistent(cache):
    used = [p for pages in cache._pages for p in pages]
    assert sorted(used + cache._free) == list(range(cache.k_pages[0].shape[0]))              # every page is somewhere once
    for b, pages in enumerate(cache._pages):
        assert len(pages) == -(-cache.lengths[b] // cache.page_size)
        assert cache.page_table[b, :len(pages)].tolist() == pages


def test_steps_and_their_lengths():
    cache = _cache()
    step = cache.step([17, 0, 1])
    _consistent(cache)
    assert step.cu_seqlens.tolist() == [0, 17, 17, 18] and step.cu_seqlens.dtype == torch.int32 and step.cu_seqlens.is_contiguous()
    assert step.ctx_len.tolist() == [17, 0, 1] and step.ctx_len.dtype == torch.int32
    assert step.position_ids.tolist() == list(range(17)) + [0] and step.position_ids.dtype == torch.int64
    assert step.last.tolist() == [16, 17] and (step.tokens, step.max_q_len, step.longest) == (18, 17, 17)
    step = cache.step([1, 3])                                                                # fewer entries than places: the first ones
    assert cache.lengths == [18, 3, 1] and step.cu_seqlens.tolist() == [0, 1, 4] and step.ctx_len.tolist() == [18, 3]
    assert step.position_ids.tolist() == [17, 0, 1, 2] and step.last.tolist() == [0, 3] and step.longest == 18
    assert cache.free_pages == 1
    _consistent(cache)
    cache.release(0)
    assert cache.free_pages == 3 and cache.lengths == [0, 3, 1]
    cache.step([33, 13, 15])                                                                 # fills pages to their ends, and the released ones again
    assert cache.free_pages == 0 and cache.lengths == [33, 16, 16]
    _consistent(cache)


def test_positions_of_many_sequences():
    step = PagedStep([2, 0, 3, 1], [5, 9, 3, 8], torch.device("cpu"))
    assert step.position_ids.tolist() == [3, 4, 0, 1, 2, 7] and step.last.tolist() == [1, 4, 5] and step.longest == 9
    assert step.position_ids.data_ptr() % 8 == 0 and step.cu_seqlens.data_ptr() % 4 == 0


def test_a_refused_step_takes_nothing():
    cache = _cache()
    cache.step([20, 16, 1])                                                                  # 2 + 1 + 1 of 5 pages
    for new, error in (([0, 33, 0], RuntimeError), ([51, 0, 0], ValueError), ([1, 1, 1, 1], ValueError), ([], ValueError), ([0, 0], ValueError), ([1, -1], ValueError)):
        with pytest.raises(error):
            cache.step(new)
        assert cache.lengths == [20, 16, 1] and cache.free_pages == 1
        _consistent(cache)
    for sequence in (-1, 3):
        with pytest.raises(IndexError):
            cache.release(sequence)
    cache.release(1)
    cache.release(1)                                                                         # of an empty place: nothing
    assert cache.free_pages == 2
    _consistent(cache)


def test_a_default_device_does_not_move_the_host_side():
    cache = _cache()
    with torch.device("meta"):
        step = cache.step([17, 0, 1])
    assert step.ctx_len.tolist() == [17, 0, 1] and cache.page_table[0, :2].tolist() == cache._pages[0]


def test_refused_caches():
    for kw in (dict(page_size=8), dict(page_size=24), dict(num_pages=0), dict(num_layers=0), dict(max_sequences=0), dict(max_ctx=0)):
        with pytest.raises(ValueError):
            _cache(**kw)
    with pytest.raises(NotImplementedError):
        _cache(dtype=torch.float32)


def _attention(**kw):
    d = dict(hidden_size=256, num_attention_heads=4, masked_softmax_config=C.MaskedSoftmaxConfig(kernel="hip"), rotary_config=C.RotaryConfig(dimensions=64, max_seq_length=32),
             device="cpu", dtype=torch.bfloat16, qkv_in_one=False, num_kv_heads=2)
    d.update(kw)
    return ParallelSelfAttention(**d)


def test_refused_calls():
    cache = _cache()
    step = cache.step([3, 1])
    x = torch.zeros(1, 4, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        _attention(causal=False).paged_forward(x, cache, 0, step)
    with pytest.raises(NotImplementedError):
        _attention(dtype=torch.float32).paged_forward(x.float(), cache, 0, step)
    with pytest.raises(ValueError):
        _attention().paged_forward(x[:, :3], cache, 0, step)
    with pytest.raises(IndexError):
        _attention().paged_forward(x, cache, 2, step)                                        # a layer that the cache does not have
    step = cache.step([30, 1])
    with pytest.raises(IndexError):
        _attention().paged_forward(torch.zeros(1, 31, 256, dtype=torch.bfloat16), cache, 0, step)      # position 32 of a table of 32


def test_refused_generation():
    model = TransformerInferenceModule(_arch(), device="cpu", seed=0)
    for tokens, prompts in ((0, [[1]]), (1, []), (1, [[1], []])):
        with pytest.raises(ValueError):
            model.generate_ragged(tokens, prompts)
    with pytest.raises(IndexError):
        model.generate_ragged(100, [[1], [2] * 30])                                          # position 128 of a table of 128
    cache = model.paged_cache(3, page_size=32)
    assert len(cache.k_pages) == 2 and cache.max_ctx == 128 and cache.free_pages == 12
    assert cache.k_pages[0].shape == (12, 32, 2, 64) and cache.k_pages[0].stride() == (4096, 64, 2048, 1)
    assert model.paged_cache(3, 40, 2).free_pages == 2


def test_norms_and_rotary_in_one_go_through_own_unhooked_modules_only():
    att = _attention(key_query_norm=True)
    assert att.norm_rotary_in_one is False and _attention(norm_rotary_in_one=True).norm_rotary_in_one
    del att.__dict__["norm_rotary_in_one"]                                                   # a module stored before there was the setting
    assert att.norm_rotary_in_one is False
    assert att._own_norms()["layer_norm"] and att._own_norms()["q_bias"] is att.norm_query.bias
    rotary, interleaved = att._own_rotary(None)
    assert rotary[0].shape == (32, 64) and not interleaved
    handle = att.norm_key.register_forward_hook(lambda *a: None)
    assert att._own_norms() is None
    handle.remove()
    assert att._own_norms() is not None
    att.norm_key.eps = 1e-3
    assert att._own_norms() is None
    att.rotary_embedding = torch.nn.Identity()
    assert att._own_rotary(None) == (None, False)

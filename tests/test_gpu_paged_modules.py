"""Norms, rotary, append and paged attention together, as the modules use them."""

import pytest
import torch

import oracle
from scaling_amd import ops
from scaling_amd.inference import TransformerInferenceModule
from scaling_amd.layer import InferenceSettings, TransformerLayer, TransformerLayerIO
from scaling_amd.nn import PagedKVCache, RotaryEmbedding
from tests.kernels import launched
from tests.parity import check
from tests.test_gpu_modules import _arch, _oracle_layer, _seeded_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"

LAYERS = [
    ("gqa_norms", dict(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, mlp_factor=2.5, key_query_norm=True)),
    ("gqa", dict(hidden_size=512, num_attention_heads=4, attention_num_kv_heads=2)),
    ("fused_qkv_bias", dict(attention_qkv_in_one=True, attention_bias=True, mlp_bias=True)),
    ("layernorm_gelu_norms", dict(norm_type="layernorm", mlp_type="default", mlp_factor=4.0, attention_bias=True, mlp_bias=True, key_query_norm=True)),
    ("complex_norms_float16", dict(precision="float16", relative_position_embedding_type="rotary_complex", key_query_norm=True)),
    ("partial_rotary", dict(rotary_percentage=0.5, key_query_norm=True)),
    ("no_rotary", dict(relative_position_embedding_type="none")),
]


@pytest.mark.parametrize("name,kw", LAYERS, ids=lambda x: x if isinstance(x, str) else "")
def test_layer_over_pages(name, kw):
    """Sequences that come in chunks, drafts and single tokens, one of them later than the others: the layer's outputs against the oracle's on whole sequences."""
    print(f"case {name}", flush=True)
    cfg = _arch(**kw)
    layer = _seeded_layer(cfg, seed=0).eval()
    dtype, g = cfg.precision.dtype, torch.Generator().manual_seed(2)
    steps = [[40, 7, 0], [1, 1, 0], [3, 1, 65], [1, 0, 1]]
    total = [sum(s[b] for s in steps) for b in range(3)]
    x = [torch.randn(n, cfg.hidden_size, generator=g).to(dtype) for n in total]
    att = layer.self_attention
    cache = PagedKVCache(1, 12, 3, 128, att.num_attention_heads, att.num_kv_heads_per_partition, att.hidden_size_per_attention_head, dtype, DEV, page_size=16)
    done, out = [0, 0, 0], [[], [], []]
    for new in steps:
        step = cache.step(new)
        h = torch.cat([x[b][done[b]:done[b] + n] for b, n in enumerate(new)]).to(DEV)
        y = layer.paged_step(h.view(1, -1, cfg.hidden_size), cache, step)[0].cpu()
        for b, part in enumerate(y.split(new)):
            out[b].append(part)
            done[b] += new[b]
    got = torch.cat([torch.cat(o) for o in out])
    cu = torch.tensor([0, total[0], total[0] + total[1], sum(total)], dtype=torch.int32)
    pos = torch.cat([torch.arange(n) for n in total]).view(1, -1)
    weights, whole = layer.state_dict(), torch.cat(x).view(1, -1, cfg.hidden_size)
    ref, order = (_oracle_layer(cfg, weights, whole, cu, pos, torch.ones_like(whole), t)[0] for t in (torch.float32, dtype))
    check(f"paged {name}", got.view_as(whole), ref, order, module_level=True)
    # the same layer without a cache sees the same
    plain = layer(TransformerLayerIO(activations=whole.to(DEV), position_ids=pos.to(DEV), cumulative_seq_lengths=cu.to(DEV))).activations
    check(f"uncached {name}", plain, ref, order, module_level=True)


def test_a_layer_launches_one_append_and_no_norms_of_its_own():
    cfg = _arch(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, key_query_norm=True)
    layer = _seeded_layer(cfg, seed=0).eval()
    cache = PagedKVCache(1, 12, 3, 64, 8, 2, 64, torch.bfloat16, DEV, page_size=16)
    x = torch.randn(1, 3, 512, device=DEV, dtype=torch.bfloat16)
    layer.paged_step(x, cache, cache.step([1, 1, 1]))
    step = cache.step([1, 1, 1])
    names = launched(lambda: layer.self_attention.paged_forward(x, cache, 0, step))
    assert sum("head_rows" in n for n in names) == 1 and sum("paged_rows" in n for n in names) == 1 and not any("norm" in n for n in names if "head_rows" not in n), names


@pytest.mark.parametrize("kw", [dict(norm_type="layernorm", mlp_type="default", mlp_factor=4.0), dict(), dict(rotary_percentage=0.5),
                                dict(relative_position_embedding_type="rotary_complex", attention_qkv_in_one=True), dict(relative_position_embedding_type="none"),
                                dict(attention_num_kv_heads=2, precision="float32")],
                         ids=["layernorm", "rms", "partial", "complex", "none", "float32"])
def test_training_with_norms_and_rotary_in_one(kw):
    """Outputs and gradients of a layer against the oracle's; the setting is off unless asked for."""
    cfg = _arch(key_query_norm=True, **kw)
    layer = _seeded_layer(cfg, seed=0)
    dtype, g = cfg.precision.dtype, torch.Generator().manual_seed(1)
    b, s = 2, 96
    x, dy = (torch.randn(b, s, cfg.hidden_size, generator=g).to(dtype) for _ in range(2))
    cu, pos = torch.tensor([0, 40, s, 2 * s], dtype=torch.int32), torch.cat([torch.arange(40), torch.arange(s - 40), torch.arange(s)]).view(b, s)
    ref = _oracle_layer(cfg, layer.state_dict(), x, cu, pos, dy, torch.float32)
    order = _oracle_layer(cfg, layer.state_dict(), x, cu, pos, dy, dtype)

    def run():
        layer.zero_grad()
        xg = x.to(DEV).requires_grad_()
        y = layer(TransformerLayerIO(activations=xg, position_ids=pos.to(DEV), cumulative_seq_lengths=cu.to(DEV))).activations
        y.backward(dy.to(DEV))
        return y.detach(), xg.grad, {k: p.grad.clone() for k, p in layer.named_parameters()}

    assert not any("head_rows" in n for n in launched(run))
    layer.self_attention.norm_rotary_in_one = True
    names = launched(run)
    assert sum("head_rows" in n for n in names) >= 2, names
    y, dx, grads = run()
    check("y", y, ref[0], order[0], module_level=True)
    check("dx", dx, ref[1], order[1], module_level=True)
    for k in ("self_attention.norm_query.weight", "self_attention.norm_key.weight"):
        # as far from the exact ones as the reference's order is, the rounding of the result, and what float32 evaluations of 28 roundings each are apart
        exact = ref[2][k].double()
        off, theirs = (grads[k].cpu().double() - exact).norm(), (order[2][k].double() - exact).norm()
        assert off <= 1.25 * theirs + (torch.finfo(dtype).eps / 2 + 2 * 28 * 2.0 ** -24) * exact.norm(), (k, float(off), float(theirs))


def _model(**kw):
    d = dict(precision="float16", key_query_norm=True, hidden_size=256, num_attention_heads=4, attention_num_kv_heads=2, num_layers=2)
    d.update(kw)
    return TransformerInferenceModule(_arch(**d), device=DEV, init_std=0.1, seed=5)


# Final rows are off by at most half a step of the type for each of 28 roundings on the way (13 stored tensors a layer, final norm and head), twice as two
# evaluations are compared; a logit by that of the row's size times the size of the head's row.
def _margin(model):
    weight = model._layers[-1].linear.weight
    return 2 * 28 * 2.0 ** -11 * float(weight.detach().float().norm(dim=1).max()) * weight.shape[1] ** 0.5


def _uncached(model, ids):
    """logits of one document, whatever ids it has (by itself `forward` starts another one behind id 0)"""
    return model.forward(ids.view(1, -1), torch.arange(len(ids)).view(1, -1), torch.tensor([0, len(ids)], dtype=torch.int32))[0]


PROMPTS = [[5, 17, 3, 90, 41, 8, 63], [7], list(range(1, 71)), [44, 2, 9] * 6]


def test_ragged_generation():
    """Every id is a greedy choice of the uncached model, within what its logits are off by."""
    model = _model()
    out = model.generate_ragged(9, PROMPTS, page_size=16)
    assert [len(o) for o in out] == [9] * 4
    margin = _margin(model)
    for prompt, ids in zip(PROMPTS, out):
        logits = _uncached(model, torch.tensor(prompt + ids))[len(prompt) - 1:-1].float()
        behind = logits.max(dim=1).values - logits.gather(1, torch.tensor(ids, device=DEV).view(-1, 1))[:, 0]
        print(f"prompt of {len(prompt)}: behind the best by {float(behind.max()):.4f} of {margin:.4f}, spread {float(logits.std()):.2f}", flush=True)
        assert float(behind.max()) <= margin
    assert model.generate_ragged(9, PROMPTS, page_size=16) == out
    assert model.generate_ragged(1, PROMPTS) == [o[:1] for o in out]


def test_stop_tokens_end_a_sequence():
    model = _model()
    free = model.generate_ragged(8, PROMPTS, page_size=16)
    stop = free[1][2]
    out = model.generate_ragged(8, PROMPTS, stop_tokens=[stop], page_size=16)
    first = min(o.index(stop) for o in free if stop in o)                # the batch is the same until somebody leaves it
    for a, b in zip(out, free):
        assert a[:first + 1] == b[:first + 1]
        assert (stop not in a[:-1]) and (len(a) == 8 or a[-1] == stop)


def test_sequences_come_and_go():
    """A place and its pages are used again by another sequence, beside one that goes on: logits against the uncached model's."""
    model = _model()
    cache = model.paged_cache(2, 64, 6, page_size=16)
    g = torch.Generator().manual_seed(0)
    a, b, c = (torch.randint(0, 96, (n,), generator=g) for n in (30, 33, 50))
    margin = _margin(model)

    def behind(logits, *sequences):
        for row, s in zip(logits, sequences):
            want = _uncached(model, s)[-1]
            assert float((row.float() - want.float()).abs().max()) <= margin

    behind(model.paged_forward(torch.cat([a[:20], b]), cache, cache.step([20, 33])), a[:20], b)
    behind(model.paged_forward(a[20:21], cache, cache.step([1])), a[:21])
    cache.release(1)
    behind(model.paged_forward(torch.cat([a[21:24], c[:40]]), cache, cache.step([3, 40])), a[:24], c[:40])
    behind(model.paged_forward(torch.cat([a[24:30], c[40:]]), cache, cache.step([6, 10])), a, c)
    with pytest.raises(RuntimeError):
        cache.step([30, 0])
    behind(model.paged_forward(torch.cat([a[:1], c[:1]]), cache, cache.step([1, 1])), torch.cat([a, a[:1]]), torch.cat([c, c[:1]]))


def test_another_stream_and_a_captured_step():
    """A step of a layer on a side stream, and one captured and replayed with other activations, have the bits of the plain call."""
    cfg = _arch(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, key_query_norm=True)
    layer = _seeded_layer(cfg, seed=0).eval()
    make = lambda: PagedKVCache(1, 12, 3, 64, 8, 2, 64, torch.bfloat16, DEV, page_size=16)       # noqa: E731
    caches = [make() for _ in range(3)]
    prompt = torch.randn(1, 50, 512, device=DEV, dtype=torch.bfloat16)
    token = torch.randn(1, 3, 512, device=DEV, dtype=torch.bfloat16)
    for cache in caches:
        layer.paged_step(prompt, cache, cache.step([20, 1, 29]))
    with torch.no_grad():
        want = layer.paged_step(token, caches[0], caches[0].step([1, 1, 1]))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = layer.paged_step(token, caches[1], caches[1].step([1, 1, 1]))
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        cache = caches[2]
        step = cache.step([1, 1, 1])
        x = torch.zeros_like(token)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.paged_step(x, cache, step)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.paged_step(x, cache, step)
        held = cache.workspace()
        cache.workspace()
        assert cache.workspace() is held                     # what the graph reads stays where it is
        for _ in range(3):
            x.zero_()
            graph.replay()
            assert not torch.equal(y, want)
            x.copy_(token)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_the_first_call_over_a_cache_may_be_a_captured_one():
    """What the calls over a cache share is ready before any of them: an eager call in front of the graph's first replay, and the replays."""
    cfg = _arch(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, key_query_norm=True, sequence_length=1024)
    layer = _seeded_layer(cfg, seed=0).eval()
    g = torch.Generator().manual_seed(3)
    fill = [torch.randn(24, 2, 64, 64, generator=g).bfloat16().to(DEV).transpose(1, 2) for _ in range(2)]
    x = torch.randn(1, 2, 512, generator=g).bfloat16().to(DEV)

    def make():
        cache = PagedKVCache(1, 24, 2, 1024, 8, 2, 64, torch.bfloat16, DEV, page_size=64)
        cache.k_pages[0].copy_(fill[0])
        cache.v_pages[0].copy_(fill[1])
        cache.step([700, 500])
        return cache, cache.step([1, 1])

    with torch.no_grad():
        want = layer.paged_step(x, *make())                  # (the projections' libraries are ready, too)
        cache, step = make()
        assert cache._workspace is not None and int(cache._workspace.tickets.abs().sum()) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.paged_step(x, cache, step)
            made_inside = ops.paged_workspace(2, 2, 8, 2, 64, DEV)
        assert not hasattr(made_inside, "tickets")
        for _ in range(3):
            assert torch.equal(layer.paged_step(x, cache, step), want)
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
        assert int(cache.workspace().tickets.abs().sum()) == 0


@pytest.mark.parametrize("kw", [dict(norm_type="layernorm", mlp_type="default", mlp_factor=4.0), dict(relative_position_embedding_type="rotary_complex")], ids=["layernorm", "complex"])
def test_cached_calls_round_their_keys_alike(kw):
    """With the setting on, a prompt and the tokens behind it go into a KVCache as they do without it; a call without a cache is the one that takes the launch."""
    cfg = _arch(key_query_norm=True, **kw)
    layer = _seeded_layer(cfg, seed=0).eval()
    att, g = layer.self_attention, torch.Generator().manual_seed(4)
    x = torch.randn(2, 21, cfg.hidden_size, generator=g).to(cfg.precision.dtype).to(DEV)

    def io(a, b, settings):
        s = b - a
        return TransformerLayerIO(activations=x[:, a:b], position_ids=torch.arange(a, b, device=DEV).repeat(2, 1), cumulative_seq_lengths=torch.tensor([0, s, 2 * s], dtype=torch.int32, device=DEV),
                                  inference_settings=settings)

    def generate():
        with torch.no_grad():
            out = [layer(io(0, 19, InferenceSettings(use_cache=True, reset_cache=True))).activations] + \
                [layer(io(i, i + 1, InferenceSettings(use_cache=True, reset_cache=False))).activations for i in (19, 20)]
        return (*out, att.cache[0].k[:, :21].clone(), att.cache[0].v[:, :21].clone())
    plain = generate()
    att.norm_rotary_in_one = True
    assert not any("head_rows" in n for n in launched(generate))
    for a, b in zip(plain, generate()):
        assert torch.equal(a, b)
    assert sum("head_rows" in n for n in launched(lambda: layer(io(0, 19, None)))) == 1


def test_a_step_is_not_captured():
    cache = PagedKVCache(1, 12, 3, 64, 8, 2, 64, torch.bfloat16, DEV, page_size=16)
    cache.step([5, 1])
    x = torch.zeros(8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="capture"):
            cache.step([20, 1])
    assert cache.lengths == [5, 1, 0] and cache.free_pages == 10
    assert cache.step([20, 1]).ctx_len.tolist() == [25, 2]


class _Rotary(RotaryEmbedding):
    """A rotary of somebody's own: the package's arithmetic, in another class."""

    def rotate_tokens(self, *args, **kwargs):
        self.calls = getattr(self, "calls", 0) + 1
        return super().rotate_tokens(*args, **kwargs)


@pytest.mark.parametrize("hooked,replaced", [(True, False), (False, True), (True, True)], ids=["hooked-norm", "replaced-rotary", "both"])
def test_norms_and_rotary_of_somebodys_own(hooked, replaced):
    """Over pages and, with the setting on, in a training step: what was hooked or replaced is called, and the outputs are the layer's."""
    cfg = _arch(key_query_norm=True, rotary_percentage=0.5)     # (the rotary of a whole head is the attention kernels', by its tables)
    layer = _seeded_layer(cfg, seed=0)
    att, dtype, g = layer.self_attention, cfg.precision.dtype, torch.Generator().manual_seed(6)
    att.norm_rotary_in_one = True
    seen = []
    if hooked:
        att.norm_key.register_forward_hook(lambda module, args, out: seen.append(out.shape[0]))
    if replaced:
        att.rotary_embedding.__class__ = _Rotary
    n = 37
    x, dy = (torch.randn(1, n, cfg.hidden_size, generator=g).to(dtype) for _ in range(2))
    cu, pos = torch.tensor([0, n], dtype=torch.int32), torch.arange(n).view(1, n)
    ref, order = (_oracle_layer(cfg, layer.state_dict(), x, cu, pos, dy, t) for t in (torch.float32, dtype))

    def train():
        xg = x.to(DEV).requires_grad_()
        y = layer(TransformerLayerIO(activations=xg, position_ids=pos.to(DEV), cumulative_seq_lengths=cu.to(DEV))).activations
        y.backward(dy.to(DEV))
        return y.detach(), xg.grad
    names = launched(train)
    assert any("head_rows" in name for name in names) == (not hooked), names       # norms alone where the rotary is another's
    y, dx = train()
    check("y", y, ref[0], order[0], module_level=True)
    check("dx", dx, ref[1], order[1], module_level=True)
    assert (not hooked or seen == [n, n]) and (not replaced or att.rotary_embedding.calls == 4)
    layer.eval()
    cache = PagedKVCache(1, 8, 1, 64, 4, 4, 64, dtype, DEV, page_size=16)
    out = [layer.paged_step(x[:, a:b].to(DEV), cache, cache.step([b - a])) for a, b in ((0, 20), (20, 36), (36, n))]
    check("paged", torch.cat(out, 1), ref[0], order[0], module_level=True)
    assert (not hooked or seen[2:] == [20, 16, 1]) and (not replaced or att.rotary_embedding.calls == 10)

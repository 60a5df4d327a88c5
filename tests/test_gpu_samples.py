"""Sampling, steps planned on the GPU and attention over shared prefixes together, as the modules use them."""

import pytest
import torch

from scaling_amd import ops
from scaling_amd.nn import PagedBranches, PagedKVCache
from tests.parity import check
from tests.test_gpu_modules import _arch, _oracle_layer, _seeded_layer
from tests.test_gpu_paged_modules import PROMPTS, _margin, _model, _uncached

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("name,kw", [("gqa_norms", dict(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, mlp_factor=2.5, key_query_norm=True)),
                                     ("complex_float16", dict(precision="float16", relative_position_embedding_type="rotary_complex")),
                                     ("no_rotary_fused_qkv", dict(relative_position_embedding_type="none", attention_qkv_in_one=True, attention_bias=True))],
                         ids=lambda x: x if isinstance(x, str) else "")
def test_layer_over_branches(name, kw):
    """Three branches of each of two prompts, with single tokens, drafts, idle ones and one that ends and starts again: outputs against the oracle's on whole sequences."""
    print(f"case {name}", flush=True)
    cfg = _arch(**kw)
    layer = _seeded_layer(cfg, seed=0).eval()
    dtype, g, att = cfg.precision.dtype, torch.Generator().manual_seed(2), layer.self_attention
    prompts = [torch.randn(n, cfg.hidden_size, generator=g).to(dtype) for n in (40, 7)]
    steps = [[1, 1, 1, 1, 1, 1], [3, 0, 20, 1, 2, 0], [1, -1, 1, 0, 1, 1], [1, 4, 0, 1, 1, 18]]
    total = [sum(max(s[b], 0) for s in steps) for b in range(6)]
    x = [torch.randn(n, cfg.hidden_size, generator=g).to(dtype) for n in total]
    cache = PagedKVCache(1, 30, 2, 64, att.num_attention_heads, att.num_kv_heads_per_partition, att.hidden_size_per_attention_head, dtype, DEV, page_size=16)
    h = layer.paged_step(torch.cat(prompts).to(DEV).view(1, -1, cfg.hidden_size), cache, cache.step([40, 7]))
    free = cache.free_pages
    branches = PagedBranches(cache, [0, 1], 3, 32, 14)
    assert cache.free_pages == free - 14
    done, out = [0] * 6, [[] for _ in range(6)]
    for new in steps:
        tokens = sum(max(n, 0) for n in new) + 2            # rows that belong to nobody
        plan = branches.step(_ints(new), tokens, max(new))
        h = torch.cat([x[b][done[b]:done[b] + max(n, 0)] for b, n in enumerate(new)] + [x[0][:1]] * 2).to(DEV)
        y = layer.paged_step(h.view(1, -1, cfg.hidden_size), cache, plan)[0].cpu()
        for b, part in enumerate(y[:tokens - 2].split([max(n, 0) for n in new])):
            out[b].append(part)
            done[b] += max(new[b], 0)
    branches.check()
    assert branches.ctx_len.tolist() == [6, 4, 22, 3, 5, 20]
    branches.close()
    assert cache.free_pages == free and sorted(cache._free) == sorted(set(cache._free))
    # whole sequences: the second branch's tokens after its end follow the prompt again
    parts, got = [], []
    for b in range(6):
        pieces = [x[b][:1], x[b][1:]] if b == 1 else [x[b]]
        for piece in pieces:
            parts.append(torch.cat((prompts[b // 3], piece)))
        got += [torch.cat(out[b])[:1], torch.cat(out[b])[1:]] if b == 1 else [torch.cat(out[b])]
    ends = torch.tensor([0] + [len(p) for p in parts]).cumsum(0)
    cu, pos, whole = ends.to(torch.int32), torch.cat([torch.arange(len(p)) for p in parts]).view(1, -1), torch.cat(parts).view(1, -1, cfg.hidden_size)
    refs = [_oracle_layer(cfg, layer.state_dict(), whole, cu, pos, torch.ones_like(whole), t)[0][0] for t in (torch.float32, dtype)]
    ref, order = (torch.cat([r[ends[i] + len(parts[i]) - len(got[i]):ends[i + 1]] for i in range(len(parts))]) for r in refs)
    check(f"branches {name}", torch.cat(got), ref, order, module_level=True)


def _logprobs(model, prompt, ids):
    return torch.log_softmax(_uncached(model, torch.tensor(prompt + ids))[len(prompt) - 1:-1].float(), dim=-1)


def test_samples_follow_the_model():
    """Log-probabilities are those of the uncached model, within what its logits are off by (twice: a logit and the logarithm of the sum); so are greedy choices."""
    model = _model()
    margin = _margin(model)
    ids, logprobs = model.generate_samples(9, PROMPTS, 3, page_size=16, generator=torch.Generator(device=DEV).manual_seed(0))
    assert [[len(s) for s in p] for p in ids] == [[9] * 3] * 4 == [[len(s) for s in p] for p in logprobs]
    assert len({tuple(s) for p in ids for s in p}) > 6
    worst = 0.0
    for prompt, answers, lps in zip(PROMPTS, ids, logprobs):
        for answer, lp in zip(answers, lps):
            want = _logprobs(model, prompt, answer).gather(1, torch.tensor(answer, device=DEV).view(-1, 1))[:, 0]
            worst = max(worst, float((torch.tensor(lp, device=DEV) - want).abs().max()))
    print(f"log-probabilities off by {worst:.4f} of {2 * margin:.4f}", flush=True)
    assert worst <= 2 * margin
    greedy, zeros = model.generate_samples(9, PROMPTS, 2, temperature=0.0, page_size=16)
    assert all(lp == 0.0 for p in zeros for s in p for lp in s)
    for prompt, answers in zip(PROMPTS, greedy):
        for answer in answers:
            lp = _logprobs(model, prompt, answer)
            assert float((lp.max(dim=1).values - lp.gather(1, torch.tensor(answer, device=DEV).view(-1, 1))[:, 0]).max()) <= margin


@pytest.mark.parametrize("kw", [dict(), dict(key_query_norm=False, norm_type="layernorm", mlp_type="default", mlp_factor=4.0, attention_qkv_in_one=True, attention_num_kv_heads=None)],
                         ids=["rms", "layernorm"])
def test_a_captured_loop_draws_what_an_eager_one_does(kw):
    """With and without stop tokens, which end some answers and not others; the given numbers decide."""
    model = _model(**kw)
    u = torch.rand(20, 12, generator=torch.Generator().manual_seed(1))
    parameters = dict(samples=3, temperature=0.8, top_k=40, top_p=0.95, min_p=0.001, uniforms=u, page_size=16)
    free = model.generate_samples(20, PROMPTS, graph=False, **parameters)
    assert model.generate_samples(20, PROMPTS, graph=True, **parameters) == free
    assert model.generate_samples(20, PROMPTS, graph=True, **parameters) == free
    first = model.generate_samples(1, PROMPTS, **{**parameters, "uniforms": u[:1]})
    assert first[0] == [[s[:1] for s in p] for p in free[0]]
    stop = [free[0][0][0][4], free[0][2][1][7], free[0][3][2][0]]
    ended = model.generate_samples(20, PROMPTS, stop_tokens=stop, graph=False, **parameters)
    assert model.generate_samples(20, PROMPTS, stop_tokens=stop, graph=True, **parameters) == ended
    lengths = [len(s) for p in ended[0] for s in p]
    assert min(lengths) < 20
    for p, (some, every) in enumerate(zip(ended[0], free[0])):
        for a, b in zip(some, every):
            assert not set(a[:-1]) & set(stop) and (len(a) == 20 or a[-1] in stop)
    assert ended[0][3][2] == free[0][3][2][:1]              # drawn before anybody left
    assert [[len(s) for s in p] for p in ended[1]] == [[len(s) for s in p] for p in ended[0]]


def test_everybody_ends_early():
    model = _model()
    every = list(range(model.architecture_config.vocab_size))
    ids, logprobs = model.generate_samples(40, PROMPTS, 2, stop_tokens=every, page_size=16)
    assert [[len(s) for s in p] for p in ids] == [[1] * 2] * 4


def test_branches_refuse_and_tell():
    cache = PagedKVCache(1, 10, 2, 64, 4, 2, 64, torch.bfloat16, DEV, page_size=16)
    cache.step([20, 3])
    for bad in (([], 1, 4), ([2], 1, 4), ([0], 0, 4), ([0], 1, 0)):
        with pytest.raises(ValueError):
            PagedBranches(cache, *bad)
    with pytest.raises(RuntimeError):
        PagedBranches(cache, [0], 8, 16)
    assert cache.free_pages == 7
    branches = PagedBranches(cache, [0, 1], 2, 40, 5)
    branches.step(_ints([17, 1, 1, 0]), 19, 17)
    branches.check()
    branches.step(_ints([0, 16, 16, 16]), 48, 16)            # three pages, one is left
    branches.step(_ints([24, 0, 0, 0]), 24, 24)              # 41 keys
    branches.step(_ints([1, 1, 0, 0]), 1, 1)
    with pytest.raises(RuntimeError, match="pages ran out.*pass 40 tokens.*more tokens than rows"):
        branches.check()
    assert branches.ctx_len.tolist() == [17, 1, 1, 0]
    other = PagedKVCache(1, 10, 2, 64, 4, 2, 64, torch.bfloat16, DEV, page_size=16)
    layer = _seeded_layer(_arch(num_attention_heads=4, attention_num_kv_heads=2, hidden_size=256), seed=0).eval()
    plan = branches.step(_ints([1, 0, 0, 0]), 1, 1)
    with pytest.raises(ValueError, match="another cache"):
        layer.paged_step(torch.zeros(1, 1, 256, dtype=torch.bfloat16, device=DEV), other, plan)


def test_generation_refuses():
    model = _model()
    for bad in (dict(max_tokens=0), dict(samples=0), dict(prompts=[]), dict(prompts=[[1], []]), dict(uniforms=torch.zeros(2, 3)), dict(uniforms=torch.zeros(3, 2).double())):
        with pytest.raises(ValueError):
            model.generate_samples(**{**dict(max_tokens=3, prompts=[[1, 2]], samples=2), **bad})
    with pytest.raises(IndexError):
        model.generate_samples(100, [[1], [2] * 30], 2)


def test_other_numbers_other_answers_on_another_stream():
    """Two loops at once on two streams, each with its own graph, state and scratch."""
    model = _model()
    u = [torch.rand(12, 6, generator=torch.Generator().manual_seed(s)) for s in (3, 4)]
    want = [model.generate_samples(12, PROMPTS[:3], 2, uniforms=x, page_size=16) for x in u]
    assert want[0] != want[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert model.generate_samples(12, PROMPTS[:3], 2, uniforms=u[1], page_size=16) == want[1]
    torch.cuda.current_stream().wait_stream(side)
    assert ops.sample_rows(torch.zeros(1, 4, device=DEV), torch.zeros(1, device=DEV)).tolist() == [0]


def test_branches_of_one_sequence_twice_and_of_an_empty_one():
    """The same sequence named twice, and one that holds nothing yet: what branches of each by itself give."""
    cfg = _arch(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, mlp_factor=2.5)
    layer = _seeded_layer(cfg, seed=0).eval()
    dtype, att, g = cfg.precision.dtype, layer.self_attention, torch.Generator().manual_seed(7)
    prompt, x = torch.randn(37, cfg.hidden_size, generator=g).to(dtype), torch.randn(4, cfg.hidden_size, generator=g).to(dtype).to(DEV)

    def outputs(sequences, rows):
        cache = PagedKVCache(1, 40, 2, 64, att.num_attention_heads, att.num_kv_heads_per_partition, att.hidden_size_per_attention_head, dtype, DEV, page_size=16)
        layer.paged_step(prompt.to(DEV).view(1, -1, cfg.hidden_size), cache, cache.step([37, 0]))
        branches = PagedBranches(cache, sequences, 1, 16)
        out = [layer.paged_step(x[rows].view(1, -1, cfg.hidden_size), cache, branches.step(_ints([1] * len(rows)), len(rows), 1))[0] for _ in range(3)]
        branches.check()
        return torch.stack(out, 1)
    together = outputs([0, 0, 1, 0], [0, 1, 2, 0])
    assert torch.equal(together[0], together[3]) and not torch.equal(together[0], together[1])
    alone = torch.cat([outputs([0], [0]), outputs([0], [1]), outputs([1], [2])])
    # values of about 1 through one layer of 16-bit roundings, in products and sums cut otherwise for other batches: a few steps
    assert float((together[:3].float() - alone.float()).abs().max()) <= 16 * torch.finfo(dtype).eps * float(alone.float().abs().max())


def test_replays_behind_the_end():
    """A captured step of branches, replayed after they were closed and their pages went to another sequence: it takes nothing, says so, and leaves the pages alone."""
    cfg = _arch(hidden_size=512, num_attention_heads=8, attention_num_kv_heads=2, mlp_factor=2.5)
    layer = _seeded_layer(cfg, seed=0).eval()
    dtype, att, g = cfg.precision.dtype, layer.self_attention, torch.Generator().manual_seed(11)
    rows = lambda n: torch.randn(1, n, cfg.hidden_size, generator=g).to(dtype).to(DEV)
    cache = PagedKVCache(1, 5, 2, 64, att.num_attention_heads, att.num_kv_heads_per_partition, att.hidden_size_per_attention_head, dtype, DEV, page_size=16)
    layer.paged_step(rows(20), cache, cache.step([20, 0]))
    branches = PagedBranches(cache, [0], 3, 16)
    x, new = rows(3), _ints([1, 1, 1])
    step = lambda: layer.paged_step(x, cache, branches.step(new, 3, 1))
    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
    branches.check()
    assert branches.ctx_len.tolist() == [5, 5, 5]
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x.add(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            branches.close()
    branches.close()
    layer.paged_step(rows(48), cache, cache.step([0, 48]))       # all that they had
    assert cache.free_pages == 0
    pages = [t.clone() for t in (cache.k_pages[0], cache.v_pages[0])]
    for now in ([1, 1, 1], [-1, 1, 0], [1, 0, -1]):
        new.copy_(_ints(now))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.k_pages[0], pages[0]) and torch.equal(cache.v_pages[0], pages[1])
        assert branches.ctx_len.tolist() == [0, 0, 0] and branches.state.tolist() == [0, 1]
    with pytest.raises(RuntimeError, match="pages ran out"):
        branches.check()


class _Loop:
    """Branches of one prompt through one layer, whose outputs are the next inputs; every step's are kept."""

    def __init__(self, layer, cfg, seed, prompt, count, steps):
        att, dtype, g = layer.self_attention, cfg.precision.dtype, torch.Generator().manual_seed(seed)
        rows = lambda n: torch.randn(1, n, cfg.hidden_size, generator=g).to(dtype).to(DEV)
        self.layer, self.count = layer, count
        self.cache = PagedKVCache(1, -(-prompt // 16) + count * 8, 1, prompt, att.num_attention_heads, att.num_kv_heads_per_partition, att.hidden_size_per_attention_head, dtype, DEV,
                                  page_size=16)
        layer.paged_step(rows(prompt), self.cache, self.cache.step([prompt]))
        self.branches = PagedBranches(self.cache, [0], count, 128)
        self.x, self.drafts, self.one, self.at = rows(count), rows(20 * count), _ints([1] * count), torch.zeros(1, dtype=torch.int64, device=DEV)
        self.out = torch.zeros(steps, count, cfg.hidden_size, dtype=dtype, device=DEV)

    def step(self):
        y = self.layer.paged_step(self.x, self.cache, self.branches.step(self.one, self.count, 1))
        self.out.index_copy_(0, self.at, y)
        self.at.add_(1)
        self.x.copy_(y / y.float().square().mean(-1, keepdim=True).sqrt().to(y.dtype))

    def draft(self, n):
        self.layer.paged_step(self.drafts[:, :n * self.count], self.cache, self.branches.step(_ints([n] * self.count), n * self.count, n))

    def capture(self, stream):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            self.step()
        return graph


def _wide_layer():
    cfg = _arch(hidden_size=1024, num_attention_heads=8, attention_num_kv_heads=2, mlp_factor=2.5, sequence_length=4096)
    return cfg, _seeded_layer(cfg, seed=0).eval()


def test_two_captured_loops_run_at_once():
    """Two caches, each with branches, a captured step and scratch of its own: replayed on two streams that run at the same time, they give what each gives alone."""
    cfg, layer = _wide_layer()
    steps, alone = 14, []
    shapes = ((3, 700, 40), (4, 3000, 24))
    for seed, prompt, count in shapes:
        loop = _Loop(layer, cfg, seed, prompt, count, steps)
        for _ in range(steps):
            loop.step()
        loop.branches.check()
        alone.append(loop.out)
    loops, streams = [_Loop(layer, cfg, *shape, steps) for shape in shapes], [torch.cuda.Stream() for _ in shapes]
    for loop in loops:
        loop.step()
        loop.step()
    graphs = [loop.capture(stream) for loop, stream in zip(loops, streams)]
    torch.cuda.synchronize()
    for stream in streams:                                   # both wait until everything is issued
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)
    for _ in range(steps - 2):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for loop, want in zip(loops, alone):
        loop.branches.check()
        assert bool(torch.isfinite(want.float()).all()) and torch.equal(loop.out, want)


def test_a_captured_step_keeps_its_scratch():
    """Drafts between replays need more scratch than the captured step has, and what they leave is others' memory then: the replays give what eager steps do."""
    cfg, layer = _wide_layer()
    graph, outs = None, []
    for captured in (False, True):
        loop = _Loop(layer, cfg, 5, 900, 30, 9)
        loop.step()
        first = loop.branches.workspace(30).data_ptr()
        if captured:
            graph = loop.capture(torch.cuda.Stream())
        for drafts in (0, 2, 0, 20, 0, 5, 1, 0):
            if drafts:
                loop.draft(drafts)
            held = [torch.full((1 << 22,), float("nan"), device=DEV) for _ in range(16)]
            if captured:
                graph.replay()
            else:
                loop.step()
            torch.cuda.synchronize()
            del held
        loop.branches.check()
        assert loop.branches.workspace(30).data_ptr() != first
        outs.append(loop.out)
    assert bool(torch.isfinite(outs[0].float()).all()) and torch.equal(outs[0], outs[1])


def test_generation_is_on_the_module_s_device(monkeypatch):
    """Streams and graphs belong to a device, the current one unless told otherwise: they are made where the module's is current."""
    model, current, made = _model(), [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            current.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            current.pop()
            return super().__exit__(*args)
    stream, graph = torch.cuda.Stream, torch.cuda.graph
    monkeypatch.setattr(torch.cuda, "device", Device)

    def of_current(make):
        def call(*a, **kw):
            if make is graph or not (a or kw):               # (torch itself makes streams that it names)
                made.append(list(current))
            return make(*a, **kw)
        return call
    monkeypatch.setattr(torch.cuda, "Stream", of_current(stream))
    monkeypatch.setattr(torch.cuda, "graph", of_current(graph))
    want = model.generate_samples(6, PROMPTS, 2, uniforms=torch.full((6, 8), 0.4), page_size=16)
    assert len(made) >= 2 and all(made), made
    assert not current and [len(s) for p in want[0] for s in p] == [6] * 8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_generation_under_another_default_type(dtype):
    model = _model()
    u = torch.rand(5, 8, generator=torch.Generator().manual_seed(9))
    want = model.generate_samples(5, PROMPTS, 2, uniforms=u, page_size=16)
    drawn = model.generate_samples(5, PROMPTS, 2, generator=torch.Generator(device=DEV).manual_seed(9), page_size=16)
    torch.set_default_dtype(dtype)
    try:
        got = model.generate_samples(5, PROMPTS, 2, uniforms=u, page_size=16)
        again = model.generate_samples(5, PROMPTS, 2, generator=torch.Generator(device=DEV).manual_seed(9), page_size=16)
    finally:
        torch.set_default_dtype(torch.float32)
    assert got == want and again == drawn

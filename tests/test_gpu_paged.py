"""Paged KV cache: appends and attention of ragged chunks over it, against float64."""

import math

import pytest
import torch

from scaling_amd import ops
from tests import paged_oracle as oracle
from tests.kernels import launched
from tests.test_gpu_head_rows import ROUNDINGS, _close, _tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cache(new, ctx, nkv, d, page, dtype, seed, layout="heads", extra=2, stale=math.nan, spare=1):
    """pages with valid keys in the slots of ctx and `stale` elsewhere, page table (entries past a sequence's pages are junk), cu_seqlens, ctx_len"""
    g = torch.Generator().manual_seed(seed)
    needed = [-(-max(c, 0) // page) for c in ctx]
    n_pages = sum(needed) + extra
    order = torch.randperm(n_pages, generator=g)
    width = max(max(needed), 1) + spare
    table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(ctx), width), generator=g).to(torch.int32)
    shape = (n_pages, nkv, page, d) if layout == "heads" else (n_pages, page, nkv, d)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    valid, used = torch.zeros(n_pages, page, dtype=torch.bool), 0
    for b, n in enumerate(needed):
        table[b, :n] = order[used:used + n].to(torch.int32)
        for i in range(n):
            valid[order[used + i], :min(page, ctx[b] - i * page)] = True
        used += n
    for x in (k, v):
        x[~valid] = stale
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return k, v, table, cu


def _device(x):
    """on the GPU, with its strides"""
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=DEV).copy_(x)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check(name, out, q, k, v, table, cu, ctx, causal, scale):
    """Within the bound; infinities and NaN where the definition has them."""
    ref, bound, owned = oracle.attention(q, k, v, table, cu, ctx, causal, scale)
    ref, bound, got = ref[owned], bound[owned], out.cpu().double()[owned]
    finite = torch.isfinite(ref) & torch.isfinite(bound)
    diff = (got - ref).abs()[finite]
    print(f"{name}: max error / bound {float((diff / bound[finite].clamp_min(1e-300)).max()) if diff.numel() else 0:.2f}", flush=True)
    assert bool((diff <= bound[finite]).all()), f"{name}: over the bound by {float((diff - bound[finite]).max()):.3e}"
    assert bool(torch.isnan(got[torch.isnan(ref)]).all()) and torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])


ATTENTION = [
    # new tokens, keys with them, q heads, kv heads, d, page
    ([1], [1], 4, 2, 64, 16),
    ([1], [200], 32, 8, 128, 16),
    ([1, 1, 1], [17, 1000, 33], 8, 2, 128, 64),
    ([1] * 7, [5, 64, 65, 128, 129, 300, 16], 3, 1, 96, 48),
    ([1, 0, 1, 2], [40, 0, 16, 700], 4, 4, 32, 32),
    ([3, 5, 1, 4], [3, 100, 31, 260], 16, 4, 64, 16),            # drafts: up to 16 rows and just over
    ([4, 5], [513, 514], 16, 4, 128, 16),
    ([1, 1], [130, 3], 32, 1, 64, 128),                          # more rows a token than the small kernel's blocks
    ([70], [70], 4, 4, 64, 16),                                  # a prompt from its start
    ([129], [200], 8, 2, 128, 16),
    ([257, 1, 40], [300, 77, 41], 2, 2, 32, 64),
    ([65, 64, 63], [65, 1024, 700], 4, 1, 96, 32),
    ([300], [2000], 3, 1, 128, 256),
    ([33, 1, 2, 90, 0, 17], [50, 900, 2, 90, 12, 400], 12, 3, 64, 48),
    ([20, 1], [7, 1], 4, 2, 64, 16),                             # fewer keys than tokens: rows without keys
    ([2, 30, 1], [0, 0, 0], 4, 2, 128, 16),                      # no keys at all
    ([1] * 70, [i % 90 + 1 for i in range(70)], 2, 1, 64, 16),   # more sequences than lanes
    ([1, 6] * 40, [37 * (i % 11) + 7 for i in range(80)], 4, 1, 32, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_attention(case, causal, dtype):
    new, ctx, nq, nkv, d, page = case
    print(f"case {case} {causal} {dtype}", flush=True)
    k, v, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=sum(ctx) + d, layout="heads" if d != 64 else "tokens")
    q = (1.5 * torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(d + nq))).to(dtype)
    args = (q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    out = ops.paged_attention(*args, causal=causal)
    torch.cuda.synchronize()
    _check("o", out, q, k, v, table, cu, ctx, causal, 1 / math.sqrt(d))
    # a bound of the lengths and a workspace do not change the result; neither does a second call
    ws = ops.paged_workspace(len(ctx), cu[-1], nq, nkv, d, DEV)
    bare = ws.clone()                                       # without tickets
    for kwargs in (dict(max_q_len=max(new)), dict(workspace=ws), dict(workspace=ws, max_q_len=max(new)), dict(workspace=bare)):
        assert torch.equal(out, ops.paged_attention(*args, causal=causal, **kwargs)), kwargs
    torch.cuda.synchronize()
    assert not hasattr(bare, "tickets") and int(ws.tickets.abs().sum()) == 0


@pytest.mark.parametrize("nq,nkv,d,page,n,length", [(8, 2, 128, 64, 1, 30000), (4, 4, 64, 16, 1, 20000), (8, 2, 128, 16, 100, 9000), (2, 1, 64, 128, 700, 5000)])
def test_long_caches_are_split(nq, nkv, d, page, n, length):
    """One long sequence among short ones; the splits are merged."""
    new, ctx = [1, n, 1], [3, length, 40]
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=length)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(7)).bfloat16()
    args = (q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    out = ops.paged_attention(*args)
    names = launched(lambda: ops.paged_attention(*args, max_q_len=n))
    assert any("merge" in x for x in names), names
    ws = ops.paged_workspace(3, cu[-1], nq, nkv, d, DEV)
    names = launched(lambda: ops.paged_attention(*args, max_q_len=n, workspace=ws))
    assert any("merge" in x for x in names) == (n > 1), names
    for _ in range(3):                                      # whoever is last
        assert torch.equal(out, ops.paged_attention(*args, max_q_len=n, workspace=ws))
    torch.cuda.synchronize()
    assert int(ws.tickets.abs().sum()) == 0
    # a few tokens of the long one, all of the others
    keep = [0, 1, n // 2 + 1, n, n + 1]
    for t in sorted(set(keep)):
        b = 0 if t == 0 else (2 if t == n + 1 else 1)
        i = t - cu[b]
        ref, bound, _ = oracle.attention(q[t:t + 1], k, v, table[b:b + 1], [0, 1], [ctx[b] - (new[b] - 1 - i)], True, 1 / math.sqrt(d))
        diff = (out[t:t + 1].cpu().double() - ref).abs()
        assert bool((diff <= bound).all()), (t, float((diff / bound).max()))


def test_strides_padding_and_rows_left_alone():
    new, ctx, nq, nkv, d, page = [1, 40, 3], [90, 64, 33], 8, 2, 64, 32
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=1, layout="tokens")
    total = cu[-1] + 5                                      # tokens behind the last sequence
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(total, (nq + 2 * nkv) * d, generator=g).bfloat16()
    fused[cu[-1]:] = math.nan
    q = fused[:, :nq * d].view(total, nq, d)
    qd = fused.to(DEV)[:, :nq * d].view(total, nq, d)
    wide = torch.full((total, nq, 2 * d), 7.0, dtype=torch.bfloat16, device=DEV)
    out = wide[..., d:]
    args = (qd, _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    got = ops.paged_attention(*args, out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    _check("o", out, q, k, v, table, cu, ctx, True, 1 / math.sqrt(d))
    assert bool((wide[..., :d] == 7.0).all()) and bool((out[cu[-1]:] == 7.0).all())
    plain = ops.paged_attention(qd.contiguous(), *args[1:])
    assert torch.equal(plain[:cu[-1]], out[:cu[-1]])
    # another layout of the pages, a wider table and a scale of one's own
    other = ops.paged_attention(qd, _device(k).transpose(1, 2).contiguous().transpose(1, 2), _device(v).transpose(1, 2).contiguous().transpose(1, 2),
                                torch.cat((table, table), 1).to(DEV)[:, :table.shape[1]], *args[4:], softmax_scale=1 / math.sqrt(d))
    assert torch.equal(other[:cu[-1]], out[:cu[-1]])
    twice = ops.paged_attention(*args, softmax_scale=0.4)
    _check("scale", twice, q, k, v, table, cu, ctx, True, 0.4)


def test_shared_pages():
    """Two sequences whose first pages are the same (a shared prompt)."""
    new, ctx, nq, nkv, d, page = [1, 20], [100, 130], 8, 2, 128, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.float16, seed=3)
    table[0, :5] = table[1, :5]
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).half()
    out = ops.paged_attention(q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    _check("o", out, q, k, v, table, cu, ctx, True, 1 / math.sqrt(d))


def test_non_finite_values_behind_the_mask():
    """Keys that a row must not see do not reach it, whatever they hold; rows that see them get what arithmetic gives."""
    for new, ctx, nq, nkv in (([3], [40], 4, 1), ([100], [150], 4, 2)):
        d, page = 64, 16
        k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.float16, seed=4)
        q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).half()
        rest = (table.to(DEV), _ints(cu), _ints(ctx))
        clean = ops.paged_attention(q.to(DEV), _device(k), _device(v), *rest)
        at = ctx[0] - 2                                      # the key of the last but one new token
        for value in (math.nan, math.inf, -math.inf):
            for which in range(2):
                pages = [k.clone(), v.clone()]
                pages[which][int(table[0, at // page]), at % page, 0, 3] = value
                out = ops.paged_attention(q.to(DEV), _device(pages[0]), _device(pages[1]), *rest)
                torch.cuda.synchronize()
                _check(f"{value} {which}", out, q, *pages, table, cu, ctx, True, 1 / math.sqrt(d))
                heads = nq // nkv
                assert torch.equal(out[:, heads:], clean[:, heads:])      # the other KV heads
        q2 = q.clone()
        q2[1, 0] = math.nan                                  # a row of its own
        out = ops.paged_attention(q2.to(DEV), _device(k), _device(v), *rest)
        keep = torch.ones(cu[-1], nq, dtype=torch.bool)
        keep[1, 0] = False
        assert torch.equal(out.cpu()[keep], clean.cpu()[keep]) and bool(torch.isnan(out[1, 0]).all())


def test_extreme_scores():
    """Scores of the type's range: the maximum is subtracted before anything overflows."""
    new, ctx, nq, nkv, d, page = [1, 40], [300, 80], 4, 2, 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=6, stale=3.0)
    k = k * 300
    q = (300 * torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2))).bfloat16()
    out = ops.paged_attention(q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    assert bool(torch.isfinite(out).all())
    # differences of scores beside which 2 (d + 8) 2^-24 of their size is not small: rows where one key leads by far
    ref, _, _ = oracle.attention(q, k, v, table, cu, ctx, True, 1 / math.sqrt(d))
    p_diff = (out.cpu().double() - ref).abs()
    assert float(p_diff.median()) < 0.01


def test_lengths_and_pages_outside_the_cache():
    """Lengths beyond the page table count its room; pages outside the cache read the nearest inside; negative lengths are none."""
    new, nq, nkv, d, page = [1, 1, 30, 1], 8, 2, 64, 16
    ctx = [40, 25, 50, 20]
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=8, stale=1.0, spare=0)
    table[0, 1], table[2, 0] = -7, 2 ** 31 - 1
    said = [10 ** 9, 25, 50, -3]
    table[0, 2:] = torch.arange(table.shape[1] - 2, dtype=torch.int32)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = ops.paged_attention(q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(said))
    torch.cuda.synchronize()
    _check("o", out, q, k, v, table, cu, said, True, 1 / math.sqrt(d))


APPEND = [
    # new tokens, keys with them, q heads, kv heads, d, page, rotated, interleaved, norm, layer norm
    ([1], [1], 4, 2, 64, 16, 64, False, True, False),
    ([1, 1, 1], [17, 100, 33], 8, 2, 128, 64, 128, True, True, True),
    ([5, 0, 1, 33], [5, 3, 70, 48], 4, 4, 96, 48, 96, False, True, False),
    ([20, 7], [32, 64], 6, 3, 64, 16, 32, False, False, False),
    ([3, 2], [3, 2], 2, 1, 32, 32, 0, False, True, True),
    ([1, 2], [9, 2], 2, 1, 40, 16, 0, False, False, False),       # any head
    ([4, 2], [9, 50], 2, 1, 64, 16, 20, False, True, False),      # halves that are not whole vectors
    ([1] * 40, [i + 1 for i in range(40)], 4, 2, 128, 16, 128, False, True, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("with_q", [True, False], ids=["q", "no-q"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[4]}-{c[5]}-{c[6]}")
def test_append(case, with_q, dtype):
    new, ctx, nq, nkv, d, page, r, interleaved, norm, layer_norm = case
    print(f"case {case} {with_q} {dtype}", flush=True)
    k_pages, v_pages, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=d, layout="heads" if d == 64 else "tokens", stale=2.0)
    total = cu[-1] + 3
    g = torch.Generator().manual_seed(11)
    fused = torch.randn(total, (nq + 2 * nkv) * d, generator=g).to(dtype)

    def parts(x):
        return (x[:, :nq * d].view(total, nq, d), x[:, nq * d:(nq + nkv) * d].view(total, nkv, d), x[:, (nq + nkv) * d:].view(total, nkv, d))
    q, k, v = parts(fused)
    qd, kd, vd = parts(fused.to(DEV))
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)] + [(0.2 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    ids = torch.randint(0, 64, (total,), generator=g)
    kwargs, rotate = {}, oracle.no_rotation
    if r:
        cos, sin = _tables(64, r, dtype, interleaved)
        rotate = oracle.rotation(cos, sin, ids, d, interleaved)
        kwargs = dict(rotary=(cos.to(DEV), sin.to(DEV), ids.to(DEV)), interleaved=interleaved)
    if norm:
        kwargs.update(k_weight=w[1].to(DEV), layer_norm=layer_norm)
        if layer_norm:
            kwargs.update(k_bias=w[3].to(DEV))
        if with_q:
            kwargs.update(q_weight=w[0].to(DEV))
            if layer_norm:
                kwargs.update(q_bias=w[2].to(DEV))
    kp, vp = _device(k_pages), _device(v_pages)
    out = ops.paged_append(kd, vd, kp, vp, table.to(DEV), _ints(cu), _ints(ctx), q=qd if with_q else None, **kwargs)
    torch.cuda.synchronize()

    def of(x, i):
        if norm:
            return oracle.norm_rotary(x, w[i], w[i + 2] if layer_norm else None, 1e-5, layer_norm, rotate)
        return rotate(x.double()), rotate(x.double().abs(), magnitude=True)
    if with_q:
        _close("q", out, *of(q, 0))
    else:
        assert out is None
    ref, size = of(k, 1)
    written = torch.zeros(k_pages.shape[:2], dtype=torch.bool)
    where = oracle.slots(table, cu, ctx, page, k_pages.shape[0], total)
    stored = [t for t in range(total) if where[t] is not None]
    assert stored == list(range(cu[-1]))
    rows = torch.stack([kp[where[t]].cpu() for t in stored])
    _close("k", rows, ref[stored], size[stored])
    for t in stored:
        written[where[t]] = True
        assert torch.equal(vp[where[t]].cpu(), v[t])
    assert torch.equal(kp.cpu()[~written], k_pages[~written]) and torch.equal(vp.cpu()[~written], v_pages[~written])


def test_append_without_a_place_is_dropped():
    new, ctx, nq, nkv, d, page = [3, 2, 4, 2], [5, 64, 2, 40], 4, 2, 64, 16
    k_pages, v_pages, table, cu = _cache(new, [5, 48, 4, 40], nkv, d, page, torch.bfloat16, seed=5, stale=2.0, spare=0)
    n_pages = k_pages.shape[0]
    table[3, 2] = n_pages                                    # a page outside the cache (keys 32 on), a negative one
    table[0, 0] = -1
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(cu[-1] + 2, nkv, d, generator=g).bfloat16() for _ in range(2))
    kp, vp = _device(k_pages), _device(v_pages)
    ops.paged_append(k.to(DEV), v.to(DEV), kp, vp, table.to(DEV), _ints(cu), _ints(ctx))
    torch.cuda.synchronize()
    where = oracle.slots(table, cu, ctx, page, n_pages, cu[-1] + 2)
    assert [w is not None for w in where] == [False] * 5 + [False, False, True, True] + [False] * 4     # 64 keys: past the table of 48; 2 keys of 4 tokens
    want_k, want_v = k_pages.clone(), v_pages.clone()
    for t, w in enumerate(where):
        if w is not None:
            want_k[w], want_v[w] = k[t], v[t]
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)


def test_append_then_attend_as_a_server_does():
    """Prompts in chunks, then single tokens, of sequences of different lengths: every output against attention over everything so far."""
    nq, nkv, d, page, dtype = 8, 2, 64, 16, torch.bfloat16
    lens = [37, 5, 80]
    chunks = [[20, 5, 33], [17, 0, 47], [1, 1, 1], [1, 1, 1]]
    g = torch.Generator().manual_seed(3)
    total = [n + 2 for n in lens]
    q, k, v = ([torch.randn(n, h, d, generator=g).to(dtype) for n in total] for h in (nq, nkv, nkv))
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    cos, sin = _tables(128, d, dtype, False)
    width = -(-max(total) // page)
    n_pages = 3 * width
    table = torch.randperm(n_pages, generator=g).to(torch.int32).view(3, width)
    kp, vp = (torch.full((n_pages, nkv, page, d), math.nan, dtype=dtype, device=DEV).transpose(1, 2) for _ in range(2))
    ctx_len, ws = torch.zeros(3, dtype=torch.int32, device=DEV), ops.paged_workspace(3, 128, nq, nkv, d, DEV)
    done = [0, 0, 0]
    for new in chunks:
        ids = torch.cat([torch.arange(a, a + n) for a, n in zip(done, new)])
        cu = [0, new[0], new[0] + new[1], sum(new)]
        pick = lambda x: torch.cat([t[a:a + n] for t, a, n in zip(x, done, new)]).to(DEV)     # noqa: E731
        ctx_len += _ints(new)
        rot_q = ops.paged_append(pick(k), pick(v), kp, vp, table.to(DEV), _ints(cu), ctx_len, q=pick(q), q_weight=w[0].to(DEV), k_weight=w[1].to(DEV),
                                 rotary=(cos.to(DEV), sin.to(DEV), ids.to(DEV)))
        out = ops.paged_attention(rot_q, kp, vp, table.to(DEV), _ints(cu), ctx_len, max_q_len=max(new), workspace=ws)
        done = [a + n for a, n in zip(done, new)]
        _check("step", out, rot_q.cpu(), kp.cpu(), vp.cpu(), table, cu, done, True, 1 / math.sqrt(d))
    # what the cache holds is what norm_rotary gives
    for b in range(3):
        ids = torch.arange(total[b]).to(DEV)
        want = ops.norm_rotary(q[b].to(DEV), k[b].to(DEV), w[0].to(DEV), w[1].to(DEV), rotary=(cos.to(DEV), sin.to(DEV), ids))[1]
        got = kp[table[b].long().to(DEV)].flatten(0, 1)[:total[b]]
        assert torch.equal(got, want)
        assert torch.equal(vp[table[b].long().to(DEV)].flatten(0, 1)[:total[b]].cpu(), v[b])


def test_streams_and_graphs():
    """A captured step replayed with other lengths, two graphs with workspaces of their own at once, and another stream."""
    nq, nkv, d, page = 8, 2, 128, 16
    new, ctx = [1, 1, 30], [300, 4000, 64]
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=12, stale=1.0)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    args = [q, _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx)]
    want = ops.paged_attention(*args)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        ws, out = ops.paged_workspace(3, cu[-1], nq, nkv, d, DEV), torch.zeros_like(want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.paged_attention(*args, workspace=ws)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(*args, workspace=ws, out=out)
        graphs.append((graph, ws))
        outs.append(out)
    for lens in (ctx, [5, 17, 40], [1, 4000, 30], ctx):
        args[5].copy_(_ints(lens))
        for out in outs:
            out.zero_()
        want = ops.paged_attention(*args)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, (side, other)):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs), lens


def test_offsets_past_32_bits():
    """Pages more than 2^32 bytes (and 2^31 elements) into the cache."""
    nq, nkv, d, page = 4, 2, 128, 64
    n_pages = 2 ** 32 // (page * nkv * d) + 40                # 8 GiB of bfloat16 each
    pool_k, pool_v = (torch.zeros(n_pages, nkv, page, d, dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2))
    g = torch.Generator().manual_seed(5)
    new, ctx = [90, 1], [90, 1]
    table = torch.tensor([[n_pages - 1, n_pages // 2 + 3], [n_pages - 20, 0]], dtype=torch.int32)
    k, v = (torch.randn(91, nkv, d, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(91, nq, d, generator=g).bfloat16()
    cu = [0, 90, 91]
    ops.paged_append(k.to(DEV), v.to(DEV), pool_k, pool_v, table.to(DEV), _ints(cu), _ints(ctx))
    out = ops.paged_attention(q.to(DEV), pool_k, pool_v, table.to(DEV), _ints(cu), _ints(ctx))
    torch.cuda.synchronize()
    small = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    near_k, near_v = (x[table.flatten().long().to(DEV)].cpu() for x in (pool_k, pool_v))
    assert torch.equal(near_k[0], k[:64]) and torch.equal(near_k[1, :26], k[64:90]) and torch.equal(near_v[2, 0], v[90])
    _check("o", out, q, near_k, near_v, small, cu, ctx, True, 1 / math.sqrt(d))


def test_refusals():
    new, ctx, nq, nkv, d, page = [2, 1], [20, 9], 4, 2, 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=1, stale=1.0)
    q = torch.randn(3, nq, d).bfloat16().to(DEV)
    good = dict(k_pages=_device(k), v_pages=_device(v), page_table=table.to(DEV), cu_seqlens=_ints(cu), ctx_len=_ints(ctx))
    rows = dict(k=torch.randn(3, nkv, d).bfloat16().to(DEV), v=torch.randn(3, nkv, d).bfloat16().to(DEV))
    for change in [
        dict(k_pages=_device(k).half()), dict(v_pages=_device(v)[:-1]), dict(v_pages=_device(v).contiguous() if not v.is_contiguous() else _device(v.transpose(1, 2).contiguous().transpose(1, 2))),
        dict(page_table=table.to(DEV).long()), dict(page_table=table.to(DEV)[:1]), dict(page_table=table.to(DEV)[0]), dict(page_table=table),
        dict(cu_seqlens=_ints(cu)[:-1]), dict(cu_seqlens=_ints(cu).long()), dict(ctx_len=_ints(ctx).long()), dict(ctx_len=_ints(ctx).cpu()),
        dict(page_table=table.to(DEV)[:, :0]),
        dict(k_pages=_device(k)[:, :8], v_pages=_device(v)[:, :8]),                     # pages of 8 and of 20 keys
        dict(k_pages=torch.zeros(4, 20, nkv, d, dtype=torch.bfloat16, device=DEV), v_pages=torch.zeros(4, 20, nkv, d, dtype=torch.bfloat16, device=DEV)),
    ]:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.paged_attention(q, **{**good, **change})
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.paged_append(**rows, **{**good, **change})
    for bad in [dict(q=q.float()), dict(q=q.cpu()), dict(q=torch.randn(3, 3, d).bfloat16().to(DEV)), dict(q=torch.randn(3, nq, 80).bfloat16().to(DEV)),
                dict(q=q, out=torch.empty(2, nq, d, dtype=torch.bfloat16, device=DEV)), dict(q=q, out=torch.empty(3, nq, d, device=DEV)),
                dict(q=q, softmax_scale=0.0), dict(q=q, softmax_scale=-1.0), dict(q=q, max_q_len=0),
                dict(q=q, workspace=torch.empty(8, device=DEV)), dict(q=q, workspace=torch.empty(8)),
                dict(q=torch.randn(3, nq, d + 1).bfloat16().to(DEV)[..., 1:])]:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.paged_attention(**{**good, **bad})
    w = torch.ones(d, dtype=torch.bfloat16, device=DEV)
    for bad in [dict(v=rows["v"][:2]), dict(v=rows["v"].half()), dict(k=rows["k"].float(), v=rows["v"].float()), dict(q=q, q_weight=w), dict(q=q, k_weight=w),
                dict(q_weight=w, k_weight=w), dict(k_weight=w, k_bias=w), dict(q=q[:2]), dict(k_weight=w[:32])]:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.paged_append(**{**rows, **good, **bad})
    # no tokens: nothing happens
    before = good["k_pages"].clone()
    assert ops.paged_attention(q[:0], good["k_pages"], good["v_pages"], good["page_table"], _ints([0, 0, 0]), good["ctx_len"]).shape == (0, nq, d)
    assert ops.paged_append(rows["k"][:0], rows["v"][:0], good["k_pages"], good["v_pages"], good["page_table"], _ints([0, 0, 0]), good["ctx_len"], q=q[:0]).shape == (0, nq, d)
    torch.cuda.synchronize()
    assert torch.equal(good["k_pages"], before)


@pytest.mark.parametrize("new,ctx", [([6], [300]), ([8], [3000]), ([9, 2], [500, 40]), ([5, 1] * 9, [40 * i + 6 for i in range(18)])], ids=["block", "splits", "blocks", "many"])
def test_non_finite_values_behind_the_mask_of_drafts(new, ctx):
    """Blocks of 32 rows: keys that a row must not see do not reach it, in either half of the block."""
    nq, nkv, d, page = 8, 2, 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=9)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    at = ctx[0] - 2
    for value in (math.nan, math.inf, -math.inf):
        for which in range(2):
            pages = [k.clone(), v.clone()]
            pages[which][int(table[0, at // page]), at % page, 0, 3] = value
            out = ops.paged_attention(q.to(DEV), _device(pages[0]), _device(pages[1]), table.to(DEV), _ints(cu), _ints(ctx), max_q_len=max(new))
            torch.cuda.synchronize()
            _check(f"{value} {which}", out, q, *pages, table, cu, ctx, True, 1 / math.sqrt(d))


def test_an_output_that_shares_memory_with_q_is_refused():
    new, ctx, nq, nkv, d, page = [2, 1], [20, 9], 4, 2, 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=1, stale=1.0)
    memory = torch.zeros(4, nq, d, dtype=torch.bfloat16, device=DEV)
    for q, out in ((memory[:3], memory[:3]), (memory[:3], memory[1:])):
        with pytest.raises(RuntimeError):
            ops.paged_attention(q, _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx), out=out)


@pytest.mark.parametrize("new,ctx,total,max_q_len", [
    ([3], [700], 200, 200),                                  # a buffer for a chunk with a few tokens in it
    ([100, 2, 64], [130, 900, 64], 300, 100),                # tokens for three chunks, one of them short
    ([1, 1, 1], [40, 300, 17], 64, 1),                       # a buffer of 64 for single tokens
    ([0, 90], [50, 90], 180, 90),
], ids=str)
def test_fewer_tokens_than_the_buffer_has(new, ctx, total, max_q_len):
    """Sequences shorter than the numbers of tokens and sequences let one expect; rows behind the last one stay as they are."""
    nq, nkv, d, page = 8, 2, 128, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=12)
    q = torch.randn(total, nq, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = torch.full_like(q, 7.0, device=DEV)
    ops.paged_attention(q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx), max_q_len=max_q_len, out=out)
    torch.cuda.synchronize()
    _check("o", out, q, k, v, table, cu, ctx, True, 1 / math.sqrt(d))
    assert bool((out[cu[-1]:] == 7.0).all())


# Page tables with room for more than 512 keys, whatever the lengths: sequences of many rows are computed as chunks.
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_attention_over_wide_page_tables(case, causal):
    new, ctx, nq, nkv, d, page = case
    dtype = torch.bfloat16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=sum(ctx) + d + 1, layout="heads" if d != 64 else "tokens", spare=640 // page)
    q = (1.5 * torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(d + nq))).to(dtype)
    args = (q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    out = ops.paged_attention(*args, causal=causal)
    torch.cuda.synchronize()
    _check("o", out, q, k, v, table, cu, ctx, causal, 1 / math.sqrt(d))


@pytest.mark.parametrize("new,ctx,nq,nkv", [([100], [150], 4, 2), ([100], [700], 4, 1), ([65, 3], [700, 40], 8, 2)], ids=["tile", "splits", "mixed"])
def test_non_finite_values_behind_the_mask_of_chunks(new, ctx, nq, nkv):
    """As for short page tables: keys that a row must not see do not reach it."""
    d, page = 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.float16, seed=4, spare=40)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).half()
    rest = (table.to(DEV), _ints(cu), _ints(ctx))
    clean = ops.paged_attention(q.to(DEV), _device(k), _device(v), *rest)
    at = ctx[0] - 2
    for value in (math.nan, math.inf, -math.inf):
        for which in range(2):
            pages = [k.clone(), v.clone()]
            pages[which][int(table[0, at // page]), at % page, 0, 3] = value
            out = ops.paged_attention(q.to(DEV), _device(pages[0]), _device(pages[1]), *rest)
            torch.cuda.synchronize()
            _check(f"{value} {which}", out, q, *pages, table, cu, ctx, True, 1 / math.sqrt(d))
            heads = nq // nkv
            assert torch.equal(out[:, heads:], clean[:, heads:])


def test_which_launches_a_call_makes():
    """Short page tables: blocks of few rows alone; wide ones: chunks beside them; chunks only: nothing else; short sequences: no merge."""
    nq, nkv, d, page = 8, 2, 128, 16

    def names(new, ctx, spare, **kwargs):
        k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=2, spare=spare)
        q = torch.randn(cu[-1], nq, d).bfloat16().to(DEV)
        args = (q, _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
        return [n for n in ("paged_rows", "paged_tiles", "paged_merge") for m in launched(lambda: ops.paged_attention(*args, **kwargs)) if n in m]
    assert names([100, 1], [300, 40], 1) == ["paged_rows"]
    assert names([100, 1], [300, 40], 40) == ["paged_rows", "paged_tiles", "paged_merge"]
    assert names([100, 80], [700, 600], 1, max_q_len=100) == ["paged_tiles", "paged_merge"]
    assert names([1, 1], [300, 200], 0, max_q_len=1) == ["paged_rows"]


def test_an_output_between_the_rows_of_q():
    """Slices of one tensor: an output that shares elements with q is refused however it is strided, one beside it is not."""
    new, ctx, nq, nkv, d, page = [40, 1], [90, 30], 4, 2, 64, 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, torch.bfloat16, seed=21, stale=1.0)
    q = torch.randn(41, nq, d, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    rest = (_device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    want = ops.paged_attention(q, *rest)
    one = torch.zeros(42, 3 * nq * d, dtype=torch.bfloat16, device=DEV)                          # a projection's output: q, then others
    part = lambda i, rows=slice(0, 41): one[rows, i * nq * d:(i + 1) * nq * d].view(41, nq, d)     # noqa: E731
    per_head = torch.zeros(41, nq, 3, d, dtype=torch.bfloat16, device=DEV)                       # per head q, then others
    outermost = torch.zeros(nq, 2 * 41, d, dtype=torch.bfloat16, device=DEV).transpose(0, 1)     # heads outermost
    for a, b in ((part(0), part(0)), (part(0), part(0, slice(1, 42))), (part(0), one[:41, d:(nq + 1) * d].view(41, nq, d)), (per_head[:, :, 1], per_head[:, :, 1]),
                 (outermost[:41], outermost[1:42]), (one[:41, :nq * d].view(41, nq, d), one.view(-1)[:41 * nq * d].view(41, nq, d))):
        a.copy_(q)
        with pytest.raises(RuntimeError, match="memory"):
            ops.paged_attention(a, *rest, out=b)
    for a, b in ((part(0), part(1)), (part(2), part(0)), (part(0, slice(1, 42)), part(1)), (per_head[:, :, 0], per_head[:, :, 2]), (per_head[:, :, 2], per_head[:, :, 1]),
                 (outermost[:41], outermost[41:])):
        a.copy_(q)
        assert torch.equal(ops.paged_attention(a, *rest, out=b), want) and torch.equal(b, want) and torch.equal(a, q)
    with pytest.raises(RuntimeError):                        # rows of an output that are one
        ops.paged_attention(q, *rest, out=one[:1, :nq * d].view(1, nq, d).expand(41, nq, d))

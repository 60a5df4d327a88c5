"""Attention of sequences that share a prefix in groups, against float64."""

import math

import pytest
import torch

from scaling_amd import ops
from tests import prefix_oracle as oracle
from tests.kernels import launched
from tests.test_gpu_paged import _cache, _device, _ints

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


class _Call:
    """Own pages of every sequence and pages of every prefix in one pool; what no key is holds `stale`."""

    def __init__(self, new, ctx, sizes, prefix, nq, nkv, d, page, dtype, seed, layout="heads", stale=math.nan, first=0):
        self.new, self.ctx, self.prefix = new, ctx, prefix
        self.k, self.v, table, _ = _cache(new + [0] * len(prefix), ctx + prefix, nkv, d, page, dtype, seed, layout=layout, stale=stale)
        self.table, self.prefix_table = table[:len(new)], table[len(new):]
        self.cu, self.groups = [0], [first]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        for n in sizes:
            self.groups.append(self.groups[-1] + n)
        self.q = (1.5 * torch.randn(self.cu[-1], nq, d, generator=torch.Generator().manual_seed(seed + 1))).to(dtype)
        self.scale = 1 / math.sqrt(d)

    def arguments(self):
        return (self.q.to(DEV), _device(self.k), _device(self.v), self.table.to(DEV), _ints(self.cu), _ints(self.ctx), self.prefix_table.to(DEV), _ints(self.prefix),
                _ints(self.groups))

    def check(self, name, out, causal=True):
        ref, bound, owned = oracle.attention(self.q, self.k, self.v, self.table, self.cu, self.ctx, self.prefix_table, self.prefix, self.groups, causal, self.scale)
        ref, bound, got = ref[owned], bound[owned], out.cpu().double()[owned]
        finite = torch.isfinite(ref) & torch.isfinite(bound)
        diff = (got - ref).abs()[finite]
        print(f"{name}: max error / bound {float((diff / bound[finite].clamp_min(1e-300)).max()) if diff.numel() else 0:.2f}", flush=True)
        assert bool((diff <= bound[finite]).all()), f"{name}: over the bound by {float((diff - bound[finite]).max()):.3e}"
        assert bool(torch.isnan(got[torch.isnan(ref)]).all()) and torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])


CASES = [
    # new tokens, own keys with them, sizes of groups, prefixes, q heads, kv heads, d, page
    ([1], [1], [1], [1], 4, 2, 64, 16),
    ([1, 1], [1, 40], [2], [33], 32, 8, 128, 16),
    ([1] * 3, [5, 17, 300], [3], [1000], 8, 2, 128, 64),
    ([1] * 8, [3, 20, 100, 65, 1, 16, 33, 48], [8], [1500], 32, 8, 128, 16),
    ([1] * 9, [9] * 9, [4, 5], [700, 90], 16, 4, 64, 32),
    ([1] * 7, [5, 64, 65, 128, 129, 300, 16], [2, 0, 3, 2], [40, 77, 129, 0], 3, 1, 96, 48),
    ([1] * 70, [i % 50 + 1 for i in range(70)], [70], [260], 4, 1, 64, 16),
    ([1] * 70, [i % 50 + 1 for i in range(70)], [1] * 70, [(37 * i) % 90 for i in range(70)], 2, 1, 64, 16),
    ([3, 5, 1, 4], [3, 100, 31, 260], [4], [513], 16, 4, 64, 16),
    ([3, 0, 9, 1], [30, 12, 10, 4], [3, 1], [200, 1100], 32, 8, 128, 64),
    ([70], [70], [1], [300], 4, 4, 64, 16),
    ([129, 40, 1], [200, 40, 77], [3], [400], 8, 2, 128, 16),
    ([257, 1, 40], [300, 77, 41], [2, 1], [100, 900], 2, 2, 32, 64),
    ([33, 1, 2, 90, 0, 17], [50, 900, 2, 90, 12, 400], [2, 4], [300, 31], 12, 3, 64, 48),
    ([1, 1], [130, 3], [2], [2000], 32, 1, 64, 128),
    ([2, 3], [0, 1], [2], [20], 4, 2, 64, 16),                   # fewer own keys than tokens
    ([2, 3], [0, 1], [2], [0], 4, 2, 128, 16),                   # and no prefix: rows without keys
    ([20, 1], [20, 5], [1, 1], [0, 17], 20, 4, 96, 16),
]


@DTYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-{len(c[2])}x{max(c[3])}-{c[4]}-{c[5]}-{c[6]}-{c[7]}")
def test_attention(case, causal, dtype):
    new, ctx, sizes, prefix, nq, nkv, d, page = case
    print(f"case {case} {causal} {dtype}", flush=True)
    call = _Call(new, ctx, sizes, prefix, nq, nkv, d, page, dtype, seed=sum(ctx) + d, layout="heads" if d != 64 else "tokens")
    args = call.arguments()
    out = ops.paged_prefix_attention(*args, causal=causal)
    torch.cuda.synchronize()
    call.check("o", out, causal)
    ws = ops.paged_prefix_workspace(len(new), len(prefix), call.cu[-1], nq, nkv, d, DEV)
    ws.fill_(math.nan)
    assert torch.equal(out, ops.paged_prefix_attention(*args, causal=causal, workspace=ws))
    # a bound of the tokens of a sequence may cut the work otherwise
    for _ in range(2):
        call.check("o, bounded", ops.paged_prefix_attention(*args, causal=causal, workspace=ws, max_q_len=max(new)), causal)


@pytest.mark.parametrize("nq,nkv,d,page,batch,length", [(32, 8, 128, 64, 24, 9000), (16, 4, 64, 16, 2, 12000), (4, 4, 128, 32, 90, 5000)])
def test_long_prefixes_are_split(nq, nkv, d, page, batch, length):
    call = _Call([1] * batch, [7 * i % 100 + 1 for i in range(batch)], [batch], [length], nq, nkv, d, page, torch.bfloat16, seed=length)
    args = call.arguments()
    out = ops.paged_prefix_attention(*args, max_q_len=1)
    call.check("o", out)
    for _ in range(3):
        assert torch.equal(out, ops.paged_prefix_attention(*args, max_q_len=1))


@DTYPES
@pytest.mark.parametrize("nq,nkv,d,batch,groups,length,new", [(8, 2, 96, 30, 1, 700, 1), (8, 2, 32, 30, 1, 700, 1), (4, 1, 128, 62, 2, 500, 1), (8, 1, 128, 63, 2, 300, 1), (4, 2, 64, 64, 1, 400, 1),
                                                              (8, 2, 64, 300, 3, 200, 1), (4, 1, 32, 300, 2, 90, 3), (8, 1, 96, 20, 1, 1000, 2), (4, 1, 128, 40, 1, 2000, 5),
                                                              (128, 128, 32, 30, 1, 13000, 1), (128, 128, 32, 66, 1, 13000, 1), (128, 128, 96, 66, 1, 6500, 1), (128, 128, 32, 20, 1, 13000, 17)])
def test_groups_of_many_rows(nq, nkv, d, batch, groups, length, new, dtype):
    """Prefixes and own keys in one launch, by every head size, by the number of sequences that its workgroups look for their work among, and with
    more tiles of a prefix to a workgroup than it looks up pages for at once."""
    print(f"case {nq} {nkv} {d} {batch} {groups} {length} {new} {dtype}", flush=True)
    sizes = [batch // groups] * groups
    sizes[0] += batch - sum(sizes)
    counts = [1 + i % new for i in range(batch)]
    call = _Call(counts, [n + 13 * i % 70 for i, n in enumerate(counts)], sizes, [length + 37 * g for g in range(groups)], nq, nkv, d, 16, dtype, seed=length + d)
    args = call.arguments()
    names = launched(lambda: ops.paged_prefix_attention(*args, max_q_len=new))
    assert len(names) == 2 and any("paged_prefix_kernel" in n for n in names) == (sum(counts) * nq // nkv > 64), names       # all rows together are few
    out = ops.paged_prefix_attention(*args, max_q_len=new)
    call.check("o", out)
    for _ in range(3):
        assert torch.equal(out, ops.paged_prefix_attention(*args, max_q_len=new))
    call.check("o, tokens not bounded", ops.paged_prefix_attention(*args))


def test_more_blocks_than_compute_units():
    """So many rows that nothing is cut into pieces, of more sequences than a workgroup's wavefronts look at together."""
    call = _Call([3] * 700, [3 + i % 20 for i in range(700)], [300, 400], [100, 33], 32, 32, 32, 16, torch.bfloat16, seed=21)
    args = call.arguments()
    names = launched(lambda: ops.paged_prefix_attention(*args, max_q_len=3))
    assert any("paged_tiles" in n for n in names), names
    call.check("o", ops.paged_prefix_attention(*args, max_q_len=3))


def test_no_prefix_is_paged_attention():
    """Groups of empty prefixes, and sequences outside all groups."""
    call = _Call([1, 3, 1, 1], [50, 3, 400, 1], [1, 1], [0, 0], 8, 2, 128, 16, torch.bfloat16, seed=3, first=1)
    args = call.arguments()
    out = ops.paged_prefix_attention(*args)
    call.check("o", out)
    plain = ops.paged_attention(*args[:6])
    assert float((out.float() - plain.float()).abs().max()) <= 2.0 ** -8 * float(plain.float().abs().max()) * 2
    call = _Call([1, 3, 1, 1], [50, 3, 400, 1], [2], [70], 8, 2, 128, 16, torch.float16, seed=4, first=1)
    call.check("sequences in front and behind", ops.paged_prefix_attention(*call.arguments()))


@pytest.mark.parametrize("new,sizes,nq,nkv,d,prefix", [([20] + [1] * 7, [8], 8, 2, 64, [200]), ([1, 1, 40, 1, 33, 1, 1, 90], [4, 3], 32, 8, 128, [700, 30]), ([300] + [1] * 60, [30, 31], 4, 1, 96, [90, 500]),
                                                        ([9, 1, 1], [3], 4, 2, 32, [300]), ([64, 1] * 150, [150, 150], 32, 32, 32, [60, 20])])
def test_a_bound_that_is_too_low(new, sizes, nq, nkv, d, prefix):
    """Sequences of more tokens than max_q_len are computed all the same, and so is everybody else; nothing is left of what an earlier call wrote to the workspace."""
    print(f"case {new[:8]} {sizes} {nq} {nkv} {d}", flush=True)
    call = _Call(new, [n + 11 * i % 300 for i, n in enumerate(new)], sizes, prefix, nq, nkv, d, 16, torch.bfloat16, seed=len(new) + d)
    args = call.arguments()
    ws = ops.paged_prefix_workspace(len(new), len(prefix), call.cu[-1], nq, nkv, d, DEV)
    for stale in (math.nan, 0.0, 1.0):
        ws.fill_(stale)
        for bound in (1, 2, max(new) - 1):
            call.check(f"o, bound {bound}", ops.paged_prefix_attention(*args, workspace=ws, max_q_len=bound))


@DTYPES
def test_values_that_are_not_finite(dtype):
    """Infinities and NaN reach the rows that see them and no others."""
    call = _Call([1, 1, 20], [30, 17, 60], [2, 1], [100, 40], 4, 2, 64, 16, dtype, seed=8, stale=math.inf)
    call.v[call.prefix_table[0, 2].item(), 5, 0] = math.inf
    call.v[call.table[1, 0].item(), 3, 1] = math.nan
    call.k[call.table[2, 3].item(), 8, 0] = math.nan             # key 56 of the third sequence: its last tokens see it
    call.check("o", ops.paged_prefix_attention(*call.arguments()))


def test_scores_of_minus_infinity_everywhere():
    """Prefix and own keys that all score -inf: zeros; either alone: the other's result."""
    call = _Call([1, 1], [20, 20], [2], [50], 2, 1, 64, 16, torch.bfloat16, seed=9)
    call.q.fill_(1.0)
    minus = torch.full_like(call.k, -math.inf)
    args = list(call.arguments())
    args[1] = _device(minus)
    assert float(ops.paged_prefix_attention(*args).abs().max()) == 0.0
    k = call.k.clone()
    k[call.prefix_table[0, :4].long()] = -math.inf
    args[1] = _device(k)
    alone = ops.paged_attention(args[0], args[1], *args[2:6])
    assert float((ops.paged_prefix_attention(*args).float() - alone.float()).abs().max()) <= 2.0 ** -7 * float(alone.float().abs().max())


def test_rows_behind_and_strides():
    """Rows behind the last sequence and memory between the rows of `out` stay; q and out may be slices."""
    call = _Call([1, 4, 1], [8, 40, 3], [3], [100], 4, 2, 64, 16, torch.bfloat16, seed=10)
    args = list(call.arguments())
    want = ops.paged_prefix_attention(*args)
    whole = torch.full((9, 6, 80), 7.0, dtype=torch.bfloat16, device=DEV)
    q = torch.full((9, 5, 72), math.nan, dtype=torch.bfloat16, device=DEV)
    q[:6, :4, :64] = args[0]
    out = ops.paged_prefix_attention(q[:, :4, :64], *args[1:], out=whole[:, 1:5, 8:72])
    assert torch.equal(out[:6], want) and out.data_ptr() == whole[:, 1:5, 8:72].data_ptr()
    whole[:6, 1:5, 8:72] = 7.0
    assert bool((whole == 7.0).all())


def test_numbers_from_nowhere():
    """Lengths, pages and groups outside their ranges read nothing outside the cache and write nothing outside the rows."""
    call = _Call([1, 2, 1], [30, 20, 9], [3], [64], 4, 2, 64, 16, torch.bfloat16, seed=11, stale=0.0)
    args = list(call.arguments())
    for at, value in ((3, torch.full_like(args[3], 2 ** 30)), (3, torch.full_like(args[3], -5)), (5, _ints([2 ** 31 - 1, -3, 9])), (6, torch.full_like(args[6], -1)),
                      (7, _ints([2 ** 31 - 1])), (7, _ints([-1])), (8, _ints([-4, 100])), (8, _ints([3, 1])), (4, _ints([0, 2, 1, 900])), (4, _ints([4, 4, 4, 4])),
                      (4, _ints([-9, 2, 3, 4]))):
        bad = list(args)
        bad[at] = value
        guard = torch.full((12, 4, 64), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.paged_prefix_attention(*bad, out=guard[4:8])
        torch.cuda.synchronize()
        assert bool((guard[:4] == 3.0).all()) and bool((guard[8:] == 3.0).all()), (at, value)


def test_launches_streams_and_replays():
    call = _Call([1] * 8, [20] * 8, [8], [700], 8, 2, 128, 16, torch.bfloat16, seed=12)
    args = list(call.arguments())
    ws = ops.paged_prefix_workspace(8, 1, 8, 8, 2, 128, DEV)
    want = ops.paged_prefix_attention(*args, max_q_len=1, workspace=ws)
    names = launched(lambda: ops.paged_prefix_attention(*args, max_q_len=1, workspace=ws))
    assert 1 <= len(names) <= 3, names
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.paged_prefix_attention(*args, max_q_len=1), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefix_attention(*args, max_q_len=1, workspace=ws)
    for ctx, prefix in (([1] * 8, 1), ([16, 17, 3, 30, 5, 2, 9, 31], 650), ([20] * 8, 0), ([20] * 8, 700)):
        args[5].copy_(_ints(ctx))
        args[7].copy_(_ints([prefix]))
        graph.replay()
        torch.cuda.synchronize()
        again = ops.paged_prefix_attention(*args, max_q_len=1)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16)), (ctx, prefix)        # as bits: lengths beyond the keys reach NaN
    assert torch.equal(out, want)


def test_replays_of_many_rows():
    """Prefixes and own keys in one launch: lengths change between replays, eager calls with a workspace of their own between them."""
    call = _Call([1] * 40, [60] * 40, [25, 15], [900, 500], 8, 2, 64, 16, torch.float16, seed=22)
    args = list(call.arguments())
    ws = ops.paged_prefix_workspace(40, 2, 40, 8, 2, 64, DEV)
    assert any("paged_prefix_kernel" in n for n in launched(lambda: ops.paged_prefix_attention(*args, max_q_len=1, workspace=ws)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefix_attention(*args, max_q_len=1, workspace=ws)
    for ctx, prefix, groups in (([1] * 40, [1, 0], [0, 25, 40]), ([i + 1 for i in range(40)], [899, 333], [0, 1, 40]), ([60] * 40, [0, 0], [3, 3, 40]), ([60] * 40, [900, 500], [0, 25, 40])):
        args[5].copy_(_ints(ctx))
        args[7].copy_(_ints(prefix))
        args[8].copy_(_ints(groups))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ops.paged_prefix_attention(*args, max_q_len=1).view(torch.int16)), (ctx, prefix, groups)
    call.check("o of the last replay", out)


@pytest.mark.parametrize("batch", [6, 80])
def test_one_prefix_of_two_groups(batch):
    """Groups that name the same pages, one of them for fewer keys, and a third without any key of a prefix."""
    sizes = [batch // 3, batch // 3, batch - 2 * (batch // 3)]
    call = _Call([1 + i % 2 for i in range(batch)], [2 + i % 40 for i in range(batch)], sizes, [600, 600, 0], 8, 2, 128, 16, torch.bfloat16, seed=23 + batch)
    call.prefix_table[1], call.prefix[1] = call.prefix_table[0], 411
    call.check("o", ops.paged_prefix_attention(*call.arguments(), max_q_len=2))


def test_far_pages():
    """Pages over 2^31 elements away."""
    pages = (1 << 31) // (16 * 2 * 64) + 40
    k, v = (torch.empty(pages, 2, 16, 64, dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2))
    call = _Call([1, 1, 2], [20, 5, 33], [3], [200], 4, 2, 64, 16, torch.bfloat16, seed=13)
    n = call.k.shape[0]
    args = list(call.arguments())
    k[pages - n:], v[pages - n:] = args[1], args[2]
    args[1], args[2] = k, v
    args[3], args[6] = args[3].clamp(0, n - 1) + (pages - n), args[6].clamp(0, n - 1) + (pages - n)
    call.check("o", ops.paged_prefix_attention(*args))


def test_refusals():
    call = _Call([1, 1], [5, 9], [2], [30], 4, 2, 64, 16, torch.bfloat16, seed=14)
    args = dict(zip(("q", "k_pages", "v_pages", "page_table", "cu_seqlens", "ctx_len", "prefix_table", "prefix_len", "group_seqs"), call.arguments()))
    ops.paged_prefix_attention(**args)
    empty = {**args, "q": args["q"][:0]}
    assert ops.paged_prefix_attention(**empty).shape == (0, 4, 64)
    for bad in (dict(prefix_table=args["prefix_table"].long()), dict(prefix_table=args["prefix_table"][0]), dict(prefix_len=_ints([1, 2])), dict(prefix_len=args["prefix_len"].long()),
                dict(group_seqs=_ints([0])), dict(group_seqs=_ints([0, 1, 2])), dict(prefix_table=args["prefix_table"][:, :0]), dict(prefix_table=args["prefix_table"].cpu()),
                dict(workspace=torch.empty(10, device=DEV)), dict(max_q_len=0), dict(softmax_scale=0.0), dict(softmax_scale=math.nan), dict(out=args["q"]),
                dict(q=args["q"].float()), dict(q=args["q"][..., :48].contiguous()), dict(prefix_table=args["prefix_table"][:0], prefix_len=_ints([]), group_seqs=_ints([0]))):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.paged_prefix_attention(**{**args, **bad})

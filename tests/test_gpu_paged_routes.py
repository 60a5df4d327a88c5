"""Attention over a paged cache where many sequences, blocks or splits decide how the work is cut: every row against float64."""

import math

import pytest
import torch

from scaling_amd import ops
from tests import paged_oracle as oracle
from tests.kernels import launched
from tests.test_gpu_head_rows import _close, _tables
from tests.test_gpu_paged import DEV, _cache, _device, _ints

pytestmark = pytest.mark.gpu

ROWS, TILES, MERGE = "paged_rows", "paged_tiles", "paged_merge"
ONE = [1]


def _spread(n, lo, hi):
    """n lengths between lo and hi, in no order"""
    return [lo + (i * 7919) % n * (hi - lo) // max(n - 1, 1) for i in range(n)]


# name: new tokens, keys with them, q heads, kv heads, d, page, type, whether max_q_len is given, launches (without tickets)
CALLS = {
    # Blocks for every compute unit (tokens x heads of a group / 256 x KV heads >= 256): chunks are not split.  17 x 16 blocks, longest first.
    "many_blocks": ([1100, 1050, 1200, 1001], [1100, 1400, 1210, 2950], 16, 16, 32, 16, torch.bfloat16, True, [TILES]),
    "many_blocks_f16": ([1100, 1050, 1200, 1001], [1300, 1050, 1210, 1700], 16, 16, 32, 64, torch.float16, True, [TILES]),
    "many_blocks_gqa": ([700, 820, 690], [900, 2000, 690], 32, 8, 64, 32, torch.bfloat16, True, [TILES]),
    # ... of more sequences than lanes, one after the other (21 x 16), short ones among them in blocks of few rows
    "many_blocks_70_sequences": (_spread(70, 20, 140), _spread(70, 140, 700), 16, 16, 32, 16, torch.bfloat16, True, [ROWS, TILES, MERGE]),
    # ... of as many sequences as lanes
    "many_blocks_64_chunks": ([66] * 64, _spread(64, 66, 700), 16, 16, 32, 16, torch.bfloat16, True, [TILES]),
    # ... and chunks alone (66 x 64 / 256 x 16 = 256)
    "many_blocks_66_chunks": ([64] * 66, _spread(66, 64, 700), 16, 16, 32, 16, torch.bfloat16, True, [TILES]),
    # 48 blocks of 64 that run at once, of one length: not split; of lengths far apart: split, with merges of 32 rows to a workgroup (48 x 4 blocks of 256 rows)
    "level": ([500] * 6, [3000] * 6, 16, 4, 32, 64, torch.bfloat16, True, [TILES, MERGE]),
    "not_level": ([500] * 6, [500, 600, 3000, 700, 900, 3900], 16, 4, 32, 64, torch.bfloat16, True, [TILES, MERGE]),
    "not_level_70_sequences": ([1] * 40 + [500, 1, 500, 480] + [1] * 24 + [500, 490], [60] * 40 + [500, 40, 3000, 700] + [90] * 24 + [900, 3900], 16, 4, 32, 64, torch.bfloat16, True,
                               [ROWS, TILES, MERGE]),
    # chunks behind the 64th sequence; 40 blocks of the 128 that run at once, whose splits are cut until they do
    "chunks_behind_64": ([1] * 66 + [300, 1, 290, 300, 1, 300, 270, 300, 1, 300, 260], [50 + i for i in range(66)] + [3000, 40, 3500, 900, 10, 3900, 2000, 3000, 700, 3100, 260], 8, 2, 64,
                         16, torch.bfloat16, True, [ROWS, TILES, MERGE]),
    "chunks_of_8": ([300, 290, 300, 270, 300, 260, 300, 300], [3000, 3500, 900, 3900, 2000, 3000, 3100, 260], 8, 2, 64, 16, torch.float16, True, [TILES, MERGE]),
    # few blocks of few rows each: pieces of a half and a quarter of the blocks' rows
    "short_chunks": ([20, 9, 24], [3000, 2000, 700], 16, 4, 128, 64, torch.bfloat16, True, [ROWS, TILES, MERGE]),
    "shorter_chunks": (_spread(20, 8, 16), _spread(20, 500, 3000), 16, 4, 128, 64, torch.float16, True, [ROWS, TILES, MERGE]),
    "two_blocks_of_few_rows": ([10, 9, 16], [3000, 2000, 700], 16, 4, 128, 64, torch.float16, True, [ROWS, MERGE]),
    # 32 x 8 items: cut for a quarter of the workgroups where they are of one length
    "even_tokens": (ONE * 32, [1500] * 32, 32, 8, 64, 16, torch.bfloat16, True, [ROWS, MERGE]),
    "uneven_tokens": (ONE * 32, _spread(32, 20, 3000), 32, 8, 64, 16, torch.float16, True, [ROWS, MERGE]),
    "even_drafts": ([5] * 32, [1200] * 32, 32, 8, 64, 32, torch.bfloat16, True, [ROWS, MERGE]),
    "uneven_drafts": ([i % 8 + 1 for i in range(32)], _spread(32, 20, 2500), 32, 8, 64, 32, torch.bfloat16, True, [ROWS, MERGE]),
    "tokens_of_200_sequences": (ONE * 200, _spread(200, 1, 1500), 8, 2, 64, 16, torch.bfloat16, True, [ROWS, MERGE]),
    "even_tokens_of_130_sequences": (ONE * 130, [1100] * 130, 8, 2, 32, 16, torch.bfloat16, True, [ROWS, MERGE]),
    "drafts_of_100_sequences": ([i % 6 for i in range(100)], _spread(100, 6, 1800), 16, 4, 32, 16, torch.bfloat16, True, [ROWS, MERGE]),
    # no bound of the lengths: all kernels, whatever there is for them
    "many_blocks_unbounded": ([1100, 1050, 1200, 1001], [1100, 1400, 1210, 2950], 16, 16, 32, 16, torch.bfloat16, False, [ROWS, TILES, MERGE]),
    # more tokens than keys, in some of many blocks: rows without keys
    "more_tokens_than_keys": ([1100, 1050, 1200, 1001], [500, 0, 1210, 3], 16, 16, 32, 16, torch.bfloat16, True, [TILES]),
    "more_tokens_than_keys_level": ([500] * 6, [1500, 20, 300, 1500, 0, 1500], 16, 4, 32, 64, torch.bfloat16, True, [TILES, MERGE]),
}


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("name", CALLS)
def test_every_row(name, causal):
    new, ctx, nq, nkv, d, page, dtype, bounded, launches = CALLS[name]
    print(f"case {name} {causal}", flush=True)
    k, v, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=sum(ctx) + d, spare=-(-max(0, 640 - max(ctx)) // page) + 1)
    q = (1.5 * torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(d + nq))).to(dtype)
    args = (q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    kwargs = dict(causal=causal, max_q_len=max(new) if bounded else None)
    out = torch.full_like(args[0], math.nan)
    names = launched(lambda: ops.paged_attention(*args, out=out, **kwargs))
    assert [n for n in (ROWS, TILES, MERGE) if any(n in x for x in names)] == launches, names
    ref, bound, _ = oracle.attention_by_sequence(q, k, v, table, cu, ctx, causal, 1 / math.sqrt(d))
    diff = (out.cpu().double() - ref).abs()
    worst = diff / bound.clamp_min(1e-300)
    print(f"max error / bound {float(worst.max()):.2f}", flush=True)
    assert bool((diff <= bound).all()), f"over the bound in {int((~(diff <= bound)).any(-1).sum())} of {diff.shape[0] * nq} rows, by up to {float(worst.max())}"
    ws = ops.paged_workspace(len(new), cu[-1], nq, nkv, d, DEV)
    again = torch.full_like(out, math.nan)
    for _ in range(2):                                      # with tickets: the same bits
        assert torch.equal(ops.paged_attention(*args, out=again, workspace=ws, **kwargs), out)
    torch.cuda.synchronize()
    assert int(ws.tickets.abs().sum()) == 0


# Rows whose leading key is ahead of every other by 64 in the exponent: their output is the leader's value, which the sum of at most 4000 weights of
# exp(-64) does not reach, times its weight over itself: both roundings of the weight's type (half a step each, of the result and of the weight for the product),
# and float32 ones of the exponential, the sums and the division.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,ctx,nq,nkv,d,spare,launches", [
    ([1, 40], [300, 80], 4, 2, 64, 0, [ROWS]),                          # blocks of few rows alone
    ([1, 7], [1000, 900], 8, 2, 128, 1, [ROWS, MERGE]),                 # split
    ([700, 90], [1000, 600], 4, 2, 32, 40, [TILES, MERGE]),             # chunks
    ([300], [4000], 8, 2, 128, 1, [TILES, MERGE]),
    ([1100, 1050, 1200, 1001], [1100, 1400, 1210, 1700], 16, 16, 32, 1, [TILES]),      # chunks that are not split
], ids=["rows", "splits", "chunks", "chunk-splits", "unsplit"])
def test_the_leading_key_wins(new, ctx, nq, nkv, d, spare, launches, dtype):
    """Scores that rise along the keys by 64 each (the maximum moves in every tile), that fall (the first key leads), and rows of both in one block."""
    page = 16
    k, v, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=sum(ctx), spare=spare)
    per_page = torch.zeros(k.shape[0], page, dtype=torch.int64)         # positions of the slots
    for b, length in enumerate(ctx):
        for i in range(-(-length // page)):
            per_page[table[b, i]] = page * i + torch.arange(page)
    stale = torch.isnan(k)
    k.zero_()
    k[..., 0], k[..., 1] = (per_page // 64)[..., None].to(dtype), (per_page % 64)[..., None].to(dtype)     # whole numbers below 64: exact in either type
    k[stale] = math.nan
    sign = torch.where(torch.randint(0, 2, (cu[-1], nq), generator=torch.Generator().manual_seed(1)) == 0, -1.0, 1.0)
    q = torch.zeros(cu[-1], nq, d)
    q[..., 0], q[..., 1] = 64 * 64 * sign, 64 * sign                    # score: 64 x position x sign, a whole number below 2^24
    q = q.to(dtype)
    args = (q.to(DEV), _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    names = launched(lambda: ops.paged_attention(*args, softmax_scale=1.0, max_q_len=max(new)))
    assert [n for n in (ROWS, TILES, MERGE) if any(n in x for x in names)] == launches, names
    out = ops.paged_attention(*args, softmax_scale=1.0, max_q_len=max(new)).cpu().double()
    half = torch.finfo(dtype).eps / 2
    for b, n in enumerate(new):
        pages = table[b, :-(-ctx[b] // page)].long()
        values = v[pages].reshape(-1, nkv, d)[:ctx[b]].double().repeat_interleave(nq // nkv, 1)
        rows = slice(cu[b], cu[b + 1])
        leader = torch.where(sign[rows] > 0, (ctx[b] - n + torch.arange(n))[:, None], 0)
        want = values[leader, torch.arange(nq)[None, :]]
        diff = (out[rows] - want).abs()
        bound = ((1 + half) ** 2 - 1 + 2.0 ** -18) * want.abs() + 4000 * math.exp(-64) * float(values.abs().max()) + 2.0 ** -24
        assert bool((diff <= bound).all()), (b, float((diff / bound).max()))


@pytest.mark.parametrize("new,ctx,nq,nkv,d,spare", [([3, 2], [40, 900], 8, 2, 64, 1), ([1, 1], [700, 90], 4, 2, 128, 1), ([100, 9], [150, 30], 4, 2, 64, 40), ([100], [3000], 4, 2, 64, 1),
                                                   ([1100, 1050, 1200, 1001], [1100, 1400, 1210, 1700], 16, 16, 32, 1)], ids=["drafts", "tokens", "chunks", "splits", "unsplit"])
def test_a_query_of_nan_stays_in_its_row(new, ctx, nq, nkv, d, spare):
    k, v, table, cu = _cache(new, ctx, nkv, d, 16, torch.bfloat16, seed=5, spare=spare)
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    rest = (_device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx))
    clean = ops.paged_attention(q, *rest, max_q_len=max(new))
    hit = torch.zeros(cu[-1], nq, dtype=torch.bool, device=DEV)
    for i in range(len(new)):
        hit[cu[i] + new[i] // 2, i % nq] = hit[cu[i + 1] - 1, nq - 1] = True
    q[..., 5].masked_fill_(hit, math.nan)
    out = ops.paged_attention(q, *rest, max_q_len=max(new))
    assert bool(torch.isfinite(clean).all()) and bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("name", ["sequences_150", "sequences_65", "float32_tables", "first_token_later"])
def test_appends_by_other_ways(name):
    """More sequences than lanes, empty ones among them; float32 tables; tokens in front of the first sequence."""
    nq, nkv, d, page, dtype = 4, 2, 64, 16, torch.bfloat16
    n = int(name.split("_")[1]) if name.startswith("sequences") else 5
    new = [(i * 5) % 4 for i in range(n)]
    new[0], new[-1] = 0, 2
    ctx = [c + (i * 37) % 90 for i, c in enumerate(new)]
    k_pages, v_pages, table, cu = _cache(new, ctx, nkv, d, page, dtype, seed=n, stale=2.0)
    front = 3 if name == "first_token_later" else 0
    cu = [c + front for c in cu]
    total, g = cu[-1] + 2, torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(total, h, d, generator=g).to(dtype) for h in (nq, nkv, nkv))
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    ids = torch.randint(0, 64, (total,), generator=g)
    cos, sin = _tables(64, d, dtype, False, torch.float32 if name == "float32_tables" else None)
    rotate = oracle.rotation(cos, sin, ids, d, False)
    kp, vp = _device(k_pages), _device(v_pages)
    out = ops.paged_append(k.to(DEV), v.to(DEV), kp, vp, table.to(DEV), _ints(cu), _ints(ctx), q=q.to(DEV), q_weight=w[0].to(DEV), k_weight=w[1].to(DEV),
                           rotary=(cos.to(DEV), sin.to(DEV), ids.to(DEV)))
    torch.cuda.synchronize()
    _close("q", out, *oracle.norm_rotary(q, w[0], None, 1e-5, False, rotate))
    where = oracle.slots(table, cu, ctx, page, k_pages.shape[0], total)
    stored = [t for t in range(total) if where[t] is not None]
    assert stored == list(range(cu[0], cu[-1]))
    at = tuple(torch.tensor(i) for i in zip(*(where[t] for t in stored)))
    ref, size = oracle.norm_rotary(k, w[1], None, 1e-5, False, rotate)
    _close("k", kp.cpu()[at], ref[stored], size[stored])
    assert torch.equal(vp.cpu()[at], v[stored])
    written = torch.zeros(k_pages.shape[:2], dtype=torch.bool)
    written[at] = True
    assert torch.equal(kp.cpu()[~written], k_pages[~written]) and torch.equal(vp.cpu()[~written], v_pages[~written])


@pytest.mark.parametrize("new,ctx,spare", [([3, 1], [40, 900], 1), ([100, 9], [150, 30], 40), ([100], [3000], 1)], ids=["rows", "chunks", "splits"])
def test_keys_that_all_score_minus_infinity_give_zeros(new, ctx, spare):
    """As a row without keys does; a score of plus infinity among them gives NaN."""
    nq, nkv, d = 4, 2, 64
    k, v, table, cu = _cache(new, ctx, nkv, d, 16, torch.bfloat16, seed=6, spare=spare, stale=0.5)
    k[..., 7] = -math.inf
    q = torch.randn(cu[-1], nq, d, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    q[..., 7] = 1.0
    q[cu[-1] - 1, 1, 7] = -1.0
    out = ops.paged_attention(q, _device(k), _device(v), table.to(DEV), _ints(cu), _ints(ctx), max_q_len=max(new))
    assert bool(torch.isnan(out[-1, 1]).all())
    out[-1, 1] = 0.0
    assert float(out.abs().max()) == 0.0

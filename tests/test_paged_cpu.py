"""CPU checks of the paged cache: how work is cut (the header compiled for the host), and refusals of the C entry points."""

import ctypes
import os
import subprocess

import pytest

from scaling_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "%s/scaling_amd/csrc/paged_plan.h"
#include <stdio.h>
#include <stdlib.h>
#include <vector>
static unsigned long long state = 88172645463325252ull;
static unsigned rnd() { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return (unsigned)(state >> 11); }
static int fail(const char* what, int i) { printf("case %%d: %%s\n", i, what); return 1; }
template <int BLOCK, int TILE>
static int kernel(int c, int over, int up_to, int batch, int n_rep, int total, int capacity, int longest, bool good, bool causal, const std::vector<int>& cu,
                  const std::vector<int>& ctx, std::vector<int>& taken) {
    PagedPlan p = {over, up_to, longest, rnd() %% 4 == 0 ? 0 : 1 << rnd() %% 9, 0, 0, 1 + (int)(rnd() %% 6), 0, 0};
    if (rnd() & 1) p.even = rnd() & 1;
    else if (rnd() & 1) p.fit = p.share >> rnd() %% 3;
    const int max_tiles = (capacity + TILE - 1) / TILE;
    const int64_t most = paged_max_blocks<BLOCK>(p, total, batch, longest, n_rep);
    p.max_slots = (int)paged_max_slots(p, most, max_tiles);
    p.max_partials = (int)paged_max_partials(p, most, max_tiles);
    int64_t units = 0, slots = 0, partials = 0, blocks = 0, split_blocks = 0;
    for (int b = 0; b < batch; ++b) {
        const PagedSeq s = paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity);
        if (s.first < 0 || s.n < 0 || s.first + s.n > total || s.len < 0 || s.len > capacity) return fail("a sequence outside the tokens or the table", c);
        const PagedWork w = paged_work<BLOCK, TILE>(p, s, n_rep);
        units += (int64_t)w.blocks * w.tiles;
    }
    int64_t all = 0, reached = 0;
    int longest_tiles = 0;
    for (int b = 0; b < batch; ++b) {
        const PagedWork w = paged_work<BLOCK, TILE>(p, paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity), n_rep);
        all += w.blocks;
        const int r = paged_reached<TILE>(paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity), w, causal);
        if (r > (int64_t)w.blocks * w.tiles) return fail("tiles of the middle block", c);
        reached += r;
        if (w.blocks > 0 && w.tiles > longest_tiles) longest_tiles = w.tiles;
    }
    const bool level = paged_level(p, all, longest_tiles, reached);
    if (level && (all > p.fit || paged_few(p, all))) return fail("level", c);
    int S = level ? 0x1000000 : paged_split_tiles(p, units, all, longest_tiles);
    for (int step = 0; p.share > 0 && step <= kPagedSteps; ++step) {
        int64_t n = 0;
        for (int b = 0; b < batch; ++b) {
            const PagedWork w = paged_work<BLOCK, TILE>(p, paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity), n_rep);
            n += (int64_t)w.blocks * paged_splits(p, w, S);
        }
        const int next = paged_next_tiles(p, S, units, all, n, step);
        if (next == S || (step < kPagedSteps && next < S)) {
            if (next != S || (paged_few(p, all) && n > p.fit && next < 0x1000000)) return fail("tiles of a split do not grow", c);
            break;
        }
        S = next;
    }
    if (S < 1) return fail("no tiles to a split", c);
    for (int b = 0; b < batch; ++b) {
        const PagedSeq s = paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity);
        const PagedWork w = paged_work<BLOCK, TILE>(p, s, n_rep);
        const int splits = paged_splits(p, w, S);
        if (splits < 1) return fail("no split", c);
        const bool fits = paged_fits(p, w, splits, (int)slots, (int)partials);
        if (good && w.blocks > 0 && !fits) return fail("a sequence left out", c);
        if (fits && w.blocks > 0 && slots + (int64_t)w.blocks * splits > p.max_slots) return fail("a workgroup that is not there", c);
        blocks += w.blocks;
        slots += (int64_t)w.blocks * splits;
        if (splits > 1) { partials += (int64_t)w.blocks * splits; split_blocks += w.blocks; }
        if (fits && splits > 1 && w.blocks > 0 && partials > p.max_partials) return fail("a partial result outside the workspace", c);
        if (w.blocks > 0 && good) for (int i = 0; i < s.n; ++i) ++taken[s.first + i];
        int at = 0;
        for (int i = 0; i < splits; ++i) {                 // splits cover the keys once, in order, in whole tiles
            int k0, k1;
            paged_split_keys<TILE>(s, w, splits, i, k0, k1);
            if (k0 != at || k1 < k0 || k1 > s.len || (k0 %% TILE != 0 && k0 != s.len) || (k1 - k0 + TILE - 1) / TILE > (S > p.least ? S : p.least)) return fail("keys of a split", c);
            at = k1;
        }
        if (at != s.len) return fail("keys left out", c);
        for (int i = 0; i < s.n; i += 1 + s.n / 5) {
            const int64_t want = causal ? (int64_t)s.ctx - s.n + i + 1 : s.len;
            const int got = paged_limit(s, i, causal);
            if (got != (want < 0 ? 0 : want > s.len ? s.len : (int)want)) return fail("limit of a row", c);
        }
    }
    if (good && BLOCK == 256 && batch <= 64) {             // longest first: every block once
        std::vector<int> seen(all, 0), before(batch, 0);
        for (int b = 1; b < batch; ++b) before[b] = before[b - 1] + paged_work<BLOCK, TILE>(p, paged_seq(cu[b - 1], cu[b], ctx[b - 1], total, capacity), n_rep).blocks;
        int previous = 0x7fffffff;
        for (int wanted = 0; wanted < all; ++wanted) {
            int lo = -1, hi = 0;
            const auto above = [&](int b, int x) {
                const PagedSeq s = paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity);
                return paged_above<BLOCK, TILE>(s, paged_work<BLOCK, TILE>(p, s, n_rep), n_rep, causal, x);
            };
            const auto sum = [&](int x) { int64_t n = 0; for (int b = 0; b < batch; ++b) n += above(b, x); return n; };
            for (int b = 0; b < batch; ++b) { const int t = (paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity).len + TILE - 1) / TILE; if (t > hi) hi = t; }
            if (sum(-1) != all || sum(hi) != 0) return fail("blocks above the ends", c);
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (sum(mid) > wanted) lo = mid; else hi = mid; }
            if (lo > previous) return fail("a longer block later", c);
            previous = lo;
            int in = wanted - (int)sum(hi), at = -1;
            for (int b = 0; b < batch && at < 0; ++b) {
                const int width = above(b, lo) - above(b, hi);
                if (width < 0) return fail("blocks beyond more keys that are not beyond fewer", c);
                if (in < width) at = before[b] + above(b, hi) + in;
                else in -= width;
            }
            if (at < 0 || at >= all || seen[at]++) return fail("a block twice", c);
        }
    }
    if (good && (blocks > most || (blocks == 0) < (most == 0))) return fail("more blocks than the bound", c);
    if (good && (slots > p.max_slots || partials > p.max_partials || split_blocks > paged_max_split_blocks(p, most))) return fail("more workgroups or partial results than the bound", c);
    return 0;
}
int main() {
    for (int c = 0; c < 4000; ++c) {
        const int batch = 1 + rnd() %% (c %% 5 == 0 ? 300 : 9), n_rep = 1 + rnd() %% 40, nkv = 1 + rnd() %% 9, pages = 1 + rnd() %% 70, page = 16 * (1 + rnd() %% 9);
        const int capacity = pages * page;
        const bool good = c %% 3 != 0, causal = rnd() & 1;
        std::vector<int> cu(batch + 1), ctx(batch);
        int total = 0;
        for (int b = 0; b < batch; ++b) {
            const int n = rnd() %% 4 == 0 ? rnd() %% 700 : rnd() %% 3;
            cu[b] = total;
            total += n;
            ctx[b] = (int)(rnd() %% (capacity + 40));
            if (!good) { if (rnd() %% 3 == 0) cu[b] = (int)(rnd() - 2147483648u); if (rnd() %% 3 == 0) ctx[b] = (int)(rnd() - 2147483648u); }
        }
        cu[batch] = good ? total : (int)(rnd() - 2147483648u);
        int longest = 0;
        std::vector<int> taken(good ? total : 0, 0);
        for (int b = 0; b < batch; ++b) { const PagedSeq s = paged_seq(cu[b], cu[b + 1], ctx[b], total, capacity); if (s.n > longest) longest = s.n; }
        if (c & 1) {
            if (kernel<16, 128>(c, 0, 32, batch, n_rep, total, capacity, longest, good, causal, cu, ctx, taken)) return 1;
        } else if (kernel<32, 128>(c, 0, 32, batch, n_rep, total, capacity, longest, good, causal, cu, ctx, taken)) return 1;
        if (kernel<256, 64>(c, 32, 0x7fffffff, batch, n_rep, total, capacity, longest, good, causal, cu, ctx, taken)) return 1;
        for (int t : taken) if (t != 1) return fail("a token that is not exactly one kernel's", c);
    }
    printf("ok\n");
    return 0;
}
"""


def test_work_is_cut_within_its_bounds(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(PROGRAM % ROOT)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout + done.stderr


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


@pytest.fixture()
def base():
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf)
    yield at + (-at) % 16
    del buf


def test_struct_layouts(tmp_path):
    header = os.path.join(ROOT, "include", "mi355_layer.h")
    names = {"mi_norm_rotary_args": (_lib.MiNormRotaryArgs, "stream"), "mi_norm_rotary_bwd_args": (_lib.MiNormRotaryBwdArgs, "workspace"),
             "mi_paged_append_args": (_lib.MiPagedAppendArgs, "max_pages"), "mi_paged_attn_args": (_lib.MiPagedAttnArgs, "stream")}
    lines = "".join(f'printf("%zu %zu\\n",sizeof({n}),offsetof({n},{f}));' for n, (_, f) in names.items())
    src = tmp_path / "sz.c"
    src.write_text(f'#include "{header}"\n#include <stdio.h>\n#include <stddef.h>\nint main(){{{lines}return 0;}}\n')
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "sz")], check=True)
    out = subprocess.run([str(tmp_path / "sz")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [v for s, f in names.values() for v in (ctypes.sizeof(s), getattr(s, f).offset)]


def _rows(base):
    a = _lib.MiNormRotaryArgs()
    a.q = a.k = a.q_out = a.k_out = a.q_weight = a.k_weight = a.rotary_cos = a.rotary_sin = a.position_ids = base
    a.n_tokens, a.table_rows, a.n_q_heads, a.n_kv_heads, a.head_dim, a.rot_dim, a.eps = 4, 4, 2, 2, 64, 64, 1e-5
    a.q_stride_token = a.k_stride_token = a.q_out_stride_token = a.k_out_stride_token = 128
    a.q_stride_head = a.k_stride_head = a.q_out_stride_head = a.k_out_stride_head = 64
    return a


def _set(a, **fields):
    for name, value in fields.items():
        setattr(a, name, value)
    return a


ROWS_REFUSED = [
    (dict(n_tokens=-1), -3), (dict(n_q_heads=-1), -3), (dict(n_q_heads=0, n_kv_heads=0), -3), (dict(head_dim=0), -3), (dict(head_dim=257), -3),
    (dict(n_tokens=2 ** 30), -3), (dict(n_q_heads=70000), -3), (dict(dtype=7), -2), (dict(q=None), -1), (dict(k=None), -1), (dict(eps=-1.0), -3),
    (dict(eps=float("nan")), -3), (dict(rotary_sin=None), -1), (dict(rotary_cos=None), -1), (dict(position_ids=None), -1), (dict(table_rows=0), -3),
    (dict(rot_dim=63), -3), (dict(rot_dim=66), -3), (dict(rot_dim=0), -3), (dict(rotary_interleaved=1), -3), (dict(rotary_interleaved=1, table_dtype=2, rot_dim=32), -3),
    (dict(table_dtype=1), -2),
]


def test_norm_rotary_refusals(lib, base):
    assert lib.mi_norm_rotary_fwd(None) == -1 and lib.mi_norm_rotary_bwd(None) == -1
    for fields, status in ROWS_REFUSED + [(dict(q_out=None), -1), (dict(k_out=None), -1), (dict(q_weight=None), -1), (dict(k_weight=None), -1)]:
        assert lib.mi_norm_rotary_fwd(ctypes.byref(_set(_rows(base), **fields))) == status, fields
    assert lib.mi_norm_rotary_fwd(ctypes.byref(_set(_rows(base), n_tokens=0, q=None))) == 0            # nothing to do
    b = _lib.MiNormRotaryBwdArgs()
    b.d_q_out = b.d_k_out = b.dq = b.dk = b.dq_weight = b.dk_weight = b.workspace = base
    b.workspace_bytes = lib.mi_norm_rotary_bwd_workspace_bytes(64)
    assert b.workspace_bytes >= 64 * 8 and lib.mi_norm_rotary_bwd_workspace_bytes(0) == 0
    for fields, status in ROWS_REFUSED + [(dict(q_weight=None), -1), (dict(n_tokens=0), -3)]:
        b.fwd = _set(_rows(base), **fields)
        assert lib.mi_norm_rotary_bwd(ctypes.byref(b)) == status, fields
    b.fwd = _rows(base)
    for field in ("d_q_out", "d_k_out", "dq", "dk"):
        setattr(b, field, None)
        assert lib.mi_norm_rotary_bwd(ctypes.byref(b)) == -1, field
        setattr(b, field, base)
    for fields in (dict(workspace=None), dict(workspace=base + 4), dict(workspace_bytes=16)):
        kept = {n: getattr(b, n) for n in fields}
        assert lib.mi_norm_rotary_bwd(ctypes.byref(_set(b, **fields))) == -5, fields
        _set(b, **kept)


def test_paged_append_refusals(lib, base):
    assert lib.mi_paged_append(None) == -1

    def args(**fields):
        a = _lib.MiPagedAppendArgs()
        a.rows = _set(_rows(base), **{n: v for n, v in fields.items() if hasattr(_lib.MiNormRotaryArgs, n)})
        a.v = a.k_pages = a.v_pages = a.page_table = a.cu_seqlens = a.ctx_len = base
        a.v_stride_token, a.v_stride_head, a.page_stride, a.page_stride_token, a.page_stride_head = 128, 64, 16 * 128, 128, 64
        a.page_table_stride = a.max_pages = 3
        a.batch, a.n_pages, a.page_size = 1, 5, 16
        return _set(a, **{n: v for n, v in fields.items() if hasattr(_lib.MiPagedAppendArgs, n)})
    for fields, status in ROWS_REFUSED + [
            (dict(dtype=2, table_dtype=2), -2), (dict(n_kv_heads=0), -3), (dict(batch=0), -3), (dict(n_pages=0), -3), (dict(max_pages=0), -3), (dict(page_size=8), -3), (dict(page_size=24), -3),
            (dict(max_pages=2 ** 28), -3), (dict(v=None), -1), (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(page_table=None), -1), (dict(cu_seqlens=None), -1),
            (dict(ctx_len=None), -1), (dict(q_out=None), -1), (dict(k_pages=base + 2), -4), (dict(page_stride=4), -4), (dict(page_stride_token=4), -4), (dict(page_stride_head=4), -4)]:
        assert lib.mi_paged_append(ctypes.byref(args(**fields))) == status, fields
    assert lib.mi_paged_append(ctypes.byref(args(n_tokens=0))) == 0


def test_paged_attention_refusals(lib, base):
    assert lib.mi_paged_attn(None) == -1

    def args(**fields):
        a = _lib.MiPagedAttnArgs()
        a.q = a.k_pages = a.v_pages = a.o = a.page_table = a.cu_seqlens = a.ctx_len = a.workspace = base
        a.total_q, a.batch, a.n_pages, a.page_size, a.max_pages, a.page_table_stride = 5, 2, 9, 16, 40, 40
        a.n_q_heads, a.n_kv_heads, a.head_dim, a.causal, a.softmax_scale = 4, 2, 64, 1, 0.125
        a.q_stride_token = a.o_stride_token = 256
        a.q_stride_head = a.o_stride_head = 64
        a.page_stride, a.page_stride_token, a.page_stride_head = 16 * 128, 128, 64
        a.workspace_bytes = lib.mi_paged_attn_workspace_bytes(5, 4, 2, 64)
        return _set(a, **fields)
    for fields, status in [
            (dict(total_q=-1), -3), (dict(total_q=2 ** 31), -3), (dict(batch=0), -3), (dict(n_pages=0), -3), (dict(max_pages=0), -3), (dict(max_pages=2 ** 27), -3), (dict(page_size=0), -3),
            (dict(page_size=20), -3), (dict(max_q_len=-1), -3), (dict(n_kv_heads=3), -3), (dict(n_q_heads=0), -3), (dict(n_kv_heads=0), -3), (dict(head_dim=80), -3), (dict(dtype=2), -2),
            (dict(q=None), -1), (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(o=None), -1), (dict(page_table=None), -1), (dict(cu_seqlens=None), -1), (dict(ctx_len=None), -1),
            (dict(softmax_scale=0.0), -3), (dict(softmax_scale=float("nan")), -3), (dict(q=base + 2), -4), (dict(o=base + 8), -4), (dict(q_stride_token=4), -4), (dict(o_stride_head=2), -4),
            (dict(page_stride=4), -4), (dict(page_stride_token=2 ** 27), -3), (dict(page_stride_token=-128), -3), (dict(workspace=None), -5), (dict(workspace=base + 4), -5),
            (dict(workspace_bytes=64), -5), (dict(tickets=base, n_tickets=3), -5), (dict(tickets=base + 2, n_tickets=10 ** 6), -5), (dict(total_q=2 ** 30), -3), (dict(n_q_heads=70000, n_kv_heads=70000), -3)]:
        assert lib.mi_paged_attn(ctypes.byref(args(**fields))) == status, fields
    assert lib.mi_paged_attn(ctypes.byref(args(total_q=0, q=None))) == 0
    sizes = [lib.mi_paged_attn_workspace_bytes(t, 32, 8, 128) for t in (1, 4, 5, 1000, 10 ** 6)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.mi_paged_attn_tickets(0) == 0 and lib.mi_paged_attn_tickets(8) > 0
    assert lib.mi_paged_attn_workspace_bytes(0, 32, 8, 128) == 0 and lib.mi_paged_attn_workspace_bytes(5, 32, 7, 128) == 0

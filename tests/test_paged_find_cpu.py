"""The search that every workgroup of paged attention makes for its work, compiled for the host over an array of 64 lanes."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

REACHED = r"""
#include "%s/scaling_amd/csrc/paged_plan.h"
#include <initializer_list>
#include <stdio.h>
int main() {
    const PagedPlan p = {0, 0x7fffffff, 0x7fffffff, 64, 0, 64, 6, 0, 0};
    for (int n = 1; n <= 1 << 22; n = n * 3 + 1)
        for (int ctx : {0, 1, 20, 300, 5000, 1 << 20, 1 << 30})
            for (int n_rep : {1, 4, 64}) {
                const PagedSeq s = paged_seq(0, n, ctx, n, 1 << 30);
                const PagedWork w = paged_work<256, 64>(p, s, n_rep);
                if ((int64_t)w.blocks * w.tiles > 0x7fffffff) continue;      // refused by the host
                for (int causal = 0; causal < 2; ++causal) {
                    const int r = paged_reached<64>(s, w, causal);
                    if (r < 0 || r > w.blocks * w.tiles) { printf("%%d tokens, %%d keys: %%d\n", n, ctx, r); return 1; }
                }
            }
    printf("ok\n");
    return 0;
}
"""


PROGRAM = r"""
#include "%s/scaling_amd/csrc/paged_plan.h"
#include <stdio.h>
#include <array>
#include <map>
#include <set>
#include <tuple>
#include <vector>
static unsigned long long state = 88172645463325252ull;
static unsigned rnd() { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return (unsigned)(state >> 11); }
static int fail(const char* what, int i) { printf("case %%d: %%s\n", i, what); return 1; }

struct Lane64 : std::array<int, 64> {
    Lane64 operator-(const Lane64& o) const { Lane64 r; for (int i = 0; i < 64; ++i) r[i] = (*this)[i] - o[i]; return r; }
};
struct Call {
    std::vector<int> cu, ctx;
    int batch, n_rep, total, capacity, longest;
    bool causal, good;
};
template <int BLOCK, int TILE> struct Lanes {
    const Call& c;
    const PagedPlan& plan;
    PagedSeq s[64];
    PagedWork w[64];
    void look(int base) {
        for (int l = 0; l < 64; ++l) {
            const int b = base + l, i = b < c.batch ? b : c.batch - 1;
            s[l] = paged_seq(c.cu[i], c.cu[i + 1], c.ctx[i], c.total, c.capacity);
            w[l] = paged_work<BLOCK, TILE>(plan, s[l], c.n_rep);
            if (b >= c.batch) w[l].blocks = s[l].n = 0;
        }
    }
    template <class F> Lane64 of(const F& f) const { Lane64 v; for (int l = 0; l < 64; ++l) v[l] = f(s[l], w[l]); return v; }
    template <class F> Lane64 of(const Lane64& x, const F& f) const { Lane64 v; for (int l = 0; l < 64; ++l) v[l] = f(w[l], x[l]); return v; }
    int value(const Lane64& v, int l) const { return v[l]; }
    int64_t total(const Lane64& v) const { int64_t n = 0; for (int x : v) n += x; return n; }
    int most(const Lane64& v) const { int m = v[0]; for (int x : v) m = x > m ? x : m; return m; }
    Lane64 upto(const Lane64& v) const { Lane64 r; int n = 0; for (int l = 0; l < 64; ++l) r[l] = n += v[l]; return r; }
    int holder(const Lane64& v, const Lane64& upto, int x) const { for (int l = 0; l < 64; ++l) if (x >= upto[l] - v[l] && x < upto[l]) return l; return -1; }
    PagedSeq seq(int l) const { return s[l]; }
    PagedWork work(int l) const { return w[l]; }
};
static int n_longest, n_level, n_cut, n_split, n_merged, n_left_out;

// all workgroups of a launch of BLOCK rows, and those that merge
template <int BLOCK, int TILE, PagedOrder ORDER> static int launch(int i, const Call& c, PagedPlan p, std::vector<int>& taken) {
    const int max_tiles = (c.capacity + TILE - 1) / TILE;
    const int64_t most = paged_max_blocks<BLOCK>(p, c.total, c.batch, c.longest, c.n_rep);
    const uint32_t share_m = p.share > 1 ? (uint32_t)((1ull << 32) / p.share + 1) : 0;
    p.max_slots = (int)paged_max_slots(p, most, max_tiles);
    p.max_partials = (int)paged_max_partials(p, most, max_tiles);
    Lanes<BLOCK, TILE> lanes{c, p, {}, {}};
    std::set<std::tuple<int, int, int>> seen;                  // sequence, split, block
    std::map<int, PagedFound> split;                            // sequences with several splits
    std::set<int> partials;
    int64_t reach = -1;
    for (int slot = 0; slot < p.max_slots + 3; ++slot) {
        const PagedFound f = paged_find<BLOCK, TILE, ORDER>(lanes, p, share_m, c.batch, c.n_rep, c.causal, slot);
        if (f.b < 0) { ++n_left_out; continue; }
        if (slot >= p.max_slots) {                              // (sequences that share tokens have blocks that no workgroup is left for)
            if (c.good || p.share > 0) return fail("work behind the last workgroup", i);
            continue;
        }
        const PagedSeq s = paged_seq(c.cu[f.b], c.cu[f.b + 1], c.ctx[f.b], c.total, c.capacity);
        const PagedWork w = paged_work<BLOCK, TILE>(p, s, c.n_rep);
        if (s.first != f.seq.first || s.n != f.seq.n || s.ctx != f.seq.ctx || s.len != f.seq.len || w.blocks != f.work.blocks || w.tiles != f.work.tiles) return fail("another sequence", i);
        const int in = slot - f.at;
        if (in < 0 || in >= f.work.blocks * f.splits) return fail("a slot outside its sequence", i);
        const int part = in / f.work.blocks, block = f.work.blocks - 1 - (in - part * f.work.blocks);
        if (!seen.insert({f.b, part, block}).second) return fail("a block twice", i);
        if (f.splits > 1) {
            ++n_split;
            if (f.partial < 0 || f.partial + in >= p.max_partials) return fail("a partial result outside the workspace", i);
            if (!partials.insert(f.partial + in).second) return fail("a partial result twice", i);
            const auto other = split.insert({f.b, f}).first->second;
            if (other.partial != f.partial || other.splits != f.splits) return fail("splits that disagree", i);
        } else if (p.share == 0 && ORDER == kLongestFirst && c.batch <= 64 && c.good) {      // by the most whole tiles that a block reaches beyond
            ++n_longest;
            int x = -1;
            while (paged_above<BLOCK, TILE>(s, w, c.n_rep, c.causal, x + 1) > w.blocks - 1 - block) ++x;
            if (reach >= 0 && x > reach) return fail("a longer block later", i);
            reach = x < 0 ? 0 : x;
        }
        if (part == 0 && block == 0) for (int t = 0; t < s.n; ++t) ++taken[s.first + t];
    }
    if (c.good) {
        size_t want = 0;
        int64_t blocks = 0;
        for (int b = 0; b < c.batch; ++b) {
            const PagedWork w = paged_work<BLOCK, TILE>(p, paged_seq(c.cu[b], c.cu[b + 1], c.ctx[b], c.total, c.capacity), c.n_rep);
            const auto at = split.find(b);
            want += (size_t)w.blocks * (at == split.end() ? 1 : at->second.splits);
            blocks += w.blocks;
        }
        if (seen.size() != want) return fail("work that nobody does", i);
        if (p.share > 0 && paged_few(p, blocks)) { ++n_cut; if ((int64_t)seen.size() > p.fit) return fail("more workgroups than run at once", i); }
        if (p.fit > 0 && !paged_few(p, blocks) && blocks > 1 && split.empty()) ++n_level;
    }
    std::set<std::pair<int, int>> merged;
    const int groups = (int)paged_max_split_blocks(p, most);
    for (int at = 0; at < groups + 3; ++at) {
        const PagedFound f = paged_find<BLOCK, TILE, kSplitBlocks>(lanes, p, share_m, c.batch, c.n_rep, c.causal, at);
        if (f.b < 0) continue;
        if (at >= groups) {
            if (c.good) return fail("a merge behind the last workgroup", i);
            continue;
        }
        const auto other = split.find(f.b);
        if (other == split.end() || other->second.partial != f.partial || other->second.splits != f.splits) return fail("a merge of what nobody computed", i);
        const int block = at - f.at;
        if (block < 0 || block >= f.work.blocks || !merged.insert({f.b, block}).second) return fail("a merge twice", i);
        for (int part = 0; part < f.splits; ++part)
            if (!seen.count({f.b, part, block}) || !partials.count(f.partial + part * f.work.blocks + block)) return fail("a merge of a split that nobody computed", i);
        ++n_merged;
    }
    size_t want = 0;
    for (const auto& x : split) want += x.second.work.blocks;
    if (c.good && merged.size() != want) return fail("splits that nobody merges", i);
    return 0;
}

int main() {
    for (int i = 0; i < 1500; ++i) {
        Call c;
        c.batch = 1 + rnd() %% (i %% 5 == 0 ? 300 : i %% 5 == 1 ? 70 : 9);
        c.n_rep = 1 + rnd() %% 40;
        c.capacity = (1 + rnd() %% 70) * 16 * (1 + rnd() %% 9);
        c.good = i %% 3 != 0;
        c.causal = rnd() & 1;
        c.cu.resize(c.batch + 1);
        c.ctx.resize(c.batch);
        c.total = 0;
        const unsigned chunks = rnd() %% 4, alike = rnd() %% 3;
        const int same = (int)(rnd() %% c.capacity) + 1;
        for (int b = 0; b < c.batch; ++b) {
            const int n = rnd() %% 4 < chunks ? rnd() %% 700 : rnd() %% 3;
            c.cu[b] = c.total;
            c.total += n;
            c.ctx[b] = alike == 0 ? same : (int)(rnd() %% (c.capacity + 40));
            if (!c.good && rnd() %% 3 == 0) c.cu[b] = (int)(rnd() %% 4000u) - 100;
            if (!c.good && rnd() %% 3 == 0) c.ctx[b] = (int)(rnd() - 2147483648u);
        }
        c.cu[c.batch] = c.total;
        c.longest = 0;
        for (int b = 0; b < c.batch; ++b) { const PagedSeq s = paged_seq(c.cu[b], c.cu[b + 1], c.ctx[b], c.total, c.capacity); if (s.n > c.longest) c.longest = s.n; }
        std::vector<int> taken(c.total, 0);
        const int share = rnd() %% 3 == 0 ? 0 : 1 << rnd() %% 9;
        // as the host makes them: rows 0 to `limit` with `even`, chunks over it with `fit`
        const int limit = rnd() %% 8 == 0 ? 0 : rnd() & 1 ? 32 : 64, fit = share >> rnd() %% 3;
        const PagedPlan rows = {0, limit, c.longest, rnd() %% 4 == 0 ? 0 : 1 << rnd() %% 9, (int)(rnd() & 1), 0, 1 + (int)(rnd() %% 6), 0, 0};
        const PagedPlan tiles = {limit, 0x7fffffff, c.longest, share, 0, share == 0 || fit == 0 ? 0 : fit, 1 + (int)(rnd() %% 6), 0, 0};
        if (limit > 0 && (i & 1 ? launch<16, 128, kSlots>(i, c, rows, taken) : launch<32, 128, kSlots>(i, c, rows, taken))) return 1;
        if (launch<256, 64, kLongestFirst>(i, c, tiles, taken)) return 1;
        if (c.good) for (int t : taken) if (t != 1) return fail("a token that is not exactly one kernel's", i);
    }
    if (!n_longest || !n_level || !n_cut || !n_split || !n_merged || !n_left_out) return fail("a way of cutting that no case takes", -1);
    // the shares of a plan by their multiplier, and quotients that start beside the right one
    for (int i = 0; i < 400000; ++i) {
        PagedPlan p{};
        p.share = 1 + (int)(rnd() %% (1u << rnd() %% 16));
        const uint32_t share_m = p.share > 1 ? (uint32_t)((1ull << 32) / p.share + 1) : 0;
        uint32_t u = rnd() >> rnd() %% 31 & 0x7fffffffu;
        if (i & 1) { const int64_t x = (int64_t)(u / p.share) * p.share + (int)(rnd() %% 3) - 1; u = x < 0 ? 0 : x > 0x7fffffff ? 0x7fffffff : (uint32_t)x; }
        if (paged_by_share(p, u, share_m) != (int)(u / (uint32_t)p.share)) return fail("a share", (int)u);
        const int a = (int)(rnd() >> rnd() %% 24 & 0xffffff), b = 1 + (int)(rnd() >> rnd() %% 24 & 0xffffff);
        for (int off = -2; off <= 2; ++off) {
            const int64_t q = (int64_t)a / b + off;
            if (q * b > 0x7fffffff - b || a - q * b > 0x7fffffff) continue;
            if (paged_corrected(a, b, (int)q) != a / b) return fail("a quotient", a);
        }
    }
    printf("ok\n");
    return 0;
}
"""


def _run(tmp_path, program):
    src, exe = tmp_path / "program.cpp", tmp_path / "program"
    src.write_text(program % ROOT)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout + done.stderr


def test_tiles_that_blocks_reach_are_no_fewer_than_none(tmp_path):
    """Of sequences of more tokens than keys, too: their sums over 64 sequences are taken as numbers without a sign."""
    _run(tmp_path, REACHED)


def test_every_workgroup_finds_its_work(tmp_path):
    """Every block and split once, by the workgroups that there are; partial results apart; the merges of just these; the arithmetic of the divisions."""
    _run(tmp_path, PROGRAM)

// Who computes what in attention over a paged cache: sequences, their key ranges and how their work is cut, from lengths that lie on the device.  Plain
// arithmetic, the same for every workgroup of a launch and for the launch that merges; compiles for the host alone too.
//
// A sequence's rows are (new token, query head of a group): token i of n and head r of n_rep make row i * n_rep + r, so all heads that share keys share a
// block of rows.  A kernel takes the sequences whose number of rows it suits, in blocks of rows, with keys in tiles.  The keys of a sequence are cut into
// splits of at most S tiles each, with S such that all splits together are about `share` workgroups per KV head:
//     W = sum over sequences of blocks * tiles,   S = floor(W / share) + 1,   splits_b = ceil(tiles_b / S), of short sequences 1
// Then splits of all blocks are at most share + blocks in number, and those of sequences with more than one split at most 2 * share (tiles > S gives
// ceil(tiles / S) < 2 tiles / S).  Lengths may be anything: sequences are clamped to the tokens and the page table that there are, and where lengths that
// overlap make more workgroups or partial results than there are, sequences are left out as a whole.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define MI_PLAN_FN static __host__ __device__ __forceinline__
#else
#define MI_PLAN_FN static inline
#endif

struct PagedSeq {
    int first, n;     // new tokens
    int ctx, len;     // keys by ctx_len, and those that the page table has room for
};

MI_PLAN_FN int paged_clamp(int64_t x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : (int)x); }

MI_PLAN_FN PagedSeq paged_seq(int cu0, int cu1, int ctx, int total, int capacity) {
    PagedSeq s;
    s.first = paged_clamp(cu0, 0, total);
    s.n = paged_clamp(cu1, s.first, total) - s.first;
    s.ctx = ctx < 0 ? 0 : ctx;
    s.len = s.ctx < capacity ? s.ctx : capacity;
    return s;
}

// keys that new token i may attend to: the first so many
MI_PLAN_FN int paged_limit(const PagedSeq& s, int i, bool causal) {
    return causal ? paged_clamp((int64_t)s.ctx - s.n + i + 1, 0, s.len) : s.len;
}

// a / b for a < 2^24, 0 < b, by a reciprocal and corrections (the compiler's division is five times as long, and a workgroup's first steps wait for it)
MI_PLAN_FN int paged_quotient(int a, int b) {
#ifdef __HIP_DEVICE_COMPILE__
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));      // two units in the last place of up to 24 bits: off by at most 2
    int r = a - q * b;
    for (int i = 0; i < 2; ++i) {
        const int by = r < 0 ? -1 : r >= b ? 1 : 0;
        q += by;
        r -= by * b;
    }
    return q;
#else
    return a / b;
#endif
}

struct PagedPlan {
    int rows_over, rows_up_to;    // sequences with more than rows_over and at most rows_up_to rows
    int max_n;                    // ... and at most so many new tokens
    int share;                    // workgroups per KV head aimed at; 0: never split
    int even;                     // sequences of about one length: cut for a quarter of the share
    int fit;                      // workgroups per KV head that run at once: few blocks are cut for no more of them; 0: no such line
    int least;                    // sequences of no more tiles are not split
    int max_slots, max_partials;  // (set by the host) workgroups and partial results per KV head that there are
};

struct PagedWork {
    int blocks, tiles;            // blocks 0: not this kernel's
};
// BLOCK rows to a block, TILE keys to a tile: powers of two
template <int BLOCK, int TILE> MI_PLAN_FN PagedWork paged_work(const PagedPlan& p, const PagedSeq& s, int n_rep) {
    const int rows = s.n * n_rep;                           // of all tokens: fewer than 2^31
    PagedWork w;
    w.blocks = rows > p.rows_over && rows <= p.rows_up_to && s.n <= p.max_n ? (int)(((uint32_t)rows + BLOCK - 1) / BLOCK) : 0;
    w.tiles = s.len > 0 ? (s.len + TILE - 1) / TILE : 1;    // rows without keys are written too
    return w;
}
// What is divided by the share for the tiles of a split, less one.  units: W; blocks: of all sequences; most: tiles of the longest
MI_PLAN_FN bool paged_few(const PagedPlan& p, int64_t blocks) { return p.fit > 0 && 2 * blocks <= p.fit; }
MI_PLAN_FN uint32_t paged_units(const PagedPlan& p, int64_t units, int64_t blocks, int most) {
    if (p.even && most * blocks * 4 <= units * 5) units *= 4;
    if (paged_few(p, blocks)) units *= p.share / p.fit;
    return (uint32_t)(units < 0x7fffffff ? units : 0x7fffffff);
}
MI_PLAN_FN int paged_split_tiles(const PagedPlan& p, int64_t units, int64_t blocks, int most) {
    if (p.share == 0) return 0x1000000;                    // no sequence has more
    return (int)(paged_units(p, units, blocks, most) / (uint32_t)p.share) + 1;
}
// Tiles that a sequence's blocks have, by the middle one of them (which of more tokens than keys may have none)
template <int TILE> MI_PLAN_FN int paged_reached(const PagedSeq& s, const PagedWork& w, bool causal) {
    const int64_t all = (int64_t)w.blocks * w.tiles, hidden = causal ? (int64_t)w.blocks * s.n / (2 * TILE) : 0;
    return all > hidden ? (int)(all - hidden) : 0;
}
// Blocks that run at once, more than half of what does, of which the longest is no more than half again a workgroup's share of all: not split, as twice the
// pieces of half the length would take two rounds, and a merge.  (6 x 500 tokens of 3000 keys, 16 / 4 heads of 128, 192 blocks: 123 us split, 105 not; one prompt of 3900 tokens, whose
// blocks reach from 4 to 61 tiles: 103 split, 130 not.)
MI_PLAN_FN bool paged_level(const PagedPlan& p, int64_t blocks, int most, int64_t reached) {
    return p.fit > 0 && !paged_few(p, blocks) && blocks <= p.fit && 2 * most * (int64_t)p.fit <= 3 * reached;
}
// Of few blocks S grows until their splits run at once: one workgroup more would take as long as all others.  `slots`: splits of all blocks at S.  After
// kPagedSteps steps S is W / (fit - blocks) + 1, which sum(ceil(tiles / S)) < W / S + blocks leaves no more than fit of.
constexpr int kPagedSteps = 3;
MI_PLAN_FN int paged_next_tiles(const PagedPlan& p, int split_tiles, int64_t units, int64_t blocks, int64_t slots, int step) {
    if (!paged_few(p, blocks) || slots <= p.fit) return split_tiles;
    if (step == kPagedSteps) return paged_clamp((int64_t)((float)units / (float)(p.fit - blocks) * 1.000001f) + 1, 1, 0x1000000);
    const int64_t next = (int64_t)((float)split_tiles * (float)slots / (float)p.fit);
    return paged_clamp(next > split_tiles ? next : (int64_t)split_tiles + 1, 1, 0x1000000);
}
MI_PLAN_FN int paged_splits(const PagedPlan& p, const PagedWork& w, int split_tiles) { return w.tiles <= p.least ? 1 : paged_quotient(w.tiles - 1, split_tiles) + 1; }
// keys [k0, k1) of split i
template <int TILE> MI_PLAN_FN void paged_split_keys(const PagedSeq& s, const PagedWork& w, int splits, int i, int& k0, int& k1) {
    const int64_t per = (int64_t)(paged_quotient(w.tiles - 1, splits) + 1) * TILE;
    k0 = paged_clamp(per * i, 0, s.len);
    k1 = paged_clamp(per * i + per, 0, s.len);
}
// Of work that is not split: how many blocks of a sequence, the last ones, reach keys beyond x tiles (about: by the tokens that whole blocks have); all for x < 0.
// The order of blocks is by the most x that they reach beyond, longest first, so that no long one starts when others are done.
template <int BLOCK, int TILE> MI_PLAN_FN int paged_above(const PagedSeq& s, const PagedWork& w, int n_rep, bool causal, int x) {
    if (x < 0) return w.blocks;
    if ((int64_t)x * TILE >= s.len) return 0;
    const int64_t over = (int64_t)x * TILE - ((int64_t)s.ctx - s.n);      // keys of new tokens below
    if (!causal || over <= 0) return w.blocks;
    const int64_t below = over * n_rep / BLOCK;
    return below >= w.blocks ? 0 : w.blocks - (int)below;
}
// Whether a launch computes a sequence whose first slot and first partial result are these: all of its splits or none.
MI_PLAN_FN bool paged_fits(const PagedPlan& p, const PagedWork& w, int splits, int slot, int partial) {
    const int64_t n = (int64_t)w.blocks * splits;
    return slot >= 0 && slot + n <= p.max_slots && (splits == 1 || (partial >= 0 && partial + n <= p.max_partials));
}

// Upper bounds for the host: blocks of rows that `tokens` tokens of `batch` sequences make, at most max_q_len of them in one; workgroups per KV head; and
// partial results per KV head, of sequences of up to max_tiles tiles.
template <int BLOCK> MI_PLAN_FN int64_t paged_max_blocks(const PagedPlan& p, int64_t tokens, int64_t batch, int64_t max_q_len, int n_rep) {
    int64_t rows = max_q_len * n_rep;                       // of one sequence
    if (rows <= p.rows_over) return 0;
    if (rows > p.rows_up_to) rows = p.rows_up_to;
    const int64_t each = (rows + BLOCK - 1) / BLOCK * batch;
    const int64_t least = (int64_t)p.rows_over + 1;         // rows of a sequence that is this kernel's
    const int64_t sequences = tokens * n_rep / least < batch ? tokens * n_rep / least : batch;
    const int64_t together = tokens * n_rep / BLOCK + sequences;
    return each < together ? each : together;
}
MI_PLAN_FN int64_t paged_max_slots(const PagedPlan& p, int64_t blocks, int64_t max_tiles) {
    const int64_t each = blocks * max_tiles, together = paged_few(p, blocks) ? p.fit : blocks + p.share + 1;
    return p.share == 0 || blocks == 0 ? blocks : each < together ? each : together;
}
// blocks of sequences with more than one split
MI_PLAN_FN int64_t paged_max_split_blocks(const PagedPlan& p, int64_t blocks) { return p.share == 0 ? 0 : blocks < p.share + 1 ? blocks : p.share + 1; }
MI_PLAN_FN int64_t paged_max_partials(const PagedPlan& p, int64_t blocks, int64_t max_tiles) {
    if (p.share == 0) return 0;
    const int64_t each = blocks * max_tiles, together = 2 * (int64_t)p.share + 2;
    return each < together ? each : together;
}

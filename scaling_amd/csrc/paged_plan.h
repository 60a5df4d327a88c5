// Who computes what in attention over a paged cache: sequences, their key ranges and how their work is cut, from lengths that lie on the device.  Plain
// arithmetic, the same for every workgroup of a launch and for the launch that merges; compiles for the host alone too.
//
// A sequence's rows are (new token, query head of a group): token i of n and head r of n_rep make row i * n_rep + r, so all heads that share keys share a
// block of rows.  A kernel takes the sequences whose number of rows it suits, in blocks of `block_rows`, with keys in tiles of `tile_keys`.  Where blocks are
// few, the keys of a sequence are cut into splits of at most S tiles each, with S such that all splits together are about `target` workgroups:
//     W = sum over sequences of blocks * tiles (per KV head),   S = floor(W * nkv / target) + 1,   splits_b = ceil(tiles_b / S)
// Then splits of all blocks are at most target / nkv + blocks in number, and those of sequences with more than one split at most 2 * target / nkv (tiles > S
// gives ceil(tiles / S) < 2 tiles / S).  Lengths may be anything: sequences are clamped to the tokens and the page table that there are, and where lengths that
// overlap make more partial results than the workspace holds, those are left out.
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

struct PagedPlan {
    int rows_over, rows_up_to;    // sequences with more than rows_over and at most rows_up_to rows
    int block_rows, tile_keys;
    int target;                   // workgroups aimed at; 0: never split
    int nkv;
};

struct PagedWork {
    int blocks, tiles;            // blocks 0: not this kernel's
};
MI_PLAN_FN PagedWork paged_work(const PagedPlan& p, const PagedSeq& s, int n_rep) {
    const int64_t rows = (int64_t)s.n * n_rep;
    PagedWork w;
    w.blocks = rows > p.rows_over && rows <= p.rows_up_to ? (int)((rows + p.block_rows - 1) / p.block_rows) : 0;
    w.tiles = s.len > 0 ? (int)(((int64_t)s.len + p.tile_keys - 1) / p.tile_keys) : 1;      // rows without keys are written too
    return w;
}
// tiles of a split; `units` is W
MI_PLAN_FN int paged_split_tiles(const PagedPlan& p, int64_t units) { return p.target > 0 ? paged_clamp(units * p.nkv / p.target + 1, 1, 0x7fffffff) : 0x7fffffff; }
MI_PLAN_FN int paged_splits(const PagedWork& w, int split_tiles) { return (w.tiles - 1) / split_tiles + 1; }
// keys [k0, k1) of split i
MI_PLAN_FN void paged_split_keys(const PagedPlan& p, const PagedSeq& s, const PagedWork& w, int splits, int i, int& k0, int& k1) {
    const int64_t per = (int64_t)((w.tiles + splits - 1) / splits) * p.tile_keys;
    const int64_t a = per * i, b = a + per;
    k0 = a < s.len ? (int)a : s.len;
    k1 = b < s.len ? (int)b : s.len;
}

// Upper bounds for the host: blocks of rows that `tokens` tokens of `batch` sequences make, at most max_q_len of them in one; workgroups per KV head; and
// partial results per KV head.
MI_PLAN_FN int64_t paged_max_blocks(const PagedPlan& p, int64_t tokens, int64_t batch, int64_t max_q_len, int n_rep) {
    int64_t rows = max_q_len * n_rep;                       // of one sequence
    if (rows <= p.rows_over) return 0;
    if (rows > p.rows_up_to) rows = p.rows_up_to;
    const int64_t each = (rows + p.block_rows - 1) / p.block_rows * batch;
    const int64_t least = (int64_t)p.rows_over + 1;         // rows of a sequence that is this kernel's
    const int64_t sequences = tokens * n_rep / least < batch ? tokens * n_rep / least : batch;
    const int64_t together = tokens * n_rep / p.block_rows + sequences;
    return each < together ? each : together;
}
MI_PLAN_FN int64_t paged_max_slots(const PagedPlan& p, int64_t blocks) { return blocks == 0 ? 0 : blocks + (p.target > 0 ? p.target / p.nkv + 1 : 0); }
MI_PLAN_FN int64_t paged_max_partials(const PagedPlan& p) { return p.target > 0 ? 2 * (int64_t)p.target / p.nkv + 2 : 0; }

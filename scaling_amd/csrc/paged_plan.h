// Who computes what in attention over a paged cache: sequences, their key ranges and how their work is cut, from lengths that lie on the device.  Plain
// arithmetic, the same for every workgroup of a launch and for the launch that merges; compiles for the host alone too.
//
// A sequence's rows are (new token, query head of a group): token i of n and head r of n_rep make row i * n_rep + r, so all heads that share keys share a
// block of rows.  A kernel takes the sequences whose number of rows it suits, in blocks of rows, with keys in tiles.  The keys of a sequence are cut into
// splits of at most S tiles each, with S such that all splits together are about `share` workgroups per KV head:
//     W = sum over sequences of blocks * tiles,   S = floor(W / share) + 1,   splits_b = ceil(tiles_b / S), of short sequences 1
// Then splits of all blocks are at most share + blocks in number, and those of sequences with more than one split at most 2 * share (tiles > S gives
// ceil(tiles / S) < 2 tiles / S).  Lengths may be anything: sequences are clamped to the tokens and the page table that there are, and where lengths that
// overlap make more workgroups or partial results than there are, what is too many is left out (of work that is split: sequences as a whole).
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

// a / b, of a q that is off by at most 2
MI_PLAN_FN int paged_corrected(int a, int b, int q) {
    int r = a - q * b;
    for (int i = 0; i < 2; ++i) {
        const int by = r < 0 ? -1 : r >= b ? 1 : 0;
        q += by;
        r -= by * b;
    }
    return q;
}
// a / b for a < 2^24, 0 < b, by a reciprocal and corrections (the compiler's division is five times as long, and a workgroup's first steps wait for it)
MI_PLAN_FN int paged_quotient(int a, int b) {
#ifdef __HIP_DEVICE_COMPILE__
    return paged_corrected(a, b, (int)((float)a * __builtin_amdgcn_rcpf((float)b)));      // two units in the last place of up to 24 bits
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
// u / share for u < 2^31: with m = 2^32 / share + 1 (of a share of 1: 0) the high half of a product is the quotient or one more
MI_PLAN_FN int paged_by_share(const PagedPlan& p, uint32_t u, uint32_t m) {
    const uint32_t q = (uint32_t)((uint64_t)u * m >> 32);
    return (int)(m == 0 ? u : q * (uint32_t)p.share > u ? q - 1 : q);
}

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
MI_PLAN_FN int paged_split_tiles(const PagedPlan& p, int64_t units, int64_t blocks, int most, uint32_t share_m) {
    return paged_by_share(p, paged_units(p, units, blocks, most), share_m) + 1;
}
MI_PLAN_FN int paged_split_tiles(const PagedPlan& p, int64_t units, int64_t blocks, int most) {
    if (p.share == 0) return 0x1000000;                    // no sequence has more
    return paged_split_tiles(p, units, blocks, most, p.share > 1 ? (uint32_t)((1ull << 32) / (uint32_t)p.share + 1) : 0);
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
// kept: a single split has a partial result too.
MI_PLAN_FN bool paged_fits(const PagedPlan& p, const PagedWork& w, int splits, int slot, int partial, bool kept = false) {
    const int64_t n = (int64_t)w.blocks * splits;
    return slot >= 0 && slot + n <= p.max_slots && ((splits == 1 && !kept) || (partial >= 0 && partial + n <= p.max_partials));
}

// A sequence as one workgroup meets it.
struct PagedFound {
    int b;             // -1: none
    int at;            // first slot of the sequence's blocks * splits; of split blocks the first of these; longest first: as if it were one
    int splits;
    int partial;       // first partial result of the sequence (splits > 1)
    PagedSeq seq;
    PagedWork work;
};
// What is looked for: a slot, i.e. one of the blocks * splits of a sequence; a slot, where nothing is split longest block first; or one of all blocks that
// have several splits.
enum PagedOrder { kSlots, kLongestFirst, kSplitBlocks };

// The sequence that holds `wanted`.  share_m: of paged_by_share.  It is looked for in groups of 64 sequences, one to a lane of LANES (a wavefront, or an array), which has
//     look(base)          takes up sequences base .. base + 63; behind the last one they have no blocks
//     of(f), of(v, f)     f(sequence, work), f(work, v's) of every lane: a Value, of which two can be subtracted
//     total(v), most(v)   the sum (less than 2^32) and the maximum over the lanes
//     upto(v)             of every lane the sum over the lanes up to it
//     holder(v, upto, x)  of the lanes' parts laid end to end the lane that holds place x, or -1
//     value(v, l), seq(l), work(l) of lane l
template <int BLOCK, int TILE, PagedOrder ORDER, class LANES>
MI_PLAN_FN PagedFound paged_find(LANES& lanes, const PagedPlan& p, uint32_t share_m, int batch, int n_rep, bool causal, int wanted) {
    PagedFound f;
    f.b = -1;
    f.at = f.splits = f.partial = 0;
    f.seq = PagedSeq{0, 0, 0, 0};
    f.work = PagedWork{0, 0};
    const auto blocks_of = [](const PagedSeq&, const PagedWork& w) { return w.blocks; };
    if (ORDER == kLongestFirst && p.share == 0 && batch <= 64) {
        lanes.look(0);
        auto above_lo = lanes.of(blocks_of), above_hi = lanes.of([](const PagedSeq&, const PagedWork&) { return 0; });
        if (wanted >= lanes.total(above_lo)) return f;
        int lo = -1, hi = (lanes.most(lanes.of([](const PagedSeq& s, const PagedWork&) { return s.len; })) + TILE - 1) / TILE;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            const auto above = lanes.of([&](const PagedSeq& s, const PagedWork& w) { return paged_above<BLOCK, TILE>(s, w, n_rep, causal, mid); });
            if (lanes.total(above) > wanted) { lo = mid; above_lo = above; } else { hi = mid; above_hi = above; }
        }
        const auto width = above_lo - above_hi, upto = lanes.upto(width);
        const int in = wanted - (int)lanes.total(above_hi), l = lanes.holder(width, upto, in);
        f.b = l;
        f.splits = 1;
        f.seq = lanes.seq(l);
        f.work = lanes.work(l);
        f.at = wanted - (lanes.value(above_hi, l) + in - lanes.value(upto - width, l));        // the block, counted from the last one, is wanted - at
        return f;
    }
    int split_tiles = 0x1000000;                           // no sequence has more
    if (p.share > 0) {
        int64_t units = 0, blocks = 0, reached = 0;
        int most = 0;
        for (int base = 0; base < batch; base += 64) {
            lanes.look(base);
            units += lanes.total(lanes.of([](const PagedSeq&, const PagedWork& w) { return w.blocks * w.tiles; }));
            if (p.fit || p.even) {
                blocks += lanes.total(lanes.of(blocks_of));
                const int longest = lanes.most(lanes.of([](const PagedSeq&, const PagedWork& w) { return w.blocks > 0 ? w.tiles : 0; }));
                most = longest > most ? longest : most;
            }
            if (p.fit) reached += lanes.total(lanes.of([&](const PagedSeq& s, const PagedWork& w) { return paged_reached<TILE>(s, w, causal); }));
        }
        split_tiles = paged_split_tiles(p, units, blocks, most, share_m);
        if (paged_level(p, blocks, most, reached)) split_tiles = 0x1000000;
#ifdef __HIPCC__
#pragma unroll 1
#endif
        for (int step = 0; paged_few(p, blocks) && step <= kPagedSteps; ++step) {
            int64_t slots = 0;
            for (int base = 0; base < batch; base += 64) {
                if (batch > 64) lanes.look(base);
                slots += lanes.total(lanes.of([&](const PagedSeq&, const PagedWork& w) { return w.blocks * paged_splits(p, w, split_tiles); }));
            }
            if (slots <= p.fit) break;
            split_tiles = paged_next_tiles(p, split_tiles, units, blocks, slots, step);
        }
    }
    int slots = 0, partials = 0, split_blocks = 0;
    for (int base = 0; base < batch; base += 64) {
        if (batch > 64 || p.share == 0) lanes.look(base);
        const auto splits = lanes.of([&](const PagedSeq&, const PagedWork& w) { return paged_splits(p, w, split_tiles); });
        const auto n = lanes.of(splits, [](const PagedWork& w, int i) { return w.blocks * i; });
        const auto part = lanes.of(splits, [](const PagedWork& w, int i) { return i > 1 ? w.blocks * i : 0; });
        const auto split = lanes.of(splits, [](const PagedWork& w, int i) { return i > 1 ? w.blocks : 0; });
        // (all sums before they are asked for: none waits for another's)
        const auto n_upto = lanes.upto(n), part_upto = lanes.upto(part), split_upto = ORDER == kSplitBlocks ? lanes.upto(split) : split;
        const int l = ORDER == kSplitBlocks ? lanes.holder(split, split_upto, wanted - split_blocks) : lanes.holder(n, n_upto, wanted - slots);
        if (l >= 0) {
            const int slot = slots + lanes.value(n_upto - n, l);
            f.b = base + l;
            f.at = ORDER == kSplitBlocks ? split_blocks + lanes.value(split_upto - split, l) : slot;
            f.splits = lanes.value(splits, l);
            f.partial = partials + lanes.value(part_upto - part, l);
            f.seq = lanes.seq(l);
            f.work = lanes.work(l);
            if (!paged_fits(p, f.work, f.splits, slot, f.partial)) f.b = -1;
            return f;
        }
        slots += lanes.value(n_upto, 63);
        partials += lanes.value(part_upto, 63);
        if (ORDER == kSplitBlocks) split_blocks += lanes.value(split_upto, 63);
    }
    return f;
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

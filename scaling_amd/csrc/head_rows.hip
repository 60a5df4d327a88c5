// Rows of one head: norms of queries and keys over the head's features with the rotary embedding in the same pass (forward and backward), and the append
// of new tokens to a paged cache, which is the same pass with pages for its output and the values beside it.
//
//     xh = x * rsqrt(mean(x^2) + eps)   (layer norm: xh = (x - mean) * rsqrt(var + eps)),   n = xh * w (+ b),   y = R(position) n
//     backward:  dn = R^T dy,  dw = sum dn * xh,  db = sum dn,  g = dn * w,  dx = rstd * (g - xh * mean(g * xh) (- mean(g): layer norm))
//
// float32 from the load to the one rounding on the store: as a norm and a rotation of their own the row is rounded between the two.
// Bound by memory.  A row of 128 16-bit features is 256 bytes: eight lanes with two vectors each, placed so that a lane holds both features of every
// rotated pair (vector c of the first half of the rotated span and of the second), hence one pass, no LDS and three lane exchanges for a sum.
#include "common.h"

int mi_compute_units();

namespace {

constexpr int kBlock = 256;
constexpr int kMaxDim = 256;
constexpr int kGradBlocks = 1024;        // of the backward pass, each with partial sums of the weights' gradients

struct RowsOf {                          // of q, k or v: [token][head][feature]
    const void* x;
    void* out;
    const void* dy;                      // backward: `out` is dx
    const void* weight;                  // null: no norm
    const void* bias;
    int64_t xs_t, xs_h, os_t, os_h, ds_t, ds_h;
    int heads;
};

struct HeadParams {
    RowsOf rows[3];
    const void *cos, *sin;               // null: no rotation
    const int64_t* pos;
    int64_t n_tokens, table_rows;
    int per_item, head_blocks[3], blocks_all;     // heads of a work item, items per token of each tensor and of all
    uint32_t blocks_m;                   // for divide(): by blocks_all
    int dim, rot;
    bool layer_norm;
    int turn;
    float eps;
    // pages (append): rows[1] and rows[2] go there
    const int32_t *page_table, *cu, *ctx;
    int64_t table_stride, page_stride;
    int batch, n_pages, page, max_pages;
    uint32_t page_m;
    // backward: partial sums [block][dw, db][dim]
    float* partial;
    int blocks_q, blocks_k;
    uint32_t heads_q_m, heads_k_m;
};

template <typename T, int VW, bool NT> __device__ __forceinline__ void store_vec(T* p, const float* f) {
    if constexpr (VW * sizeof(T) == 16) {
        if constexpr (NT) stg_nt(reinterpret_cast<uint4*>(p), Elem<T>::pack(f));
        else *reinterpret_cast<uint4*>(p) = Elem<T>::pack(f);
    } else {
        Elem<T>::store1(p, *f);
    }
}
// What turns a slot's features: rotate-half with tables of the rows' type or float32, or neighbouring pairs (of single elements: the slot's two).
enum Turn { kHalf, kHalfF32, kPairs };

// The two vectors of slot s.  Slots below `pairs` hold vector s of either half of the rotated span, the others neighbours.
struct Slot {
    int a, b;
    bool has_a, has_b, half;
};
template <int VW, int TURN> __device__ __forceinline__ Slot slot_of(const HeadParams& p, int s) {
    const int n_pair = TURN != kPairs && p.cos != nullptr ? p.rot / 2 / VW : 0, n = p.dim / VW;
    Slot o;
    o.half = s < n_pair;
    o.a = o.half ? s : 2 * s;
    o.b = o.half ? s + n_pair : 2 * s + 1;
    o.has_a = o.a < n;
    o.has_b = o.b < n;
    return o;
}

// Table values of a slot, as they lie in memory: cosines and sines of its two vectors (kPairs: one value per pair).
template <typename T, int VW, int TURN> struct Angles {
    using Table = std::conditional_t<TURN == kHalf, T, float>;
    static constexpr int N = TURN == kPairs ? (VW == 1 ? 1 : VW / 2) : VW;      // values per vector
    static constexpr bool kWhole = VW > 1;
    static constexpr int kVecs = (N * sizeof(Table) + 15) / 16;
    typedef float f32x2v __attribute__((ext_vector_type(2)));
    using Piece = std::conditional_t<!kWhole, float, std::conditional_t<N * sizeof(Table) == 8, f32x2v, uint4>>;
    Piece c[2][kVecs], s[2][kVecs];
    __device__ __forceinline__ void load(const HeadParams& p, const Slot& o, int64_t t) {
        const bool turned = p.cos != nullptr && (TURN == kPairs ? o.has_a : o.half);
        int64_t r = turned ? p.pos[t] : 0;
        r = r < 0 ? 0 : (r >= p.table_rows ? p.table_rows - 1 : r);
        const int64_t row = r * (TURN == kPairs ? p.dim / 2 : p.rot);
        const Table *cos = (const Table*)p.cos + row, *sin = (const Table*)p.sin + row;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int at = (v ? o.b : o.a) * VW / (TURN == kPairs ? 2 : 1);
            const bool there = turned && (v == 0 || (TURN == kPairs ? VW > 1 && o.has_b : true));
#pragma unroll
            for (int k = 0; k < kVecs; ++k) {
                c[v][k] = s[v][k] = Piece{};               // of features past the head or behind the rotated span
                if (!there) continue;
                if constexpr (kWhole) {
                    c[v][k] = reinterpret_cast<const Piece*>(cos + at)[k];
                    s[v][k] = reinterpret_cast<const Piece*>(sin + at)[k];
                } else {
                    c[v][k] = Elem<Table>::load1(cos + at);
                    s[v][k] = Elem<Table>::load1(sin + at);
                }
            }
        }
    }
    __device__ __forceinline__ static void unpack(const Piece (&x)[kVecs], float (&f)[N]) {
        if constexpr (!kWhole) f[0] = x[0];
        else if constexpr (sizeof(Piece) == 8) {
            f[0] = x[0][0];
            f[1] = x[0][1];
        } else {
#pragma unroll
            for (int k = 0; k < kVecs; ++k) Elem<Table>::unpack(x[k], f + k * (16 / (int)sizeof(Table)));
        }
    }
};
// a, b := R a, b, or with BACK its transpose
template <typename T, int VW, int TURN, bool BACK>
__device__ __forceinline__ void rotate(const HeadParams& p, const Slot& o, const Angles<T, VW, TURN>& w, float (&a)[VW], float (&b)[VW]) {
    if (p.cos == nullptr) return;
    constexpr float sign = BACK ? -1.f : 1.f;
    constexpr int N = Angles<T, VW, TURN>::N;
    float ca[N], sa[N], cb[N], sb[N];
    w.unpack(w.c[0], ca);
    w.unpack(w.s[0], sa);
    w.unpack(w.c[1], cb);
    w.unpack(w.s[1], sb);
    if constexpr (TURN == kPairs) {
        if constexpr (VW == 1) {
            rotate_complex_pair(a[0], b[0], ca[0], sign * sa[0]);
        } else {
#pragma unroll
            for (int i = 0; i < VW / 2; ++i) {
                rotate_complex_pair(a[2 * i], a[2 * i + 1], ca[i], sign * sa[i]);
                rotate_complex_pair(b[2 * i], b[2 * i + 1], cb[i], sign * sb[i]);
            }
        }
    } else if (o.half) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float x0 = a[i], x1 = b[i];
            a[i] = BACK ? x0 * ca[i] + x1 * sb[i] : x0 * ca[i] - x1 * sa[i];
            b[i] = BACK ? x1 * cb[i] - x0 * sa[i] : x1 * cb[i] + x0 * sb[i];
        }
    }
}

// a, b := xh of the row that L lanes hold in them; the reciprocal deviation
template <int VW, int L, int R>
__device__ __forceinline__ float normalise(const HeadParams& p, const Slot (&s)[R], float (&a)[R][VW], float (&b)[R][VW]) {
    const float inv = 1.0f / (float)p.dim;
    if (p.layer_norm) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < VW; ++i) sum += a[r][i] + b[r][i];
        const float mean = group_sum<L>(sum) * inv;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                a[r][i] = s[r].has_a ? a[r][i] - mean : 0.f;
                b[r][i] = s[r].has_b ? b[r][i] - mean : 0.f;
            }
    }
    float square = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < VW; ++i) square += a[r][i] * a[r][i] + b[r][i] * b[r][i];
    const float rstd = rsqrtf(group_sum<L>(square) * inv + p.eps);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            a[r][i] *= rstd;
            b[r][i] *= rstd;
        }
    return rstd;
}

// Offset of token t's row in the pages, or -1 where the cache has no place for it: behind the last sequence, a position outside the page table, a page
// outside the cache.  (Reads may be clamped, as the attention kernels clamp them; a write would land in somebody else's page.)
template <int L> __device__ __forceinline__ int64_t page_row(const HeadParams& p, int64_t t, int64_t token_stride) {
    // The sequence: by counting ends that lie at or before t, lane i holding the end of sequence i: one trip to memory.  Of more than 64 by halving, a trip
    // each.
    int lo = 0, end, ctx;
    if (p.batch <= 64) {
        const int i = min((int)(threadIdx.x & 63), p.batch - 1), ends = p.cu[i + 1], lengths = p.ctx[i];
        const bool counts = (int)(threadIdx.x & 63) < p.batch - 1;
#pragma unroll
        for (int g = 0; g < 64 / L; ++g) {                 // the items of the wavefront
            const int before = __popcll(__ballot(counts && ends <= __builtin_amdgcn_readlane((int)t, g * L)));
            lo = (int)(threadIdx.x & 63) / L == g ? before : lo;
        }
        end = __shfl(ends, lo);
        ctx = __shfl(lengths, lo);
    } else {
        int hi = p.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= t) lo = mid; else hi = mid;
        }
        end = p.cu[lo + 1];
        ctx = p.ctx[lo];
    }
    const int64_t first = p.cu[lo], at = (int64_t)ctx - end + t;
    if (t < first || t >= end || at < 0 || at >= (int64_t)p.max_pages * p.page) return -1;
    const int in_table = divide((uint32_t)at, p.page, p.page_m), page = p.page_table[(int64_t)lo * p.table_stride + in_table];
    if (page < 0 || page >= p.n_pages) return -1;
    return (int64_t)page * p.page_stride + (at - (int64_t)in_table * p.page) * token_stride;
}

// Two vectors of a row as they lie in memory.
template <typename T, int VW> struct Raw {
    static constexpr bool kWhole = VW * sizeof(T) == 16;
    std::conditional_t<kWhole, uint4, float> a, b;
    __device__ __forceinline__ void load(const T* x, const Slot& s) {
        if constexpr (kWhole) {
            a = s.has_a ? *reinterpret_cast<const uint4*>(x + s.a * VW) : make_uint4(0, 0, 0, 0);
            b = s.has_b ? *reinterpret_cast<const uint4*>(x + s.b * VW) : make_uint4(0, 0, 0, 0);
        } else {
            a = s.has_a ? Elem<T>::load1(x + s.a) : 0.f;
            b = s.has_b ? Elem<T>::load1(x + s.b) : 0.f;
        }
    }
    __device__ __forceinline__ void store(T* x, const Slot& s) const {
        if constexpr (kWhole) {
            if (s.has_a) *reinterpret_cast<uint4*>(x + s.a * VW) = a;
            if (s.has_b) *reinterpret_cast<uint4*>(x + s.b * VW) = b;
        } else {
            if (s.has_a) Elem<T>::store1(x + s.a, a);
            if (s.has_b) Elem<T>::store1(x + s.b, b);
        }
    }
    __device__ __forceinline__ void unpack(float (&fa)[VW], float (&fb)[VW]) const {
        if constexpr (kWhole) {
            Elem<T>::unpack(a, fa);
            Elem<T>::unpack(b, fb);
        } else {
            fa[0] = a;
            fb[0] = b;
        }
    }
};
// NT: past the caches (for rows of 8192 x 40 heads of 128: forward 31.1 -> 30.8 us, backward 52.0 -> 49.5; with loads past them too 57)
template <typename T, int VW, bool NT> __device__ __forceinline__ void store_row(T* out, const Slot& s, const float (&a)[VW], const float (&b)[VW]) {
    if (s.has_a) store_vec<T, VW, NT>(out + s.a * VW, a);
    if (s.has_b) store_vec<T, VW, NT>(out + s.b * VW, b);
}

// A work item: some heads of one tensor at one token.  Positions' angles and the weights are loaded once for all of them; row by row they were two thirds of
// what a lane loads.
struct Item {
    int which;          // tensor
    int64_t t;
    int h0, h1;
};
template <bool PAGED> __device__ __forceinline__ Item item_of(const HeadParams& p, uint32_t item) {
    Item o;
    const int t = divide(item, p.blocks_all, p.blocks_m);
    int block = (int)item - t * p.blocks_all;
    o.t = t;
    o.which = 0;
    int heads = p.rows[0].heads;
    if (block >= p.head_blocks[0]) {
        block -= p.head_blocks[0];
        o.which = 1;
        heads = p.rows[1].heads;
        if (PAGED && block >= p.head_blocks[1]) {
            block -= p.head_blocks[1];
            o.which = 2;
            heads = p.rows[2].heads;
        }
    }
    o.h0 = block * p.per_item;
    o.h1 = min(o.h0 + p.per_item, heads);
    return o;
}

// The tensor of an item, which differs from lane to lane: by selects of its fields (an index would put all three into scratch memory).
template <bool PAGED> __device__ __forceinline__ RowsOf rows_of(const HeadParams& p, int which) {
    const RowsOf &q = p.rows[0], &k = p.rows[1], &v = p.rows[2];
    const auto pick = [&](auto a, auto b, auto c) { return which == 0 ? a : PAGED && which == 2 ? c : b; };
    RowsOf o{};
    o.x = pick(q.x, k.x, v.x); o.out = pick(q.out, k.out, v.out); o.weight = pick(q.weight, k.weight, v.weight); o.bias = pick(q.bias, k.bias, v.bias);
    o.dy = pick(q.dy, k.dy, v.dy); o.ds_t = pick(q.ds_t, k.ds_t, v.ds_t); o.ds_h = pick(q.ds_h, k.ds_h, v.ds_h);
    o.xs_t = pick(q.xs_t, k.xs_t, v.xs_t); o.xs_h = pick(q.xs_h, k.xs_h, v.xs_h); o.os_t = pick(q.os_t, k.os_t, v.os_t); o.os_h = pick(q.os_h, k.os_h, v.os_h);
    return o;
}

// L lanes to a row, R slots to a lane
template <typename T, int VW, int L, int R, int TURN, bool PAGED>
__global__ __launch_bounds__(kBlock) void head_rows_kernel(const HeadParams p) {
    const int64_t last = p.n_tokens * p.blocks_all - 1, index = (int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L;
    if (!PAGED && index > last) return;                    // the same for the lanes of a row
    Item it = item_of<PAGED>(p, (uint32_t)(index < last ? index : last));
    if (index > last) it.h1 = it.h0;                       // nothing but a part in looking for places
    const RowsOf w = rows_of<PAGED>(p, it.which);
    const T* x = (const T*)w.x + it.t * w.xs_t;
    T* out = (T*)w.out;
    Slot s[R];
    Raw<T, VW> raw[R], next[R], weight[R], bias[R];
    Angles<T, VW, TURN> angles[R];
    const bool plain = PAGED && it.which == 2;             // values: copied
#pragma unroll
    for (int r = 0; r < R; ++r) {
        s[r] = slot_of<VW, TURN>(p, threadIdx.x % L + L * r);
        next[r].load(x + (int64_t)it.h0 * w.xs_h, s[r]);
        if (!plain) angles[r].load(p, s[r], it.t);
        if (w.weight != nullptr) weight[r].load((const T*)w.weight, s[r]);
        if (w.bias != nullptr) bias[r].load((const T*)w.bias, s[r]);
    }
    out += it.t * w.os_t;
    if constexpr (PAGED) {
        const int64_t at = page_row<L>(p, it.t, w.os_t);   // by all lanes together
        if (it.which != 0) {
            if (at < 0) return;
            out = (T*)w.out + at;
        }
    }
    for (int h = it.h0; h < it.h1; ++h) {
        float a[R][VW], b[R][VW];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            raw[r] = next[r];
            raw[r].unpack(a[r], b[r]);
        }
        if (h + 1 < it.h1) {
#pragma unroll
            for (int r = 0; r < R; ++r) next[r].load(x + (int64_t)(h + 1) * w.xs_h, s[r]);
        }
        if (plain) {
#pragma unroll
            for (int r = 0; r < R; ++r) raw[r].store(out + (int64_t)h * w.os_h, s[r]);
            continue;
        }
        if (w.weight != nullptr) {
            normalise<VW, L, R>(p, s, a, b);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float wa[VW], wb[VW], ba[VW] = {}, bb[VW] = {};
                weight[r].unpack(wa, wb);
                if (w.bias != nullptr) bias[r].unpack(ba, bb);
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    a[r][i] = a[r][i] * wa[i] + ba[i];
                    b[r][i] = b[r][i] * wb[i] + bb[i];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            rotate<T, VW, TURN, false>(p, s[r], angles[r], a[r], b[r]);
            store_row<T, VW, !PAGED>(out + (int64_t)h * w.os_h, s[r], a[r], b[r]);
        }
    }
}

// Items of q (the first blocks_q workgroups) or k, a workgroup's in steps of all workgroups of its tensor; partial sums of dw and db per workgroup.
template <typename T, int VW, int L, int R, int TURN, bool LAYER>
__global__ __launch_bounds__(kBlock) void head_rows_grad_kernel(const HeadParams p) {
    constexpr int kWaves = kBlock / 64, kItems = kBlock / L;
    __shared__ float sums[kWaves][2][kMaxDim];
    const bool is_k = (int)blockIdx.x >= p.blocks_q;
    const RowsOf& w = is_k ? p.rows[1] : p.rows[0];
    const int block = blockIdx.x - (is_k ? p.blocks_q : 0), blocks = is_k ? p.blocks_k : p.blocks_q;
    const int head_blocks = is_k ? p.head_blocks[1] : p.head_blocks[0];
    const uint32_t blocks_m = is_k ? p.heads_k_m : p.heads_q_m;
    const int64_t n_items = p.n_tokens * head_blocks;
    Slot s[R];
    Raw<T, VW> weight[R];
    float dwa[R][VW], dwb[R][VW], dba[R][VW], dbb[R][VW];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        s[r] = slot_of<VW, TURN>(p, threadIdx.x % L + L * r);
        weight[r].load((const T*)w.weight, s[r]);
#pragma unroll
        for (int i = 0; i < VW; ++i) dwa[r][i] = dwb[r][i] = dba[r][i] = dbb[r][i] = 0.f;
    }
    const float inv = 1.0f / (float)p.dim;
    for (int64_t index = (int64_t)block * kItems + threadIdx.x / L; index < n_items; index += (int64_t)blocks * kItems) {
        const int64_t t = divide((uint32_t)index, head_blocks, blocks_m);
        const int h0 = ((int)index - (int)t * head_blocks) * p.per_item, h1 = min(h0 + p.per_item, w.heads);
        const T *x = (const T*)w.x + t * w.xs_t, *dy = (const T*)w.dy + t * w.ds_t;
        T* out = (T*)w.out + t * w.os_t;
        Raw<T, VW> raw[R], draw[R];
        Angles<T, VW, TURN> angles[R];
        const auto request = [&](int h) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                raw[r].load(x + (int64_t)h * w.xs_h, s[r]);
                draw[r].load(dy + (int64_t)h * w.ds_h, s[r]);
            }
        };
        request(h0);
#pragma unroll
        for (int r = 0; r < R; ++r) angles[r].load(p, s[r], t);
        for (int h = h0; h < h1; ++h) {
            float a[R][VW], b[R][VW], da[R][VW], db[R][VW];
            float dot = 0.f, sum = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                raw[r].unpack(a[r], b[r]);
                draw[r].unpack(da[r], db[r]);
            }
            if (h + 1 < h1) request(h + 1);
            const float rstd = normalise<VW, L, R>(p, s, a, b);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float wa[VW], wb[VW];
                weight[r].unpack(wa, wb);
                rotate<T, VW, TURN, true>(p, s[r], angles[r], da[r], db[r]);
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    dwa[r][i] += da[r][i] * a[r][i];
                    dwb[r][i] += db[r][i] * b[r][i];
                    if constexpr (LAYER) {
                        dba[r][i] += da[r][i];
                        dbb[r][i] += db[r][i];
                    }
                    da[r][i] *= wa[i];
                    db[r][i] *= wb[i];
                    dot += da[r][i] * a[r][i] + db[r][i] * b[r][i];
                    if constexpr (LAYER) sum += da[r][i] + db[r][i];
                }
            }
            dot = group_sum<L>(dot) * inv;
            if constexpr (LAYER) sum = group_sum<L>(sum) * inv;
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    da[r][i] = rstd * (da[r][i] - a[r][i] * dot - sum);
                    db[r][i] = rstd * (db[r][i] - b[r][i] * dot - sum);
                }
                store_row<T, VW, true>(out + (int64_t)h * w.os_h, s[r], da[r], db[r]);
            }
        }
    }
    // lanes L, 2 L, ... further on hold the same features; then the wavefronts, in order
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const auto across = [](float v) {
#pragma unroll
        for (int m = L; m < 64; m *= 2) v += __shfl_xor(v, m);
        return v;
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float va = across(dwa[r][i]), vb = across(dwb[r][i]);
            if (lane < L && s[r].has_a) sums[wave][0][s[r].a * VW + i] = va;
            if (lane < L && s[r].has_b) sums[wave][0][s[r].b * VW + i] = vb;
            if constexpr (LAYER) {
                const float ua = across(dba[r][i]), ub = across(dbb[r][i]);
                if (lane < L && s[r].has_a) sums[wave][1][s[r].a * VW + i] = ua;
                if (lane < L && s[r].has_b) sums[wave][1][s[r].b * VW + i] = ub;
            }
        }
    __syncthreads();
    for (int f = threadIdx.x; f < (LAYER ? 2 : 1) * p.dim; f += kBlock) {
        const int which = f >= p.dim, i = f - which * p.dim;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v += sums[k][which][i];
        p.partial[((int64_t)blockIdx.x * 2 + which) * p.dim + i] = v;
    }
}

// The partial sums of a tensor's workgroups, in a fixed order: 64 chains of them per feature, then the chains.
struct SumParams {
    const float* partial;
    void* out[4];                        // dw, db of q, then of k; null: not wanted
    int first[2], count[2], dim;
};
template <typename T> __global__ __launch_bounds__(1024) void head_rows_sum_kernel(const SumParams p) {
    constexpr int kChains = 64, kFeatures = 16;
    __shared__ float chains[kChains][kFeatures];
    const int f = blockIdx.x * kFeatures + threadIdx.x % kFeatures, chain = threadIdx.x / kFeatures, which = blockIdx.y & 1, tensor = blockIdx.y >> 1;
    T* out = (T*)p.out[blockIdx.y];
    if (out == nullptr) return;
    float v = 0.f;
    if (f < p.dim) {
        const float* from = p.partial + ((int64_t)p.first[tensor] * 2 + which) * p.dim + f;
        const int n = p.count[tensor];
        constexpr int kStep = 8;
        for (int i0 = chain; i0 < n; i0 += kChains * kStep) {
            float x[kStep];
#pragma unroll
            for (int i = 0; i < kStep; ++i) x[i] = i0 + i * kChains < n ? from[(int64_t)(i0 + i * kChains) * 2 * p.dim] : 0.f;
#pragma unroll
            for (int i = 0; i < kStep; ++i) v += x[i];
        }
    }
    chains[chain][threadIdx.x % kFeatures] = v;
    __syncthreads();
    if (chain != 0 || f >= p.dim) return;
    v = 0.f;
#pragma unroll 8
    for (int i = 0; i < kChains; ++i) v += chains[i][threadIdx.x];
    Elem<T>::store1(out + f, v);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------------
// f(lanes, turn, ...) of rows taken in whole vectors, lanes the power of two that covers dim / (2 vector) slots; or element by element
template <typename T, typename F> void with_shape(const HeadParams& p, bool whole, const F& f) {
    using std::integral_constant;
    constexpr int V = Elem<T>::kVec, kLeast = sizeof(T) == 2 ? 4 : 8;          // 16-bit heads up to 64, 128, 256; float32 the same
    const auto shape = [&](auto turn) {
        const auto one = integral_constant<int, 1>{};
        const auto vec = integral_constant<int, V>{};
        const int slots = (p.dim / V + 1) / 2;
        if (!whole) f(one, integral_constant<int, 64>{}, integral_constant<int, kMaxDim / 128>{}, turn);
        else if (slots <= kLeast) f(vec, integral_constant<int, kLeast>{}, one, turn);
        else if (slots <= 2 * kLeast) f(vec, integral_constant<int, 2 * kLeast>{}, one, turn);
        else f(vec, integral_constant<int, 4 * kLeast>{}, one, turn);
    };
    if (p.turn == kPairs) shape(integral_constant<int, kPairs>{});
    else if (p.turn == kHalf) shape(integral_constant<int, kHalf>{});
    else if constexpr (sizeof(T) == 2) shape(integral_constant<int, kHalfF32>{});
}

// whether every row, table row and weight is whole 16-byte vectors, the halves of the rotated span too
template <typename T> bool whole(const HeadParams& p, bool grad) {
    constexpr int V = Elem<T>::kVec;
    if (p.dim % V != 0 || (p.cos != nullptr && p.turn != kPairs && p.rot / 2 % V != 0)) return false;
    if (p.cos != nullptr && (!mi_aligned16(p.cos) || !mi_aligned16(p.sin) || p.rot % 4 != 0 || (p.turn == kPairs && p.dim % 8 != 0))) return false;
    for (const RowsOf& r : p.rows) {
        if (r.heads == 0) continue;
        if (!mi_aligned16(r.x) || !mi_aligned16(r.out) || !mi_aligned16(r.weight) || !mi_aligned16(r.bias) || r.xs_t % V || r.xs_h % V || r.os_t % V || r.os_h % V)
            return false;
        if (grad && (!mi_aligned16(r.dy) || r.ds_t % V || r.ds_h % V)) return false;
    }
    return p.page_stride % V == 0;
}

// rows of the arguments' tensors, but for where they go
int fill(const mi_norm_rotary_args* a, const char* who, HeadParams& p) {
    if (a->n_tokens < 0 || a->n_q_heads < 0 || a->n_kv_heads < 0 || a->n_q_heads + (int64_t)a->n_kv_heads == 0 || a->head_dim <= 0 || a->head_dim > kMaxDim)
        return mi_fail(MI_E_SHAPE, "%s: %lld tokens, %d and %d heads of %d features (1 to %d)", who, (long long)a->n_tokens, a->n_q_heads, a->n_kv_heads, a->head_dim, kMaxDim);
    if (a->n_tokens * (a->n_q_heads + 2 * (int64_t)a->n_kv_heads) > 0x7fffffffLL || a->n_q_heads + 2 * (int64_t)a->n_kv_heads > 0xffff)
        return mi_fail(MI_E_SHAPE, "%s: more than 2^31 rows or 65535 heads", who);
    if (a->dtype != MI_BF16 && a->dtype != MI_F16 && a->dtype != MI_F32) return mi_fail(MI_E_DTYPE, "%s: unsupported dtype code %d", who, a->dtype);
    if ((a->n_q_heads > 0 && !a->q) || (a->n_kv_heads > 0 && !a->k)) return mi_fail(MI_E_NULL, "%s: null pointer", who);
    if (a->eps < 0.f || mi_is_nan(a->eps)) return mi_fail(MI_E_SHAPE, "%s: eps must not be negative", who);
    if (!a->layer_norm && (a->q_bias || a->k_bias)) return mi_fail(MI_E_SHAPE, "%s: RMSNorm has no bias", who);
    const bool rotary = a->rotary_cos != nullptr || a->rotary_sin != nullptr;
    if (rotary) {
        if (!a->rotary_cos || !a->rotary_sin || !a->position_ids) return mi_fail(MI_E_NULL, "%s: a rotation needs cos, sin and position ids", who);
        if (a->table_rows <= 0 || a->rot_dim <= 1 || a->rot_dim > a->head_dim || (a->rot_dim & 1)) return mi_fail(MI_E_SHAPE, "%s: %d rotated features of %d, %lld table rows", who, a->rot_dim, a->head_dim, (long long)a->table_rows);
        if (a->rotary_interleaved && (a->rot_dim != a->head_dim || a->table_dtype != MI_F32))
            return mi_fail(MI_E_SHAPE, "%s: interleaved pairs cover the head, with fp32 tables", who);
        if (a->table_dtype != a->dtype && a->table_dtype != MI_F32) return mi_fail(MI_E_DTYPE, "%s: table dtype must equal the data dtype or be fp32", who);
    }
    p.rows[0] = RowsOf{a->q, a->q_out, nullptr, a->q_weight, a->q_bias, a->q_stride_token, a->q_stride_head, a->q_out_stride_token, a->q_out_stride_head, 0, 0, a->n_q_heads};
    p.rows[1] = RowsOf{a->k, a->k_out, nullptr, a->k_weight, a->k_bias, a->k_stride_token, a->k_stride_head, a->k_out_stride_token, a->k_out_stride_head, 0, 0, a->n_kv_heads};
    if (rotary) {
        p.cos = a->rotary_cos; p.sin = a->rotary_sin; p.pos = a->position_ids; p.table_rows = a->table_rows;
        p.rot = a->rot_dim; p.turn = a->rotary_interleaved ? kPairs : a->table_dtype == a->dtype ? kHalf : kHalfF32;
    }
    p.n_tokens = a->n_tokens; p.dim = a->head_dim; p.layer_norm = a->layer_norm != 0; p.eps = a->eps;
    return MI_OK;
}

// Heads of a work item: as many (up to 4) as leave every compute unit 8 wavefronts.  (8192 x 40 heads of 128, forward / backward with 1, 2, 4, 8, 32 heads to an
// item: 58.8 / 110.6, 33.0 / 55.8, 31.2 / 51.9, 33.5 / 55.8, 33.7 / 55.9 us.)
constexpr int kHeadsPerItem = 4;
void set_items(HeadParams& p, int lanes) {
    const int64_t groups = (int64_t)mi_compute_units() * 8 * 64 / lanes;
    const int64_t rows = p.n_tokens * (p.rows[0].heads + p.rows[1].heads + p.rows[2].heads);
    int n = kHeadsPerItem;
    while (n > 1 && rows < groups * n) n /= 2;
    p.per_item = n;
    p.blocks_all = 0;
    for (int i = 0; i < 3; ++i) {
        p.head_blocks[i] = (p.rows[i].heads + n - 1) / n;
        p.blocks_all += p.head_blocks[i];
    }
    p.blocks_m = divide_m(p.blocks_all);
}

template <bool PAGED> int launch_rows(HeadParams& p, int dtype, const char* who, hipStream_t st) {
    MI_DISPATCH_DTYPE(dtype, {
        if constexpr (PAGED && sizeof(T) == 4) {
            return mi_fail(MI_E_DTYPE, "%s: the caches hold bf16 or f16 elements", who);
        } else {
            with_shape<T>(p, whole<T>(p, false), [&](auto vec, auto lanes, auto slots, auto turn) {
                constexpr int VW = decltype(vec)::value, L = decltype(lanes)::value, R = decltype(slots)::value, TURN = decltype(turn)::value;
                set_items(p, L);
                const dim3 grid((unsigned)((p.n_tokens * p.blocks_all + kBlock / L - 1) / (kBlock / L)));
                head_rows_kernel<T, VW, L, R, TURN, PAGED><<<grid, dim3(kBlock), 0, st>>>(p);
            });
        }
    });
    return mi_check_launch(who);
}

}  // namespace

extern "C" int mi_norm_rotary_fwd(const mi_norm_rotary_args* a) {
    if (!a) return mi_fail(MI_E_NULL, "norm_rotary: args is null");
    if (a->n_tokens == 0) return MI_OK;                    // an empty tensor may come with a null pointer
    HeadParams p{};
    if (const int rc = fill(a, "norm_rotary", p); rc != MI_OK) return rc;
    if ((a->n_q_heads > 0 && (!a->q_out || !a->q_weight)) || (a->n_kv_heads > 0 && (!a->k_out || !a->k_weight))) return mi_fail(MI_E_NULL, "norm_rotary: null pointer");
    return launch_rows<false>(p, a->dtype, "norm_rotary", (hipStream_t)a->stream);
}

extern "C" size_t mi_norm_rotary_bwd_workspace_bytes(int32_t head_dim) {
    return head_dim <= 0 ? 0 : (size_t)kGradBlocks * 2 * head_dim * sizeof(float);
}

extern "C" int mi_norm_rotary_bwd(const mi_norm_rotary_bwd_args* b) {
    if (!b) return mi_fail(MI_E_NULL, "norm_rotary_bwd: args is null");
    const mi_norm_rotary_args* a = &b->fwd;
    HeadParams p{};
    if (const int rc = fill(a, "norm_rotary_bwd", p); rc != MI_OK) return rc;
    if (a->n_tokens == 0) return mi_fail(MI_E_SHAPE, "norm_rotary_bwd: no tokens");
    if ((a->n_q_heads > 0 && (!b->d_q_out || !b->dq || !a->q_weight)) || (a->n_kv_heads > 0 && (!b->d_k_out || !b->dk || !a->k_weight)))
        return mi_fail(MI_E_NULL, "norm_rotary_bwd: null pointer");
    const size_t need = mi_norm_rotary_bwd_workspace_bytes(a->head_dim);
    if (!b->workspace || b->workspace_bytes < need || !mi_aligned16(b->workspace)) return mi_fail(MI_E_WORKSPACE, "norm_rotary_bwd: workspace needs %zu bytes (16-byte aligned), got %zu", need, b->workspace_bytes);
    RowsOf &q = p.rows[0], &k = p.rows[1];
    q.out = b->dq; q.dy = b->d_q_out; q.ds_t = b->d_q_out_stride_token; q.ds_h = b->d_q_out_stride_head; q.os_t = b->dq_stride_token; q.os_h = b->dq_stride_head;
    k.out = b->dk; k.dy = b->d_k_out; k.ds_t = b->d_k_out_stride_token; k.ds_h = b->d_k_out_stride_head; k.os_t = b->dk_stride_token; k.os_h = b->dk_stride_head;
    q.bias = k.bias = nullptr;                             // the gradients do not depend on it
    if (!p.layer_norm && (b->dq_bias || b->dk_bias)) return mi_fail(MI_E_SHAPE, "norm_rotary_bwd: RMSNorm has no bias");
    p.partial = (float*)b->workspace;
    const hipStream_t st = (hipStream_t)a->stream;
    // workgroups in proportion to the items, no more than have one each
    const auto split = [&](int lanes) {
        set_items(p, lanes);
        p.heads_q_m = divide_m(p.head_blocks[0]); p.heads_k_m = divide_m(p.head_blocks[1]);
        const int64_t rows_q = p.n_tokens * p.head_blocks[0], rows_k = p.n_tokens * p.head_blocks[1];
        const int64_t per = kBlock / lanes, all_q = (rows_q + per - 1) / per, all_k = (rows_k + per - 1) / per;
        p.blocks_q = (int)all_q; p.blocks_k = (int)all_k;
        if (all_q + all_k > kGradBlocks) {
            int64_t n = kGradBlocks * rows_q / (rows_q + rows_k);
            if (n < 1 && rows_q > 0) n = 1;
            if (n > kGradBlocks - 1 && rows_k > 0) n = kGradBlocks - 1;
            p.blocks_q = (int)n;
            p.blocks_k = kGradBlocks - (int)n;
        }
        return dim3((unsigned)(p.blocks_q + p.blocks_k));
    };
    MI_DISPATCH_DTYPE(a->dtype, {
        with_shape<T>(p, whole<T>(p, true), [&](auto vec, auto lanes, auto slots, auto turn) {
            constexpr int VW = decltype(vec)::value, L = decltype(lanes)::value, R = decltype(slots)::value, TURN = decltype(turn)::value;
            const dim3 grid = split(L);
            if (p.layer_norm) head_rows_grad_kernel<T, VW, L, R, TURN, true><<<grid, dim3(kBlock), 0, st>>>(p);
            else head_rows_grad_kernel<T, VW, L, R, TURN, false><<<grid, dim3(kBlock), 0, st>>>(p);
        });
        if (const int rc = mi_check_launch("norm_rotary_bwd"); rc != MI_OK) return rc;
        SumParams s{p.partial, {q.heads > 0 ? b->dq_weight : nullptr, q.heads > 0 ? b->dq_bias : nullptr, k.heads > 0 ? b->dk_weight : nullptr,
                                k.heads > 0 ? b->dk_bias : nullptr}, {0, p.blocks_q}, {p.blocks_q, p.blocks_k}, p.dim};
        head_rows_sum_kernel<T><<<dim3((unsigned)((p.dim + 15) / 16), 4), dim3(1024), 0, st>>>(s);
    });
    return mi_check_launch("norm_rotary_sum");
}

extern "C" int mi_paged_append(const mi_paged_append_args* b) {
    if (!b) return mi_fail(MI_E_NULL, "paged_append: args is null");
    const mi_norm_rotary_args* a = &b->rows;
    if (a->n_tokens == 0) return MI_OK;
    HeadParams p{};
    if (const int rc = fill(a, "paged_append", p); rc != MI_OK) return rc;
    if (a->n_kv_heads < 1 || b->batch < 1 || b->n_pages < 1 || b->max_pages < 1 || b->page_size < 16 || b->page_size % 16 != 0 ||
        (int64_t)b->max_pages * b->page_size > 0x7fffffffLL)
        return mi_fail(MI_E_SHAPE, "paged_append: %d kv heads, %d sequences, %d pages of %d tokens (a multiple of 16), up to %d a sequence", a->n_kv_heads, b->batch, b->n_pages, b->page_size, b->max_pages);
    if (!b->v || !b->k_pages || !b->v_pages || !b->page_table || !b->cu_seqlens || !b->ctx_len || (a->n_q_heads > 0 && !a->q_out))
        return mi_fail(MI_E_NULL, "paged_append: null pointer");
    if (!mi_aligned16(b->k_pages) || !mi_aligned16(b->v_pages) || b->page_stride % 8 || b->page_stride_token % 8 || b->page_stride_head % 8)
        return mi_fail(MI_E_ALIGN, "paged_append: pages must be 16-byte aligned with strides multiple of 8");
    p.rows[1].out = b->k_pages; p.rows[1].os_t = b->page_stride_token; p.rows[1].os_h = b->page_stride_head;
    p.rows[2] = RowsOf{b->v, b->v_pages, nullptr, nullptr, nullptr, b->v_stride_token, b->v_stride_head, b->page_stride_token, b->page_stride_head, 0, 0, a->n_kv_heads};
    p.page_table = b->page_table; p.cu = b->cu_seqlens; p.ctx = b->ctx_len; p.table_stride = b->page_table_stride; p.page_stride = b->page_stride;
    p.batch = b->batch; p.n_pages = b->n_pages; p.page = b->page_size; p.max_pages = b->max_pages; p.page_m = divide_m(b->page_size);
    return launch_rows<true>(p, a->dtype, "paged_append", (hipStream_t)a->stream);
}

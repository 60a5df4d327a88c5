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
    uint32_t heads_m;                    // for divide(): by the heads of all tensors
    int dim, rot;
    bool layer_norm, pairs, table_f32;
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

template <typename T, int VW> __device__ __forceinline__ void load_vec(const T* p, float* f) {
    if constexpr (VW * sizeof(T) == 16) Elem<T>::unpack(*reinterpret_cast<const uint4*>(p), f);
    else {
        static_assert(VW == 1, "whole vectors or single elements");
        *f = Elem<T>::load1(p);
    }
}
template <typename T, int VW> __device__ __forceinline__ void store_vec(T* p, const float* f) {
    if constexpr (VW * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = Elem<T>::pack(f);
    else Elem<T>::store1(p, *f);
}
// N values of a rotary table, of the rows' type or float32; vectors are 16-byte aligned either way
template <typename T, int N> __device__ __forceinline__ void load_table(const void* table, bool f32, int64_t at, float* f) {
    if (f32 || sizeof(T) == 4) {
        const float* p = (const float*)table + at;
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j) Elem<float>::unpack(reinterpret_cast<const uint4*>(p)[j], f + 4 * j);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = p[j];
        }
    } else if constexpr (sizeof(T) == 2) {
        if constexpr (N == 8) Elem<T>::unpack(*reinterpret_cast<const uint4*>((const T*)table + at), f);
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = Elem<T>::load1((const T*)table + at + j);
        }
    }
}

// The two vectors of slot s.  Slots below `pairs` hold vector s of either half of the rotated span, the others neighbours.
struct Slot {
    int a, b;
    bool has_a, has_b, half;
};
template <int VW> __device__ __forceinline__ Slot slot_of(const HeadParams& p, int s) {
    const int n_pair = p.cos != nullptr && !p.pairs ? p.rot / 2 / VW : 0, n = p.dim / VW;
    Slot o;
    o.half = s < n_pair;
    o.a = o.half ? s : 2 * s;
    o.b = o.half ? s + n_pair : 2 * s + 1;
    o.has_a = o.a < n;
    o.has_b = o.b < n;
    return o;
}

// sines and cosines of a slot's features
template <int VW> struct Angles {
    float ca[VW], sa[VW], cb[VW], sb[VW];
};
template <typename T, int VW> __device__ __forceinline__ void load_angles(const HeadParams& p, const Slot& s, int64_t t, Angles<VW>& o) {
#pragma unroll
    for (int i = 0; i < VW; ++i) o.ca[i] = o.sa[i] = o.cb[i] = o.sb[i] = 0.f;      // of features past the head: zeros stay zeros
    if (p.cos == nullptr || !s.has_a) return;
    int64_t r = p.pos[t];
    r = r < 0 ? 0 : (r >= p.table_rows ? p.table_rows - 1 : r);
    if (p.pairs) {
        constexpr int H = VW == 1 ? 1 : VW / 2;            // of single elements: the pair is (a, b)
        const int64_t at = r * (p.dim / 2) + (int64_t)s.a * VW / 2;
        load_table<float, H>(p.cos, true, at, o.ca);
        load_table<float, H>(p.sin, true, at, o.sa);
        if (VW > 1 && s.has_b) {
            load_table<float, H>(p.cos, true, at + H, o.cb);
            load_table<float, H>(p.sin, true, at + H, o.sb);
        }
    } else if (s.half) {
        const int64_t row = r * p.rot;
        load_table<T, VW>(p.cos, p.table_f32, row + s.a * VW, o.ca);
        load_table<T, VW>(p.sin, p.table_f32, row + s.a * VW, o.sa);
        load_table<T, VW>(p.cos, p.table_f32, row + s.b * VW, o.cb);
        load_table<T, VW>(p.sin, p.table_f32, row + s.b * VW, o.sb);
    }
}
// a, b := R a, b, or with BACK its transpose
template <int VW, bool BACK> __device__ __forceinline__ void rotate(const HeadParams& p, const Slot& s, const Angles<VW>& w, float* a, float* b) {
    if (p.cos == nullptr) return;
    constexpr float sign = BACK ? -1.f : 1.f;
    if (p.pairs) {
        if constexpr (VW == 1) {
            rotate_complex_pair(*a, *b, w.ca[0], sign * w.sa[0]);
        } else {
#pragma unroll
            for (int i = 0; i < VW / 2; ++i) {
                rotate_complex_pair(a[2 * i], a[2 * i + 1], w.ca[i], sign * w.sa[i]);
                rotate_complex_pair(b[2 * i], b[2 * i + 1], w.cb[i], sign * w.sb[i]);
            }
        }
    } else if (s.half) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float x0 = a[i], x1 = b[i];
            if constexpr (BACK) {
                a[i] = x0 * w.ca[i] + x1 * w.sb[i];
                b[i] = x1 * w.cb[i] - x0 * w.sa[i];
            } else {
                a[i] = x0 * w.ca[i] - x1 * w.sa[i];
                b[i] = x1 * w.cb[i] + x0 * w.sb[i];
            }
        }
    }
}

template <typename T, int VW, int R> __device__ __forceinline__ void load_row(const T* x, const Slot (&s)[R], float (&a)[R][VW], float (&b)[R][VW]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < VW; ++i) a[r][i] = b[r][i] = 0.f;
        if (s[r].has_a) load_vec<T, VW>(x + s[r].a * VW, a[r]);
        if (s[r].has_b) load_vec<T, VW>(x + s[r].b * VW, b[r]);
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
__device__ __forceinline__ int64_t page_row(const HeadParams& p, int64_t t, int64_t token_stride) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid] <= t) lo = mid; else hi = mid;
    }
    const int64_t first = p.cu[lo], end = p.cu[lo + 1], at = (int64_t)p.ctx[lo] - end + t;
    if (t < first || t >= end || at < 0 || at >= (int64_t)p.max_pages * p.page) return -1;
    const int in_table = divide((uint32_t)at, p.page, p.page_m), page = p.page_table[(int64_t)lo * p.table_stride + in_table];
    if (page < 0 || page >= p.n_pages) return -1;
    return (int64_t)page * p.page_stride + (at - (int64_t)in_table * p.page) * token_stride;
}

// The tensor of a row, which differs from lane to lane: by selects of its fields (an index would put all three into scratch memory).
template <bool PAGED> __device__ __forceinline__ RowsOf rows_of(const HeadParams& p, int which) {
    const RowsOf &q = p.rows[0], &k = p.rows[1], &v = p.rows[2];
    const auto pick = [&](auto a, auto b, auto c) { return which == 0 ? a : PAGED && which == 2 ? c : b; };
    RowsOf o{};
    o.x = pick(q.x, k.x, v.x); o.out = pick(q.out, k.out, v.out); o.weight = pick(q.weight, k.weight, v.weight); o.bias = pick(q.bias, k.bias, v.bias);
    o.xs_t = pick(q.xs_t, k.xs_t, v.xs_t); o.xs_h = pick(q.xs_h, k.xs_h, v.xs_h); o.os_t = pick(q.os_t, k.os_t, v.os_t); o.os_h = pick(q.os_h, k.os_h, v.os_h);
    return o;
}

// L lanes to a row, R slots to a lane
template <typename T, int VW, int L, int R, bool PAGED>
__global__ __launch_bounds__(kBlock) void head_rows_kernel(const HeadParams p) {
    const int heads = p.rows[0].heads + p.rows[1].heads + (PAGED ? p.rows[2].heads : 0);
    const int64_t row = (int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L;
    if (row >= p.n_tokens * heads) return;                 // the same for the lanes of a row
    const int64_t t = divide((uint32_t)row, heads, p.heads_m);
    int h = (int)(row - t * heads);
    int which = 0;
    if (h >= p.rows[0].heads) {
        h -= p.rows[0].heads;
        which = 1;
        if (PAGED && h >= p.rows[1].heads) {
            h -= p.rows[1].heads;
            which = 2;
        }
    }
    const RowsOf w = rows_of<PAGED>(p, which);
    const T* x = (const T*)w.x + t * w.xs_t + (int64_t)h * w.xs_h;
    Slot s[R];
    float a[R][VW], b[R][VW];
    Angles<VW> angles[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = slot_of<VW>(p, threadIdx.x % L + L * r);
    load_row<T, VW, R>(x, s, a, b);
    T* out = (T*)w.out;
    bool store = true;
    if (PAGED && which != 0) {
        const int64_t at = page_row(p, t, w.os_t);
        store = at >= 0;
        out += at + (int64_t)h * w.os_h;
    } else {
        out += t * w.os_t + (int64_t)h * w.os_h;
    }
    if (!PAGED || which != 2) {
#pragma unroll
        for (int r = 0; r < R; ++r) load_angles<T, VW>(p, s[r], t, angles[r]);
        if (w.weight != nullptr) {
            normalise<VW, L, R>(p, s, a, b);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float wa[VW], wb[VW], ba[VW] = {}, bb[VW] = {};
                if (s[r].has_a) load_vec<T, VW>((const T*)w.weight + s[r].a * VW, wa);
                if (s[r].has_b) load_vec<T, VW>((const T*)w.weight + s[r].b * VW, wb);
                if (w.bias != nullptr) {
                    if (s[r].has_a) load_vec<T, VW>((const T*)w.bias + s[r].a * VW, ba);
                    if (s[r].has_b) load_vec<T, VW>((const T*)w.bias + s[r].b * VW, bb);
                }
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    a[r][i] = a[r][i] * wa[i] + ba[i];
                    b[r][i] = b[r][i] * wb[i] + bb[i];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) rotate<VW, false>(p, s[r], angles[r], a[r], b[r]);
    }
    if (!store) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (s[r].has_a) store_vec<T, VW>(out + s[r].a * VW, a[r]);
        if (s[r].has_b) store_vec<T, VW>(out + s[r].b * VW, b[r]);
    }
}

// Rows of q (the first blocks_q workgroups) or k, a workgroup's in steps of all workgroups of its tensor; partial sums of dw and db per workgroup.
template <typename T, int VW, int L, int R>
__global__ __launch_bounds__(kBlock) void head_rows_grad_kernel(const HeadParams p) {
    constexpr int kWaves = kBlock / 64, kRows = kBlock / L;
    __shared__ float sums[kWaves][2][kMaxDim];
    const bool is_k = (int)blockIdx.x >= p.blocks_q;
    const RowsOf& w = is_k ? p.rows[1] : p.rows[0];
    const int block = blockIdx.x - (is_k ? p.blocks_q : 0), blocks = is_k ? p.blocks_k : p.blocks_q;
    const uint32_t heads_m = is_k ? p.heads_k_m : p.heads_q_m;
    const int64_t n_rows = p.n_tokens * w.heads;
    Slot s[R];
    float wa[R][VW], wb[R][VW], dwa[R][VW], dwb[R][VW], dba[R][VW], dbb[R][VW];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        s[r] = slot_of<VW>(p, threadIdx.x % L + L * r);
#pragma unroll
        for (int i = 0; i < VW; ++i) dwa[r][i] = dwb[r][i] = dba[r][i] = dbb[r][i] = 0.f;
    }
    load_row<T, VW, R>((const T*)w.weight, s, wa, wb);
    for (int64_t row = (int64_t)block * kRows + threadIdx.x / L; row < n_rows; row += (int64_t)blocks * kRows) {
        const int64_t t = divide((uint32_t)row, w.heads, heads_m);
        const int h = (int)(row - t * w.heads);
        float a[R][VW], b[R][VW], da[R][VW], db[R][VW];
        Angles<VW> angles[R];
        load_row<T, VW, R>((const T*)w.x + t * w.xs_t + (int64_t)h * w.xs_h, s, a, b);
        load_row<T, VW, R>((const T*)w.dy + t * w.ds_t + (int64_t)h * w.ds_h, s, da, db);
#pragma unroll
        for (int r = 0; r < R; ++r) load_angles<T, VW>(p, s[r], t, angles[r]);
        const float rstd = normalise<VW, L, R>(p, s, a, b);
        float dot = 0.f, sum = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            rotate<VW, true>(p, s[r], angles[r], da[r], db[r]);
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                dwa[r][i] += da[r][i] * a[r][i];
                dwb[r][i] += db[r][i] * b[r][i];
                dba[r][i] += da[r][i];
                dbb[r][i] += db[r][i];
                da[r][i] *= wa[r][i];
                db[r][i] *= wb[r][i];
                dot += da[r][i] * a[r][i] + db[r][i] * b[r][i];
                sum += da[r][i] + db[r][i];
            }
        }
        dot = group_sum<L>(dot) / (float)p.dim;
        sum = p.layer_norm ? group_sum<L>(sum) / (float)p.dim : 0.f;
        T* out = (T*)w.out + t * w.os_t + (int64_t)h * w.os_h;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                da[r][i] = rstd * (da[r][i] - a[r][i] * dot - sum);
                db[r][i] = rstd * (db[r][i] - b[r][i] * dot - sum);
            }
            if (s[r].has_a) store_vec<T, VW>(out + s[r].a * VW, da[r]);
            if (s[r].has_b) store_vec<T, VW>(out + s[r].b * VW, db[r]);
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
            const float va = across(dwa[r][i]), vb = across(dwb[r][i]), ua = across(dba[r][i]), ub = across(dbb[r][i]);
            if (lane < L && s[r].has_a) { sums[wave][0][s[r].a * VW + i] = va; sums[wave][1][s[r].a * VW + i] = ua; }
            if (lane < L && s[r].has_b) { sums[wave][0][s[r].b * VW + i] = vb; sums[wave][1][s[r].b * VW + i] = ub; }
        }
    __syncthreads();
    for (int f = threadIdx.x; f < 2 * p.dim; f += kBlock) {
        const int which = f >= p.dim, i = f - which * p.dim;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v += sums[k][which][i];
        p.partial[((int64_t)blockIdx.x * 2 + which) * p.dim + i] = v;
    }
}

// The partial sums of a tensor's workgroups, in a fixed order: 16 chains of them per feature, then the chains.
struct SumParams {
    const float* partial;
    void* out[4];                        // dw, db of q, then of k; null: not wanted
    int first[2], count[2], dim;
};
template <typename T> __global__ __launch_bounds__(1024) void head_rows_sum_kernel(const SumParams p) {
    __shared__ float chains[16][64];
    const int f = blockIdx.x * 64 + (threadIdx.x & 63), chain = threadIdx.x >> 6, which = blockIdx.y & 1, tensor = blockIdx.y >> 1;
    T* out = (T*)p.out[blockIdx.y];
    if (out == nullptr) return;
    float v = 0.f;
    if (f < p.dim) {
        const float* from = p.partial + ((int64_t)p.first[tensor] * 2 + which) * p.dim + f;
        for (int i = chain; i < p.count[tensor]; i += 16) v += from[(int64_t)i * 2 * p.dim];
    }
    chains[chain][threadIdx.x & 63] = v;
    __syncthreads();
    if (chain != 0 || f >= p.dim) return;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += chains[i][threadIdx.x];
    Elem<T>::store1(out + f, v);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------------
// lanes of a row: the power of two that covers dim / (2 VW) slots, 64 where rows are taken element by element
template <typename F> int with_lanes(int slots, const F& f) {
    if (slots <= 2) return f(std::integral_constant<int, 2>{});
    if (slots <= 4) return f(std::integral_constant<int, 4>{});
    if (slots <= 8) return f(std::integral_constant<int, 8>{});
    if (slots <= 16) return f(std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 32>{});
}

// whether every row, table row and weight is whole 16-byte vectors, the halves of the rotated span too
template <typename T> bool whole(const HeadParams& p, bool grad) {
    constexpr int V = Elem<T>::kVec;
    if (p.dim % V != 0 || (p.cos != nullptr && !p.pairs && p.rot / 2 % V != 0)) return false;
    if (p.cos != nullptr && (!mi_aligned16(p.cos) || !mi_aligned16(p.sin) || p.rot % 4 != 0 || (p.pairs && p.dim % 8 != 0))) return false;
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
        p.rot = a->rot_dim; p.pairs = a->rotary_interleaved != 0; p.table_f32 = a->table_dtype == MI_F32;
    }
    p.n_tokens = a->n_tokens; p.dim = a->head_dim; p.layer_norm = a->layer_norm != 0; p.eps = a->eps;
    return MI_OK;
}

template <bool PAGED> int launch_rows(HeadParams& p, int dtype, const char* who, hipStream_t st) {
    const int heads = p.rows[0].heads + p.rows[1].heads + p.rows[2].heads;
    p.heads_m = divide_m(heads);
    const int64_t rows = p.n_tokens * heads;
    MI_DISPATCH_DTYPE(dtype, {
        if constexpr (PAGED && sizeof(T) == 4) return mi_fail(MI_E_DTYPE, "%s: the caches hold bf16 or f16 elements", who);
        else {
        constexpr int V = Elem<T>::kVec;
        if (whole<T>(p, false)) {
            with_lanes((p.dim / V + 1) / 2, [&](auto lanes) {
                constexpr int L = decltype(lanes)::value;
                head_rows_kernel<T, V, L, 1, PAGED><<<dim3((unsigned)((rows + kBlock / L - 1) / (kBlock / L))), dim3(kBlock), 0, st>>>(p);
                return 0;
            });
        } else {
            head_rows_kernel<T, 1, 64, kMaxDim / 128, PAGED><<<dim3((unsigned)((rows + kBlock / 64 - 1) / (kBlock / 64))), dim3(kBlock), 0, st>>>(p);
        }
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
    p.heads_q_m = divide_m(q.heads); p.heads_k_m = divide_m(k.heads);
    p.partial = (float*)b->workspace;
    const hipStream_t st = (hipStream_t)a->stream;
    const int64_t rows_q = p.n_tokens * q.heads, rows_k = p.n_tokens * k.heads;
    // workgroups in proportion to the rows, no more than have one each
    const auto split = [&](int lanes) {
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
        constexpr int V = Elem<T>::kVec;
        if (whole<T>(p, true)) {
            with_lanes((p.dim / V + 1) / 2, [&](auto lanes) {
                constexpr int L = decltype(lanes)::value;
                const dim3 grid = split(L);
                head_rows_grad_kernel<T, V, L, 1><<<grid, dim3(kBlock), 0, st>>>(p);
                return 0;
            });
        } else {
            const dim3 grid = split(64);
            head_rows_grad_kernel<T, 1, 64, kMaxDim / 128><<<grid, dim3(kBlock), 0, st>>>(p);
        }
        if (const int rc = mi_check_launch("norm_rotary_bwd"); rc != MI_OK) return rc;
        SumParams s{p.partial, {q.heads > 0 ? b->dq_weight : nullptr, q.heads > 0 ? b->dq_bias : nullptr, k.heads > 0 ? b->dk_weight : nullptr,
                                k.heads > 0 ? b->dk_bias : nullptr}, {0, p.blocks_q}, {p.blocks_q, p.blocks_k}, p.dim};
        head_rows_sum_kernel<T><<<dim3((unsigned)((p.dim + 63) / 64), 4), dim3(1024), 0, st>>>(s);
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

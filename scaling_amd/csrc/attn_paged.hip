// Attention of ragged chunks of new tokens over a paged KV cache for gfx950.
//
// Two kernels share a call by the number of rows (new tokens x query heads of a group) of a sequence: `paged_rows` for up to kRowLimit of them (single
// tokens, drafts; more in small calls), bound by the cache's bytes, and `paged_tiles` for chunks, bound by the matrix pipe.  Either cuts its work by paged_plan.h, which every
// workgroup evaluates on the lengths by itself; partial results (running maximum, sum, unscaled output) of sequences with several splits go to the
// workspace and are merged by `paged_merge`.
//
// Pages hold a multiple of 16 keys, so 16 neighbouring keys (what one row of an MFMA operand tile, or one wavefront's share of a tile's direct loads, needs)
// have one page: its number is found once per 16 keys and wavefront, and a paged cache costs next to nothing against a contiguous one.
#include "attn_common.h"
#include "paged_plan.h"

#include <algorithm>

typedef float f32x4v __attribute__((ext_vector_type(4)));

namespace {

// Rows (tokens x query heads of a KV head) of a sequence up to which paged_rows computes it: one block, or two where items are few and none has more, so that
// paged_tiles is not launched.  (us, rows / tiles, 4 query heads to a KV head, d 128: 32 sequences of 5 tokens 123 / 157, of 9 tokens 215 / 170; 8 of
// 3 - 9 tokens 39.9 / 53; one of 16 tokens 15.8 / 20.7.  32 sequences of one token of 32 heads and one KV head: 28 / 27.)
constexpr int kRowBlock = 16;        // rows of a block, or twice as many where a sequence may have more
constexpr int kRowLimit = 32;
constexpr int kRowsAlone = 64;
// Where the page tables have no room for more keys, calls whose blocks all run at once are paged_rows' with any number of rows.  (us, tiles / rows: 128 tokens of 32 / 8 heads
// of 128 over 256 keys 16.9 / 11.8, 8 x 30 - 50 tokens of 16 / 4 heads of 64 over 300 keys 18.0 / 9.7; over 1000 keys 23.8 / 25.6 and 23.3 / 22.3.)
constexpr int kRowsAloneKeys = 512;
constexpr int kRowChunk = 32;        // keys per wavefront and step of paged_rows
constexpr int kRowWaves = 4;
constexpr int kRowTile = kRowChunk * kRowWaves;
constexpr int kTileRows = 256;
constexpr int kMergeMost = 4;        // workgroups of paged_merge with 16 rows each per compute unit, more than which take 32 each
constexpr int kTileKeys = 64;
constexpr float kRescaleGap = 8.0f;  // log2 units by which a row's maximum may lag before its output is rescaled

struct PagedParams {
    const elem_t *q, *kp, *vp;
    elem_t* o;
    const int32_t *table, *cu, *ctx;
    int64_t table_stride, q_st, q_sh, o_st, o_sh, p_sp, p_st, p_sh;
    int batch, total, n_pages, page, max_pages, capacity, nq, nkv, n_rep, causal;
    uint32_t page_m, rep_m, nkv_m, share_m[2];        // for divide(); share_m: of rows and tiles
    float scale_log2;
    PagedPlan rows, tiles;
    int tile_rows;                                    // rows kept per partial result of paged_tiles
    int32_t* tickets;                                 // nullable: arrivals of the splits of paged_rows, [partial][KV head], zero between launches
    float *rows_o, *rows_ml, *tiles_o, *tiles_ml;     // partial results: [partial][KV head][row of the block][feature], and (maximum in log2 units, sum)
};

__device__ __forceinline__ f32x4v mfma_16x16x32(elem8_t a, elem8_t b, f32x4v c) {
#ifdef MI_ELEM_F16
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#endif
}

// sums over lanes 0 .. this one
__device__ __forceinline__ int prefix_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr 1, 2, 4, 8, then the last lanes of the rows in front
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// The sequences of paged_find, lane by lane of a wavefront.  (Chunks that are not split, prompts of 2048 tokens, us by sequence and longest block first: 4, 16 heads
// of 64: 97, 74; 16 of 500 - 4096, 8 heads of 64: 458, 412.)
template <int BLOCK, int TILE> struct Wavefront {
    const PagedParams& p;
    const PagedPlan& plan;
    PagedSeq s;
    PagedWork w;
    __device__ __forceinline__ void look(int base) {
        const int b = base + (int)(threadIdx.x & 63), i = min(b, p.batch - 1);
        s = paged_seq(p.cu[i], p.cu[i + 1], p.ctx[i], p.total, p.capacity);
        w = paged_work<BLOCK, TILE>(plan, s, p.n_rep);
        if (b >= p.batch) w.blocks = s.n = 0;
    }
    template <class F> __device__ __forceinline__ int of(const F& f) const { return f(s, w); }
    template <class F> __device__ __forceinline__ int of(int v, const F& f) const { return f(w, v); }
    __device__ __forceinline__ int value(int v, int l) const { return __builtin_amdgcn_readlane(v, l); }
    __device__ __forceinline__ int64_t total(int v) const { return (int64_t)(uint32_t)value(prefix_sum(v), 63); }
    __device__ __forceinline__ int most(int v) const { return group_max<64>(v); }
    __device__ __forceinline__ int upto(int v) const { return prefix_sum(v); }
    __device__ __forceinline__ int holder(int v, int upto, int x) const {
        const uint64_t found = __ballot(x >= upto - v && x < upto);
        return found != 0 ? __builtin_ctzll(found) : -1;
    }
    __device__ __forceinline__ PagedSeq seq(int l) const { return PagedSeq{value(s.first, l), value(s.n, l), value(s.ctx, l), value(s.len, l)}; }
    __device__ __forceinline__ PagedWork work(int l) const { return PagedWork{value(w.blocks, l), value(w.tiles, l)}; }
};
template <int BLOCK, int TILE, PagedOrder ORDER> __device__ __forceinline__ PagedFound find_work(const PagedParams& p, const PagedPlan& plan, uint32_t share_m, int wanted) {
    Wavefront<BLOCK, TILE> lanes{p, plan, {}, {}};
    return paged_find<BLOCK, TILE, ORDER>(lanes, plan, share_m, p.batch, p.n_rep, p.causal, wanted);
}

// Page of the 16 keys from 16 * group on.  A number outside the cache is taken for the nearest inside.
__device__ __forceinline__ int page_of(const PagedParams& p, const int32_t* table, int group) {
    const int page = table[divide((uint32_t)group * 16u, p.page, p.page_m)];
    return page < 0 ? 0 : (page >= p.n_pages ? p.n_pages - 1 : page);
}
// row of a page that the group starts at
__device__ __forceinline__ int row_in_page(const PagedParams& p, int group) {
    const int key = group * 16;
    return key - divide((uint32_t)key, p.page, p.page_m) * p.page;
}

// ---- partial results ----------------------------------------------------------------------------------------------------------------------------------
// SHARED: between workgroups of one launch, past the L2s (those of the XCDs are not coherent).
template <bool SHARED> __device__ __forceinline__ float2 load_partial(const float* at) {
    if constexpr (!SHARED) return *reinterpret_cast<const float2*>(at);
    const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)));
}
__device__ __forceinline__ void store_partial(float* at, float a, float b, bool shared) {
    if (shared) __hip_atomic_store(reinterpret_cast<uint64_t*>(at), (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else *reinterpret_cast<float2*>(at) = make_float2(a, b);
}

// A row's partial results of `splits` splits, `step` rows of results apart, by 16 lanes with D / 16 features each, 2 (i + 16 k) and the next for
// k = 0, 1, ...; those of STEP splits are requested before the first is used.
template <int D> struct RowSum {
    static constexpr int kPairs = D / 32;
    float M = -INFINITY, L = 0.f;
    float2 O[kPairs];
    __device__ __forceinline__ RowSum() {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) O[k] = make_float2(0.f, 0.f);
    }
    // N more results
    template <int N> __device__ __forceinline__ void add(const float2 (&ml)[N], const float2 (&o)[N][kPairs]) {
        float m = M;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, ml[i].x);
        const float a = M == -INFINITY ? 0.f : fast_exp2(M - m);
        L *= a;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) { O[k].x *= a; O[k].y *= a; }
        M = m;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float w = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - M);
            // (named: of two products in a sum the compiler takes either into the fma, and both launches that merge have to leave the same bits)
            L = __builtin_fmaf(w, ml[i].y, L);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                O[k].x = __builtin_fmaf(w, o[i][k].x, O[k].x);
                O[k].y = __builtin_fmaf(w, o[i][k].y, O[k].y);
            }
        }
    }
    template <bool SHARED, int STEP> __device__ __forceinline__ void add(const float* from_o, const float* from_ml, int64_t first, int64_t step, int splits) {
        constexpr int kStep = STEP;
        const int lane = threadIdx.x & 15;
        for (int s0 = 0; s0 < splits; s0 += kStep) {
            float2 ml[kStep], o[kStep][kPairs];
#pragma unroll
            for (int i = 0; i < kStep; ++i) {              // past the last split: its values again
                const int64_t at = first + min(s0 + i, splits - 1) * step;
                ml[i] = load_partial<SHARED>(from_ml + at * 2);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) o[i][k] = load_partial<SHARED>(from_o + at * D + 2 * (lane + 16 * k));
            }
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                if (s0 + i < splits) continue;             // ... with nothing in them (no weight would not do for an infinite output)
                ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) o[i][k] = make_float2(0.f, 0.f);
            }
            add(ml, o);
        }
    }
    __device__ __forceinline__ void store(elem_t* row) const {
        const int lane = threadIdx.x & 15;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) *reinterpret_cast<uint32_t*>(row + 2 * (lane + 16 * k)) = pack_elem2(O[k].x * inv, O[k].y * inv);
    }
};

// Rows r0 to r0 + n - 1 of block `block` of few rows, its splits merged by 256 threads: per row 16 / n groups of 16 lanes with a share of the splits each,
// together through LDS (16 x (D + 2) floats).
template <int D, int BLOCK, bool SHARED>
__device__ __forceinline__ void merge_rows(const PagedParams& p, const PagedFound& f, int block, int kvh, int r0, int n, float* lds) {
    const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
    int per_row = 16;
    while (per_row * n > 16) per_row /= 2;
    const int r = group / per_row, part = group - r * per_row;
    RowSum<D> sum;
    if (r < n && part < f.splits) {
        const int64_t step = (int64_t)f.work.blocks * p.nkv * BLOCK, first = ((int64_t)(f.partial + block) * p.nkv + kvh) * BLOCK + r0 + r;
        sum.template add<SHARED, 8>(p.rows_o, p.rows_ml, first + part * step, step * per_row, (f.splits - part + per_row - 1) / per_row);
    }
    float* mine = lds + group * (D + 2);
    if (lane == 0) { mine[0] = sum.M; mine[1] = sum.L; }
#pragma unroll
    for (int k = 0; k < RowSum<D>::kPairs; ++k) *reinterpret_cast<float2*>(mine + 2 + 2 * (lane + 16 * k)) = sum.O[k];
    __syncthreads();
    if (part != 0 || r >= n) return;
    for (int i = 1; i < per_row; ++i) {
        const float* other = mine + i * (D + 2);
        float2 ml[1], o[1][RowSum<D>::kPairs];
        ml[0] = make_float2(other[0], other[1]);
#pragma unroll
        for (int k = 0; k < RowSum<D>::kPairs; ++k) o[0][k] = *reinterpret_cast<const float2*>(other + 2 + 2 * (lane + 16 * k));
        sum.add(ml, o);
    }
    const int row = block * BLOCK + r0 + r, token = divide(row, p.n_rep, p.rep_m);
    sum.store(p.o + (int64_t)(f.seq.first + token) * p.o_st + (int64_t)(kvh * p.n_rep + row - token * p.n_rep) * p.o_sh);
}

// ---- rows whose products met values that are not finite -----------------------------------------------------------------------------------------------
// A matrix product multiplies a masked key's probability, zero, with whatever its value holds, and zero times infinity or NaN is NaN.  So a row that is not
// finite and has fewer keys than its workgroup multiplies is computed anew from its own keys alone, by one wavefront: key by key with a lane each
// for the scores, then feature by feature (2 lane, 2 lane + 1).  Nothing but such values pays for it.
__device__ __forceinline__ bool not_finite(float x) {
    uint32_t u = __float_as_uint(x);
    asm("" : "+v"(u));                                     // a test of these bits as they are: one of a float is compiled without NaN
    return (u & 0x7f800000u) == 0x7f800000u;
}

template <int D>
__device__ __forceinline__ void own_keys_only(const PagedParams& p, const int32_t* table, int kvh, const elem_t* q, int k0, int limit, float& M, float& L, float& O0,
                                              float& O1) {
    const int lane = threadIdx.x & 63, d = 2 * lane;
    M = -INFINITY;
    L = O0 = O1 = 0.f;
    for (int key0 = k0; key0 < limit; key0 += 64) {
        const int key = min(key0 + lane, limit - 1), n = min(64, limit - key0);
        const int64_t at = (int64_t)page_of(p, table, key >> 4) * p.p_sp + (int64_t)(row_in_page(p, key >> 4) + (key & 15)) * p.p_st + (int64_t)kvh * p.p_sh;
        float s = 0.f;
        for (int f = 0; f < D; f += 8) {
            float a[8], b[8];
            Elem<elem_t>::unpack(ld128(q + f), a);
            Elem<elem_t>::unpack(ld128(p.kp + at + f), b);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += a[i] * b[i];
        }
        s = lane < n ? s * p.scale_log2 : -INFINITY;
        const float m = fmaxf(M, group_max<64>(s)), use = m == -INFINITY ? 0.f : m, alpha = M == -INFINITY ? 0.f : fast_exp2(M - use);
        const float e = lane < n ? fast_exp2(s - use) : 0.f, e_rounded = (float)(elem_t)e;      // as the kernels' products have it
        L = L * alpha + group_sum<64>(e);
        O0 *= alpha;
        O1 *= alpha;
        M = m;
        for (int j = 0; j < n; ++j) {
            const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e_rounded), j));
            const int64_t vj = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)at, j));
            if (d < D) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(p.vp + vj + d);
                O0 += pj * elem_lo(v);
                O1 += pj * elem_hi(v);
            }
        }
    }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------------------------------
// One workgroup per (block of 16 NB rows, KV head, split); its wavefronts take chunks of 32 keys in turn:
//     S^T[key][row] = K Q^T      v_mfma_f32_16x16x32, A = K rows straight from global memory in operand layout, B = Q^T
//     online softmax over keys   a lane's column is a row: eight keys in the lane, two lane exchanges
//     O^T[feature][row] += V^T P^T    V passes through a wavefront's own LDS and is read back transposed
// Every cached element is read from memory once per block of rows.  The next chunk's K is requested as soon as the scores are computed and its V as soon as this
// chunk's is in LDS, into the same registers: 16 KB a wavefront (d 128) are always under way, and 12 wavefronts fit a compute unit.  (Two sets of registers, a
// whole chunk ahead: 8 wavefronts, 16 rows to a block at the most.)  Bound by memory: 32 x 8 items of 200 - 8192 keys of 128 features 83.8 - 85.6 us, 6.1 TB/s; few items
// by the start and the merge besides, ~10 us: 8 x 8 items of 4096 keys 32.7, a single one of 1500 9.8 (6.5 and a second launch of 5.5 without the merge in it).
template <int D, int NB>
__global__ __launch_bounds__(64 * kRowWaves, NB == 1 ? 3 : 2) void paged_rows_kernel(const PagedParams p) {
    constexpr int NWV = kRowWaves, kThreads = 64 * NWV, BLOCK = 16 * NB;
    constexpr int KS = D / 32, DT = D / 16;
    constexpr int VSTR = 2 * D + 32;          // bytes per key row of a staged V chunk: transposed reads of 8 rows x 32 bytes hit 256 distinct bytes
    constexpr int V_ITEMS = 8 * (D / 8);      // (four keys, eight features) of a chunk
    constexpr int V_PER_LANE = (V_ITEMS + 63) / 64;
    constexpr int kStaged = NWV * kRowChunk * VSTR, kResults = NWV * BLOCK * (D + 1) * 4;
    __shared__ __attribute__((aligned(16))) char pool[kStaged > kResults ? kStaged : kResults];     // V chunks, then the wavefronts' results
    __shared__ float wm_lds[NWV][BLOCK], wl_lds[NWV][BLOCK];
    __shared__ int redo_lds[BLOCK];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, G = lane >> 4;
    const int slot = divide(blockIdx.x, p.nkv, p.nkv_m), kvh = blockIdx.x - slot * p.nkv;
    const PagedFound f = find_work<BLOCK, kRowTile, kSlots>(p, p.rows, p.share_m[0], slot);
    if (f.b < 0) return;
    const int in = slot - f.at, split = paged_quotient(in, f.work.blocks), block = in - split * f.work.blocks;
    int s0, s1;
    paged_split_keys<kRowTile>(f.seq, f.work, f.splits, split, s0, s1);
    const int n_rows = min(BLOCK, f.seq.n * p.n_rep - block * BLOCK);

    // this lane's rows, l16 and 16 further on
    uint4 raw[NB][KS];
    int limit[NB], end = 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int r = 16 * nb + l16, row = block * BLOCK + min(r, n_rows - 1), token = divide(row, p.n_rep, p.rep_m), head = kvh * p.n_rep + row - token * p.n_rep;
        limit[nb] = r < n_rows ? min(paged_limit(f.seq, token, p.causal), s1) : 0;
        end = max(end, group_max<16>(limit[nb]));          // the same for the four groups of 16 lanes
        const elem_t* qr = p.q + (int64_t)(f.seq.first + token) * p.q_st + (int64_t)head * p.q_sh + 8 * G;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) raw[nb][ks] = ld128(qr + 32 * ks);
    }
    const int n_iter = __builtin_amdgcn_readfirstlane(end > s0 ? (end - s0 + kRowTile - 1) / kRowTile : 0);
    const int last = max(s1 - 1, 0), last_group = last >> 4;      // keys past the split repeat its last one

    f32x4v o_acc[NB][DT];
    float m_i[NB], l_i[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o_acc[nb][dt] = f32x4v{0.f, 0.f, 0.f, 0.f};
        m_i[nb] = -INFINITY;
        l_i[nb] = 0.f;
    }

    const int32_t* table = p.table + (int64_t)f.b * p.table_stride;
    const elem_t *kbase = p.kp + (int64_t)kvh * p.p_sh, *vbase = p.vp + (int64_t)kvh * p.p_sh;
    char* vt = pool + wave * kRowChunk * VSTR;
    const char* vt_lane = vt + (4 * G + (l16 >> 2)) * VSTR + 8 * (l16 & 3);
    // lane i: pages of both groups of this wavefront's chunk i of the 64 from `ids_from` on
    int ids[2], ids_from = 0;
    auto look_up = [&](int from) {
        ids_from = from;
        const int group = (s0 + (NWV * (from + lane) + wave) * kRowChunk) >> 4;
#pragma unroll
        for (int t = 0; t < 2; ++t) ids[t] = page_of(p, table, min(group + t, last_group));
        // waited for here: where they are used the wait would be for everything that is under way, in every step
        asm volatile("" : "+v"(ids[0]), "+v"(ids[1]));
    };
    // the chunk that is requested next: its first key, its two groups of 16 keys and where these start in the pages
    int key_next, group[2];
    int64_t at[2];
    auto place = [&](int it) {
        key_next = s0 + (NWV * it + wave) * kRowChunk;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            group[t] = min((key_next >> 4) + t, last_group);
            at[t] = (int64_t)__builtin_amdgcn_readlane(ids[t], it - ids_from) * p.p_sp + (int64_t)row_in_page(p, group[t]) * p.p_st;
        }
    };
    elem8_t kf[2][KS];
    uint4 vraw[V_PER_LANE][4];
    auto request_k = [&]() {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = min(key_next + 16 * t + l16, last) - 16 * group[t];
            const elem_t* kr = kbase + at[t] + (int64_t)r * p.p_st + 8 * G;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kf[t][ks] = __builtin_bit_cast(elem8_t, ldg_nt(reinterpret_cast<const uint4*>(kr + 32 * ks)));
        }
    };
    auto request_v = [&]() {
#pragma unroll
        for (int j = 0; j < V_PER_LANE; ++j) {
            const int item = lane + 64 * j;
            if (V_ITEMS % 64 != 0 && item >= V_ITEMS) break;
            const int quad = item / (D / 8), dg = item % (D / 8);
            const int g = quad < 4 ? group[0] : group[1];
            const elem_t* vr = vbase + (quad < 4 ? at[0] : at[1]) + 8 * dg;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int rr = min(key_next + 4 * quad + r, last) - 16 * g;
                vraw[j][r] = ldg_nt(reinterpret_cast<const uint4*>(vr + (int64_t)rr * p.p_st));
            }
        }
    };

    if (n_iter > 0) {
        look_up(0);
        place(0);
        request_k();
        request_v();
    }
    elem8_t qf[NB][KS];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[nb][ks] = __builtin_bit_cast(elem8_t, raw[nb][ks]);
    // No branch around a request or a chunk: where paths meet, the wait for a chunk would be for the next one too.  So the chunk behind the last is requested
    // as well (the split's last key over and over), and a wavefront without keys computes along with the others, with nothing in its chunk.
    for (int it = 0; it < n_iter; ++it) {
        const int key0 = key_next;
        f32x4v s_acc[NB][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                s_acc[nb][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s_acc[nb][t] = mfma_16x16x32(kf[t][ks], qf[nb][ks], s_acc[nb][t]);
            }
        if (it + 1 - ids_from >= 64) look_up(it + 1);
        place(it + 1);
        __builtin_amdgcn_sched_barrier(0);
        request_k();
        __builtin_amdgcn_sched_barrier(0);
        elem8_t pf[NB];
        float alpha[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (key0 + 16 * t + 4 * G + r >= limit[nb]) s_acc[nb][t][r] = -INFINITY;
                    mx = fmaxf(mx, s_acc[nb][t][r]);
                }
            mx = quad_max(mx);
            const float m_new = fmaxf(m_i[nb], mx * p.scale_log2), m_use = m_new == -INFINITY ? 0.f : m_new;     // a row may have no key here, or none at all
            alpha[nb] = fast_exp2(m_i[nb] - m_use);
            m_i[nb] = m_new;
            float rs = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = fast_exp2(s_acc[nb][t][r] * p.scale_log2 - m_use);
                    rs += e;
                    pf[nb][4 * t + r] = (elem_t)e;         // slot (G, i): key 16 * (i / 4) + 4 * G + i % 4; rounded for the product, as P is in mi_attn_fwd
                }
            l_i[nb] = l_i[nb] * alpha[nb] + rs;
        }
        // A wavefront's own LDS, whose accesses run in program order: fences order the compiler, and the wavefronts never wait for each other in here.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < V_PER_LANE; ++j) {
            const int item = lane + 64 * j;
            if (V_ITEMS % 64 != 0 && item >= V_ITEMS) break;
            const int quad = item / (D / 8), dg = item % (D / 8);
#pragma unroll
            for (int r = 0; r < 4; ++r) st128(vt + (4 * quad + r) * VSTR + 16 * dg, vraw[j][r]);
        }
        __builtin_amdgcn_sched_barrier(0);
        request_v();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const elem8_t a = tr_pair(vt_lane + 32 * dt, vt_lane + 16 * VSTR + 32 * dt);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                o_acc[nb][dt] = o_acc[nb][dt] * alpha[nb];
                o_acc[nb][dt] = mfma_16x16x32(a, pf[nb], o_acc[nb][dt]);
            }
        }
    }

    // ---- the wavefronts' results together; of a single split the output, else a partial result ----
    float* wo = reinterpret_cast<float*>(pool);            // [wavefront][row][feature], rows D + 1 apart
    if (tid < BLOCK) redo_lds[tid] = 0;
    const int filled = s0 + n_iter * kRowTile;             // chunks reach up to here: with keys that a row may not see, or with others once more
    __syncthreads();                                       // nobody reads V any more
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float l = quad_sum(l_i[nb]);
        if (G == 0) { wm_lds[wave][16 * nb + l16] = m_i[nb]; wl_lds[wave][16 * nb + l16] = l; }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) wo[(wave * BLOCK + 16 * nb + l16) * (D + 1) + 16 * dt + 4 * G + r] = o_acc[nb][dt][r];
    }
    __syncthreads();
    const auto emit = [&](int r, int d, float M, float L, float O0, float O1) {
        if (f.splits == 1) {
            const int rr = block * BLOCK + r, i = divide(rr, p.n_rep, p.rep_m);
            const float inv = L == 0.f ? 0.f : 1.f / L;
            *reinterpret_cast<uint32_t*>(p.o + (int64_t)(f.seq.first + i) * p.o_st + (int64_t)(kvh * p.n_rep + rr - i * p.n_rep) * p.o_sh + d) = pack_elem2(O0 * inv, O1 * inv);
        } else {
            const int64_t to = ((int64_t)(f.partial + in) * p.nkv + kvh) * BLOCK + r;
            store_partial(p.rows_o + to * D + d, O0, O1, p.tickets != nullptr);
            if (d == 0) store_partial(p.rows_ml + to * 2, M, L, p.tickets != nullptr);
        }
    };
    for (int idx = tid; idx < n_rows * (D / 2); idx += kThreads) {
        const int r = idx / (D / 2), d = 2 * (idx % (D / 2));
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NWV; ++w) M = fmaxf(M, wm_lds[w][r]);
        float L = 0.f, O0 = 0.f, O1 = 0.f;
#pragma unroll
        for (int w = 0; w < NWV; ++w) {
            const float wm = wm_lds[w][r], scale = wm == -INFINITY ? 0.f : fast_exp2(wm - M);
            const float* from = wo + (w * BLOCK + r) * (D + 1) + d;
            L += scale * wl_lds[w][r];
            O0 += scale * from[0];
            O1 += scale * from[1];
        }
        if (not_finite(O0) || not_finite(O1) || not_finite(L)) redo_lds[r] = 1;
        emit(r, d, M, L, O0, O1);
    }
    bool uneven = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) uneven |= 16 * nb + l16 < n_rows && limit[nb] < filled;
    if (__ballot(uneven) != 0) {                           // the same for the workgroup
        __syncthreads();
        for (int r = wave; r < n_rows; r += NWV) {
            const int lim = NB == 2 && r >= 16 ? __builtin_amdgcn_readlane(limit[NB - 1], r & 15) : __builtin_amdgcn_readlane(limit[0], r & 15);
            if (redo_lds[r] == 0 || lim >= filled) continue;
            const int rr = block * BLOCK + r, i = divide(rr, p.n_rep, p.rep_m);
            float M, L, O0, O1;
            own_keys_only<D>(p, table, kvh, p.q + (int64_t)(f.seq.first + i) * p.q_st + (int64_t)(kvh * p.n_rep + rr - i * p.n_rep) * p.q_sh, s0, lim, M, L, O0, O1);
            if (2 * lane < D) emit(r, 2 * lane, M, L, O0, O1);
        }
    }
    // With tickets the workgroup of a block that is last to get here merges its splits; nobody waits for anybody.  Partial results are stored past the L2 and
    // every wavefront has waited for its own before the barrier, so the count that thread 0 raises behind it comes after them in memory, and the loads of
    // the workgroup that reads the highest count come after all.  (Two launches, the second one merging, of 1500 keys of 32 / 8 heads: 11.5 us one call after the
    // other, one launch 9.6.)
    if constexpr (NB > 1) return;
    if (f.splits == 1 || p.tickets == nullptr) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        int32_t* ticket = p.tickets + (int64_t)(f.partial + block) * p.nkv + kvh;
        const int arrived = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        redo_lds[0] = arrived == f.splits - 1;
        if (arrived == f.splits - 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the next launch
    }
    __syncthreads();
    if (redo_lds[0] == 0) return;
    static_assert(NWV == 4 && sizeof(pool) >= 16 * (D + 2) * sizeof(float), "merge_rows: 256 threads, and room in LDS");
    merge_rows<D, BLOCK, true>(p, f, block, kvh, 0, n_rows, wo);
}

// ---- chunks -------------------------------------------------------------------------------------------------------------------------------------------
// Direct loads of this wavefront's 16 rows of a 64-key tile.
template <int D> struct PageDma {
    using T = LdsTile<D>;
    static constexpr int COUNT = T::kInstrs / 4;
    uint32_t off[COUNT];
    int lw, lane;
    __device__ __forceinline__ static void src_of(int n, int lw, int lane, int& row, int& unit_off) {
        int unit;
        T::dma_src(lw * COUNT + n, lane, row, unit);
        if (D == 96 && unit >= D / 8) unit = 0;
        row -= 16 * lw;
        unit_off = 16 * unit;
    }
    __device__ __forceinline__ void init(int lw_, int lane_, int64_t tok_stride) {
        lw = lw_;
        lane = lane_;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            int row, unit_off;
            src_of(j, lw, lane, row, unit_off);
            off[j] = (uint32_t)(row * (int)tok_stride * 2 + unit_off);
        }
    }
    // base: key 16 * group of the wavefront's group (uniform); rows: how many of the 16 there are (further ones repeat the last)
    __device__ __forceinline__ void issue(const elem_t* base, int64_t tok_stride, int rows, char* tile) const {
        char* dst = tile + 1024 * COUNT * lw;
        if (rows >= 16) {
#pragma unroll
            for (int j = 0; j < COUNT; ++j) DmaPlan<D, 1>::issue_one(off[j], base, dst + 1024 * j);
        } else {
            int l = lane;
            asm volatile("" : "+v"(l));
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                int row, unit_off;
                src_of(j, lw, l, row, unit_off);
                DmaPlan<D, 1>::issue_one((uint32_t)(min(row, rows - 1) * (int)tok_stride * 2 + unit_off), base, dst + 1024 * j);
            }
        }
    }
};

// One workgroup per (block of 256 rows, KV head, split): eight wavefronts of 32 rows.  Tiles of 64 keys stream through rings of four swizzled LDS stages,
// K requested three tiles ahead by the second four wavefronts and V two by the first.  The two groups of four run half a tile apart (enforced by the
// barriers), so on every SIMD one wavefront issues products while the other computes its softmax:
//     S^T = K Q^T      A = K rows from LDS, B = Q in registers
//     softmax          a lane's column is a row of the block; the maximum is raised only when it lags by 2^8, so most tiles rescale nothing; probabilities (up
//                      to 2^8 then) are rounded to the element type for the product, as in mi_attn_fwd: half a step of each, where P in two
//                      terms would be twice the products of P V.  (Relative error of the outputs against 64 bits: 0.0023 bf16, 0.00029 f16, of which one rounding
//                      of the output alone leaves 0.0017, 0.00021)
//     O^T += V^T P^T   B = P^T as the accumulators of S^T hold it, A = V^T by transposing LDS reads
// Bound by the matrix pipe (busy half of the time) and the power that it draws: 4 x 2048 tokens behind 2048 - 14336 others, 32 / 8 heads of 128, 1055 - 1106 us by the card's clock, 1.05 - 1.10 PFLOP/s, as
// mi_attn_fwd over contiguous keys; without its softmax 951, without its operand reads 890.  (Operands 2, 4, 8 products ahead instead of 3: 1104, 1076, 1093; the
// first of them before the barrier: 1150.)
template <int D>
__global__ __launch_bounds__(512, 2) void paged_tiles_kernel(const PagedParams p) {
    constexpr int NW = 8, BN = kTileKeys;
    constexpr int KS = D / 16, DT = D / 32, NS = 4;
    using Tile = LdsTile<D>;
    constexpr int RB = Tile::RB, TILE = Tile::kBytes, IPW = PageDma<D>::COUNT;
    __shared__ __attribute__((aligned(1024))) char k_lds[NS * TILE];
    __shared__ __attribute__((aligned(1024))) char v_lds[NS * TILE];
    __shared__ int end_lds[NW];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, l32 = lane & 31, g = lane >> 5;
    const int slot = divide(blockIdx.x, p.nkv, p.nkv_m), kvh = blockIdx.x - slot * p.nkv;
    const PagedFound f = find_work<kTileRows, kTileKeys, kLongestFirst>(p, p.tiles, p.share_m[1], slot);
    if (f.b < 0) return;                                   // the same for the whole workgroup
    const int in = slot - f.at, split = paged_quotient(in, f.work.blocks), block = f.work.blocks - 1 - (in - split * f.work.blocks);      // longest first
    int s0, s1;
    paged_split_keys<kTileKeys>(f.seq, f.work, f.splits, split, s0, s1);

    // ---- this lane's row, its keys [s0, limit), its part of Q ----
    const int n_rows = f.seq.n * p.n_rep, row = block * kTileRows + wave * 32 + l32;
    const int rr = min(row, n_rows - 1), token = divide(rr, p.n_rep, p.rep_m), head = kvh * p.n_rep + rr - token * p.n_rep;
    const int limit = row < n_rows ? min(paged_limit(f.seq, token, p.causal), s1) : 0;
    elem8_t qf[KS];
    {
        const elem_t* qrow = p.q + (int64_t)(f.seq.first + token) * p.q_st + (int64_t)head * p.q_sh + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = __builtin_bit_cast(elem8_t, ld128(qrow + 16 * ks));
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));     // in registers before the loop: waited for here, not behind the loop's loads
    const int wmax = group_max<64>(limit);
    if (lane == 0) end_lds[wave] = wmax;
    __syncthreads();
    int end = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) end = max(end, end_lds[w]);
    const int n_tiles = __builtin_amdgcn_readfirstlane(end > s0 ? (end - s0 + BN - 1) / BN : 0);

    f32x16_t o_acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[dt][r] = 0.f;
    float m_i = -INFINITY, l_i = 0.f;

    // ---- direct loads: wavefronts 0 - 3 of V, 4 - 7 of K; wavefront lw of either of keys 16 lw .. + 15 of a tile ----
    const bool v_role = wave < 4;
    const int lw = wave & 3, grp = wave >> 2;
    const int32_t* table = p.table + (int64_t)f.b * p.table_stride;
    const elem_t* base = (v_role ? p.vp : p.kp) + (int64_t)kvh * p.p_sh;
    char* ring = v_role ? v_lds : k_lds;
    const int last = max(s1 - 1, 0), last_group = last >> 4;
    PageDma<D> dma;
    dma.init(lw, lane, p.p_st);
    int ids = 0;                                           // lane i: page of this wavefront's keys in tile i of the current 64
    auto load_tile = [&](int tile) {
        if (tile >= n_tiles) return;
        const int group0 = (s0 >> 4) + lw;
        if ((tile & 63) == 0) {
            ids = page_of(p, table, min(group0 + 4 * (tile + lane), last_group));
            asm volatile("" : "+v"(ids));                  // waited for here, not (with all that is under way) at its use in every step
        }
        const int group = min(group0 + 4 * tile, last_group);
        const int page = __builtin_amdgcn_readlane(ids, tile & 63);
        const elem_t* from = base + (int64_t)page * p.p_sp + (int64_t)row_in_page(p, group) * p.p_st;
        dma.issue(from, p.p_st, last - 16 * group + 1, ring + (tile % NS) * TILE);
    };
    auto n_issued = [&](int a, int b) { return IPW * max(0, min(b, n_tiles) - a); };
    if (n_tiles > 0) {
        load_tile(0);
        load_tile(1);
        if (!v_role) {
            load_tile(2);
            wait_vmcnt_dyn(n_issued(1, 3));
        }
    }
    __syncthreads();
    if (grp == 1) __syncthreads();

    const float c2 = p.scale_log2;
    int v_h0, v_h1;
    Tile::tr_bases(lane, v_h0, v_h1);
    const int k_row = Tile::row_base(l32, g);
    f32x16_t s_acc[2];
    elem8_t pf[4];
    bool pending = false;
    constexpr int PV_STEPS = 4 * DT, S_STEPS = 2 * KS, kDepth = 3;
    auto mfma_phase = [&](auto mode, const char* vt, const char* ks) {
        constexpr bool kPV = (decltype(mode)::value & 1) != 0, kS = (decltype(mode)::value & 2) != 0;
        constexpr int first = kPV ? 0 : PV_STEPS, last_step = kS ? PV_STEPS + S_STEPS : PV_STEPS;
        elem8_t operands[kDepth];                          // requested three products ahead
        auto fetch = [&](int i) -> elem8_t {
            if (i < PV_STEPS) {
                const int m = i / DT, dt = i % DT;
                return tr_pair(vt + (v_h0 ^ (dt << 6)) + 16 * m * RB, vt + (v_h1 ^ (dt << 6)) + 16 * m * RB);
            }
            const int ksi = (i - PV_STEPS) >> 1, t = (i - PV_STEPS) & 1;
            return *reinterpret_cast<const elem8_t*>(ks + (k_row ^ (ksi << 5)) + 32 * t * RB);
        };
        if constexpr (kS) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) s_acc[t][r] = 0.f;
        }
#pragma unroll
        for (int i = first; i < first + kDepth && i < last_step; ++i) operands[(i - first) % kDepth] = fetch(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = first; i < last_step; ++i) {
            const elem8_t a = operands[(i - first) % kDepth];
            if (i < PV_STEPS) {
                const int m = i / DT, dt = i % DT;
                o_acc[dt] = mfma_32x32x16(a, pf[m], o_acc[dt]);
            } else {
                const int ksi = (i - PV_STEPS) >> 1, t = (i - PV_STEPS) & 1;
                s_acc[t] = mfma_32x32x16(a, qf[ksi], s_acc[t]);
            }
            if (i + kDepth < last_step) operands[(i - first) % kDepth] = fetch(i + kDepth);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int it = 0; it <= n_tiles; ++it) {
        const int kt = s0 + it * BN;
        const bool wave_active = it < n_tiles && kt < wmax;
        {
            const char* vt = v_lds + ((it + NS - 1) % NS) * TILE;
            const char* ks = k_lds + (it % NS) * TILE;
            if (pending && wave_active) mfma_phase(std::integral_constant<int, 3>{}, vt, ks);
            else if (pending) mfma_phase(std::integral_constant<int, 1>{}, vt, ks);
            else if (wave_active) mfma_phase(std::integral_constant<int, 2>{}, vt, ks);
        }
        if (it == n_tiles) break;
        if (!v_role) wait_vmcnt_dyn(n_issued(it + 2, it + 3));        // K tile it + 1 is read behind this barrier
        __syncthreads();
        pending = wave_active;
        if (wave_active) {
            if (__any(kt + BN > limit)) {
                int rel = kt + 4 * g - limit;
                asm volatile("" : "+v"(rel));              // keeps the 32 compares inside this branch
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (rel + 32 * t + 8 * (r >> 2) + (r & 3) >= 0) s_acc[t][r] = -INFINITY;
            }
            float mx = fmaxf(s_acc[0][0], s_acc[1][0]);
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, fmaxf(s_acc[0][r], s_acc[1][r]));
            mx = pair_max(mx);
            const float m_cand = mx * c2;
            if (__any(m_cand > m_i + kRescaleGap)) {
                const float m_new = fmaxf(m_i, m_cand);
                float alpha = (m_new == -INFINITY) ? 1.0f : fast_exp2(m_i - m_new);
                asm volatile("" : "+v"(alpha));            // keeps the multiplies below inside this rarely taken branch
                m_i = m_new;
                l_i *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o_acc[dt][r] *= alpha;
            }
            const float m_use = (m_i == -INFINITY) ? 0.f : m_i;
            float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int t = m >> 1, r0 = 8 * (m & 1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float ev = fast_exp2(s_acc[t][r0 + e] * c2 - m_use);
                    if (e & 1) rs1 += ev; else rs0 += ev;
                    pf[m][e] = (elem_t)ev;
                }
            }
            l_i += rs0 + rs1;
        }
        load_tile(it + (v_role ? 2 : 3));
        if (v_role) wait_vmcnt_dyn(n_issued(it + 1, it + 3));         // V tile it is read behind this barrier
        __syncthreads();
    }
    if (grp == 0) __syncthreads();

    const float l_tot = pair_sum(l_i);
    const int64_t partial = ((int64_t)(f.partial + split * f.work.blocks + block) * p.nkv + kvh) * p.tile_rows + wave * 32;     // of the wavefront's first row
    uint64_t redo = 0;
    const int filled = (s1 + BN - 1) & -BN;                // tiles are filled up to here: with keys that a row may not see, or with others once more
    if (__any(row < n_rows && limit < filled)) {
        uint32_t bad = not_finite(l_tot);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) bad |= (uint32_t)not_finite(o_acc[dt][r]);
        redo = __ballot(bad != 0 && row < n_rows && limit < filled);
        redo = (redo | redo >> 32) & 0xffffffffu;
    }
    if (row < n_rows && (redo >> l32 & 1) == 0) {
        if (f.splits == 1) {
            const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;
            elem_t* orow = p.o + (int64_t)(f.seq.first + token) * p.o_st + (int64_t)head * p.o_sh + 4 * g;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<uint2*>(orow + 32 * dt + 8 * a) = make_uint2(pack_elem2(o_acc[dt][4 * a] * inv, o_acc[dt][4 * a + 1] * inv),
                                                                                   pack_elem2(o_acc[dt][4 * a + 2] * inv, o_acc[dt][4 * a + 3] * inv));
        } else {
            float* orow = p.tiles_o + (partial + l32) * D + 4 * g;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<float4*>(orow + 32 * dt + 8 * a) = make_float4(o_acc[dt][4 * a], o_acc[dt][4 * a + 1], o_acc[dt][4 * a + 2], o_acc[dt][4 * a + 3]);
            if (g == 0) *reinterpret_cast<float2*>(p.tiles_ml + (partial + l32) * 2) = make_float2(m_i, l_tot);
        }
    }
    for (; redo != 0; redo &= redo - 1) {
        const int r = __builtin_ctzll(redo), t = __builtin_amdgcn_readlane(token, r), h = __builtin_amdgcn_readlane(head, r), d = 2 * lane;
        float M, L, O0, O1;
        own_keys_only<D>(p, table, kvh, p.q + (int64_t)(f.seq.first + t) * p.q_st + (int64_t)h * p.q_sh, s0, __builtin_amdgcn_readlane(limit, r), M, L, O0, O1);
        if (d >= D) continue;
        if (f.splits == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            *reinterpret_cast<uint32_t*>(p.o + (int64_t)(f.seq.first + t) * p.o_st + (int64_t)h * p.o_sh + d) = pack_elem2(O0 * inv, O1 * inv);
        } else {
            *reinterpret_cast<float2*>(p.tiles_o + (partial + r) * D + d) = make_float2(O0, O1);
            if (d == 0) *reinterpret_cast<float2*>(p.tiles_ml + (partial + r) * 2) = make_float2(M, L);
        }
    }
}

// ---- merge of the splits ------------------------------------------------------------------------------------------------------------------------------
// A workgroup per 16 rows of a split block and KV head of paged_rows (the first n_rows_groups), where they are not merged in their own launch, and per
// `per_group` rows of a block of paged_tiles: 16, or 32 where there may be so many workgroups that most of them, which find nothing, set the time.  (us of 16 and 32:
// up to 6000 workgroups 15.0 and 10.1, 256 of 32 splits each 9.8 and 15.4.  Two lanes to a pair of features and rows one after the other, with a workgroup
// for every partial result, most of them idle: 19 for 64 blocks of 256 rows in four splits, 8.7 so.)
template <int D, int NB>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams p, int n_rows_groups, int per_block, int per_group) {
    __shared__ float lds[16 * (D + 2)];
    if ((int)blockIdx.x < n_rows_groups) {
        constexpr int BLOCK = 16 * NB;
        const int at_kv = blockIdx.x / NB, r0 = blockIdx.x % NB * 16, at = divide(at_kv, p.nkv, p.nkv_m), kvh = at_kv - at * p.nkv;
        const PagedFound f = find_work<BLOCK, kRowTile, kSplitBlocks>(p, p.rows, p.share_m[0], at);
        if (f.b < 0) return;
        const int n = min(16, f.seq.n * p.n_rep - (at - f.at) * BLOCK - r0);
        if (n > 0) merge_rows<D, BLOCK, false>(p, f, at - f.at, kvh, r0, n, lds);
        return;
    }
    const int group = blockIdx.x - n_rows_groups, at_kv = group / per_block, z = group - at_kv * per_block;
    const int at = divide(at_kv, p.nkv, p.nkv_m), kvh = at_kv - at * p.nkv;
    const PagedFound f = find_work<kTileRows, kTileKeys, kSplitBlocks>(p, p.tiles, p.share_m[1], at);
    if (f.b < 0) return;
    const int block = at - f.at, n_rows = min(f.seq.n * p.n_rep - block * kTileRows, per_group * (z + 1));
    for (int in = per_group * z + (threadIdx.x >> 4); in < n_rows; in += 16) {
        RowSum<D> sum;
        sum.template add<false, 4>(p.tiles_o, p.tiles_ml, ((int64_t)(f.partial + block) * p.nkv + kvh) * p.tile_rows + in, (int64_t)f.work.blocks * p.nkv * p.tile_rows, f.splits);
        const int row = block * kTileRows + in, token = divide(row, p.n_rep, p.rep_m);
        sum.store(p.o + (int64_t)(f.seq.first + token) * p.o_st + (int64_t)(kvh * p.n_rep + row - token * p.n_rep) * p.o_sh);
    }
}

template <int D, int NB> int launch(const PagedParams& p, int64_t row_blocks, int64_t tile_blocks, hipStream_t st) {
    if (row_blocks > 0) {
        paged_rows_kernel<D, NB><<<dim3((unsigned)p.rows.max_slots * p.nkv), dim3(64 * kRowWaves), 0, st>>>(p);
        if (const int rc = mi_check_launch("paged_rows"); rc != MI_OK) return rc;
    }
    if (tile_blocks > 0) {
        paged_tiles_kernel<D><<<dim3((unsigned)p.tiles.max_slots * p.nkv), dim3(512), 0, st>>>(p);
        if (const int rc = mi_check_launch("paged_tiles"); rc != MI_OK) return rc;
    }
    const int64_t of_rows = p.rows.share > 0 && p.tickets == nullptr ? paged_max_split_blocks(p.rows, row_blocks) * p.nkv * NB : 0;
    const int64_t tile_groups = paged_max_split_blocks(p.tiles, tile_blocks) * p.nkv;
    const int per_group = tile_groups * p.tile_rows > 16 * kMergeMost * mi_compute_units() ? 32 : 16, per_block = (p.tile_rows + per_group - 1) / per_group;
    const int64_t groups = of_rows + tile_groups * per_block;
    if (groups == 0) return MI_OK;
    paged_merge_kernel<D, NB><<<dim3((unsigned)groups), dim3(256), 0, st>>>(p, (int)of_rows, per_block, per_group);
    return mi_check_launch("paged_merge");
}

// Workgroups per KV head that either kernel's work is cut for.  `items`: sequences x KV heads of the calls, as many as there may be.
// paged_rows, of which two or three share a compute unit: of many items small pieces keep the units even where lengths differ (8 workgroups to a unit, 6 of
// blocks of 32 rows), and 2 do where they do not; of few items more splits of each only make the merge longer.  (us of 512, 1024, 2048 workgroups, d 128: 32 x 8
// items of 200 - 8192 keys 98, 93, 87, all of 4096 keys 85, 85, 92; 8 x 8 items of 900 - 5000 keys and 3 - 9 tokens
// of 4 heads 39.9, 46.6 of 1024; 3 x 4 items of 20000 - 32768 keys of 64 features 23.9, 27.4 of 1024.  32 x 8 items of 20 rows, 200 - 8192 keys: 6 to a unit 123, 8 to a unit 130.)
constexpr int kRowsLeast = 2, kRowsMost = 8, kRowsMostWide = 6;     // per compute unit
// Up to so many keys a sequence is not split: a merge costs more.  (us, split and not, one call after the other.  Single tokens of 4 sequences, 32 / 8 heads of 128: 150 keys 9.6, 6.9, 300 keys 9.9, 9.2,
// 500 keys 10.3, 11.8; 120 tokens of 120 keys 18.7, 13.3, of 300 keys 22.4, 18.3, of 500 keys 21.7, 22.9; 6 x 200 tokens of 300 keys, 16 / 4 heads: 28.5, 20.7.)
constexpr int kUnsplitKeys = 384;
int share_of(int64_t workgroups, int nkv) { return workgroups / nkv > 0 ? (int)(workgroups / nkv) : 1; }
// paged_tiles, one to a compute unit: few blocks are cut into what runs at once.  Of many blocks of few rows (`longest` tokens to a sequence, whose partial
// results are small) pieces are up to four times smaller, as above.
struct Plans {
    PagedPlan rows, tiles;
    int row_block, tile_rows;                              // rows of a block of paged_rows; rows kept per partial result of paged_tiles
};
Plans make_plans(int64_t tokens, int64_t batch, int64_t items, int64_t longest, int64_t capacity, int n_rep, int nkv) {
    const int cus = mi_compute_units();
    const int64_t most = longest * n_rep;
    const bool few = 8 * items <= kRowsLeast * cus;
    const bool short_keys = capacity <= kRowsAloneKeys && (tokens * n_rep / (2 * kRowBlock) + batch) * nkv <= kRowsLeast * cus;
    Plans o;
    o.row_block = most <= kRowBlock ? kRowBlock : 2 * kRowBlock;
    const int limit = short_keys ? 0x7fffffff : few && most <= kRowsAlone ? kRowsAlone : kRowLimit;
    const int64_t rows_most = (o.row_block == kRowBlock ? kRowsMost : kRowsMostWide) * cus;
    o.rows = PagedPlan{0, limit, 0x7fffffff, share_of(few ? kRowsLeast * cus : std::min<int64_t>(8 * items, rows_most), nkv), 8 * items >= rows_most, 0, kUnsplitKeys / kRowTile, 0, 0};
    // Enough blocks for every compute unit: no splits, no merge.
    const bool many = tokens * n_rep / kTileRows * nkv >= cus;
    o.tile_rows = (int)std::min<int64_t>((most + 15) / 16 * 16, kTileRows);
    const int pieces = o.tile_rows * 4 <= kTileRows ? 4 : o.tile_rows * 2 <= kTileRows ? 2 : 1, at_once = share_of(cus, nkv);
    o.tiles = PagedPlan{limit, 0x7fffffff, 0x7fffffff, many ? 0 : pieces * at_once, 0, many ? 0 : at_once, kUnsplitKeys / kTileKeys, 0, 0};
    return o;
}
// Whether the last workgroup of a block merges, given tickets: no more workgroups than run at once.  Each waits for its results to be in memory, which more of them
// cannot hide: 32 x 8 items of 200 - 8192 keys in pieces for 2048 workgroups 100 us, with a launch of its own for the merge 92.
bool merges_in_launch(const PagedPlan& rows, int nkv) { return (int64_t)rows.share * nkv <= kRowsLeast * mi_compute_units(); }

size_t partial_bytes(int64_t partials, int nkv, int block_rows, int head_dim) { return (size_t)partials * nkv * block_rows * (size_t)(head_dim + 2) * sizeof(float); }
constexpr int64_t kMaxTiles = (1 << 24) + 1;              // of a sequence

}  // namespace

#ifndef MI_ELEM_F16
extern "C" int64_t mi_paged_attn_tickets(int32_t n_kv_heads) {
    if (n_kv_heads <= 0) return 0;
    return paged_max_partials(make_plans(0, 1, 0x7fffffff, 1, 1 << 30, 1, n_kv_heads).rows, kMaxTiles, kMaxTiles) * n_kv_heads;
}

extern "C" size_t mi_paged_attn_workspace_bytes(int64_t tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim) {
    if (tokens <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || head_dim <= 0) return 0;
    const int n_rep = n_q_heads / n_kv_heads;
    const bool chunks = tokens * n_rep > kRowLimit;
    // of any number of sequences, with chunks of any length: of shorter ones there are more pieces of fewer rows, no more together
    const Plans o = make_plans(0, 1, 0x7fffffff, chunks ? kTileRows : tokens, 1 << 30, n_rep, n_kv_heads);
    return partial_bytes(paged_max_partials(o.rows, kMaxTiles, kMaxTiles), n_kv_heads, o.row_block, head_dim) +
           (chunks ? partial_bytes(paged_max_partials(o.tiles, kMaxTiles, kMaxTiles), n_kv_heads, kTileRows, head_dim) : 0);
}
#endif

int MI_ENTRY(mi_paged_attn_impl)(const mi_paged_attn_args* a) {
    if (a->total_q < 0 || a->batch < 1 || a->n_pages < 1 || a->max_pages < 1 || a->page_size < 16 || a->page_size % 16 != 0 ||
        (int64_t)a->max_pages * a->page_size > (1 << 30) || a->max_q_len < 0 || a->total_q > 0x7fffffffLL)
        return mi_fail(MI_E_SHAPE, "paged_attn: %lld tokens of %d sequences, at most %d each, %d pages of %d keys (a multiple of 16), up to %d a sequence", (long long)a->total_q,
                       a->batch, a->max_q_len, a->n_pages, a->page_size, a->max_pages);
    if (a->n_q_heads <= 0 || a->n_kv_heads <= 0 || a->n_q_heads % a->n_kv_heads != 0)
        return mi_fail(MI_E_SHAPE, "paged_attn: n_q_heads=%d must be a positive multiple of n_kv_heads=%d", a->n_q_heads, a->n_kv_heads);
    if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 96 && a->head_dim != 128)
        return mi_fail(MI_E_SHAPE, "paged_attn: head_dim %d unsupported (32, 64, 96, 128)", a->head_dim);
    if (!a->q || !a->k_pages || !a->v_pages || !a->o || !a->page_table || !a->cu_seqlens || !a->ctx_len) return mi_fail(MI_E_NULL, "paged_attn: null pointer");
    if (a->softmax_scale <= 0.f || mi_is_nan(a->softmax_scale)) return mi_fail(MI_E_SHAPE, "paged_attn: softmax_scale must be positive");
    if (!mi_aligned16(a->q) || !mi_aligned16(a->k_pages) || !mi_aligned16(a->v_pages) || !mi_aligned16(a->o)) return mi_fail(MI_E_ALIGN, "paged_attn: tensors must be 16-byte aligned");
    for (const int64_t s : {a->q_stride_token, a->q_stride_head, a->o_stride_token, a->o_stride_head, a->page_stride, a->page_stride_token, a->page_stride_head})
        if (s % 8 != 0) return mi_fail(MI_E_ALIGN, "paged_attn: strides must be multiples of 8 elements");
    if (a->page_stride_token < 0 || a->page_stride_token > (1 << 26)) return mi_fail(MI_E_SHAPE, "paged_attn: a token stride of %lld elements", (long long)a->page_stride_token);
    PagedParams p{};
    p.q = (const elem_t*)a->q; p.kp = (const elem_t*)a->k_pages; p.vp = (const elem_t*)a->v_pages; p.o = (elem_t*)a->o;
    p.table = a->page_table; p.cu = a->cu_seqlens; p.ctx = a->ctx_len; p.table_stride = a->page_table_stride;
    p.q_st = a->q_stride_token; p.q_sh = a->q_stride_head; p.o_st = a->o_stride_token; p.o_sh = a->o_stride_head;
    p.p_sp = a->page_stride; p.p_st = a->page_stride_token; p.p_sh = a->page_stride_head;
    p.batch = a->batch; p.total = (int)a->total_q; p.n_pages = a->n_pages; p.page = a->page_size; p.max_pages = a->max_pages;
    p.capacity = a->max_pages * a->page_size; p.nq = a->n_q_heads; p.nkv = a->n_kv_heads; p.n_rep = a->n_q_heads / a->n_kv_heads; p.causal = a->causal != 0;
    p.page_m = divide_m(p.page); p.rep_m = divide_m(p.n_rep); p.nkv_m = divide_m(p.nkv);
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    const int64_t longest = a->max_q_len > 0 && a->max_q_len < p.total ? a->max_q_len : p.total;
    const Plans plans = make_plans(p.total, p.batch, std::min<int64_t>(p.batch, p.total) * p.nkv, longest, p.capacity, p.n_rep, p.nkv);
    p.rows = plans.rows;
    p.tiles = plans.tiles;
    p.tile_rows = plans.tile_rows;
    const bool two = plans.row_block == 2 * kRowBlock;
    // Where every sequence is a chunk, if no rows are behind the last one, there is no launch that would only find that out: a shorter one is computed as a chunk.
    // (4 x 2048 tokens behind others: 1112 -> 1088 us, the launch and its merge.)
    const bool chunks_only = std::min(longest, p.total - (p.batch - 1) * longest) * p.n_rep > plans.rows.rows_up_to;
    if (chunks_only) p.tiles.rows_over = 0;
    p.rows.max_n = p.tiles.max_n = (int)longest;
    const int64_t row_blocks = chunks_only ? 0 : two ? paged_max_blocks<2 * kRowBlock>(p.rows, p.total, p.batch, longest, p.n_rep) : paged_max_blocks<kRowBlock>(p.rows, p.total, p.batch, longest, p.n_rep);
    const int64_t tile_blocks = paged_max_blocks<kTileRows>(p.tiles, p.total, p.batch, longest, p.n_rep);
    const int64_t row_tiles = ((int64_t)p.capacity + kRowTile - 1) / kRowTile, tile_tiles = ((int64_t)p.capacity + kTileKeys - 1) / kTileKeys;
    // Sums of blocks x tiles and of rows are kept in 32 bits, and a grid has fewer than 2^31 workgroups.
    if (p.nkv > 0xffff) return mi_fail(MI_E_SHAPE, "paged_attn: more than 65535 KV heads");
    if ((int64_t)p.total * p.n_rep > 0x7fffffffLL - kTileRows || row_blocks * row_tiles > 0x7fffffffLL || tile_blocks * tile_tiles > 0x7fffffffLL ||
        (2 * row_blocks + 17 * tile_blocks + 8LL * mi_compute_units()) * p.nkv > 0x7fffffffLL)
        return mi_fail(MI_E_SHAPE, "paged_attn: %lld tokens of %d heads over up to %d keys are too many for one call", (long long)a->total_q, a->n_q_heads, p.capacity);
    const size_t need = mi_paged_attn_workspace_bytes(p.total, p.nq, p.nkv, a->head_dim);
    if (!a->workspace || a->workspace_bytes < need || !mi_aligned16(a->workspace))
        return mi_fail(MI_E_WORKSPACE, "paged_attn: workspace needs %zu bytes (16-byte aligned), got %zu", need, a->workspace_bytes);
    if (a->tickets && (a->n_tickets < mi_paged_attn_tickets(p.nkv) || (reinterpret_cast<uintptr_t>(a->tickets) & 3u) != 0))
        return mi_fail(MI_E_WORKSPACE, "paged_attn: %lld tickets (4-byte aligned), got %lld", (long long)mi_paged_attn_tickets(p.nkv), (long long)a->n_tickets);
    p.tickets = !two && merges_in_launch(p.rows, p.nkv) ? a->tickets : nullptr;
    // A page table without room for more: no splits, whatever the plan.
    if (row_tiles <= p.rows.least || row_blocks == 0) p.rows.share = 0;
    if (tile_tiles <= p.tiles.least || tile_blocks == 0) p.tiles.share = 0;
    p.share_m[0] = divide_m(p.rows.share); p.share_m[1] = divide_m(p.tiles.share);
    p.rows.max_slots = (int)paged_max_slots(p.rows, row_blocks, row_tiles);
    p.tiles.max_slots = (int)paged_max_slots(p.tiles, tile_blocks, tile_tiles);
    p.rows.max_partials = (int)paged_max_partials(p.rows, row_blocks, row_tiles);
    p.tiles.max_partials = (int)paged_max_partials(p.tiles, tile_blocks, tile_tiles);
    p.rows_o = (float*)a->workspace;
    p.rows_ml = p.rows_o + (size_t)p.rows.max_partials * p.nkv * plans.row_block * a->head_dim;
    p.tiles_o = p.rows_o + partial_bytes(p.rows.max_partials, p.nkv, plans.row_block, a->head_dim) / sizeof(float);
    p.tiles_ml = p.tiles_o + (size_t)p.tiles.max_partials * p.nkv * p.tile_rows * a->head_dim;
    const hipStream_t st = (hipStream_t)a->stream;
    const auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return two ? launch<D, 2>(p, row_blocks, tile_blocks, st) : launch<D, 1>(p, row_blocks, tile_blocks, st);
    };
    switch (a->head_dim) {
        case 32: return go(std::integral_constant<int, 32>{});
        case 64: return go(std::integral_constant<int, 64>{});
        case 96: return go(std::integral_constant<int, 96>{});
        default: return go(std::integral_constant<int, 128>{});
    }
}

// A token of every row of logits by temperature, top-k, top-p and min-p, from one given random number a row.
//
// A row's tokens are ordered by value, largest first, equal ones by index; token i weighs w_i = exp((x_i - max) / T).  Each of top-k (the first k), top-p (the
// fewest with p of their weight together) and min-p (those of at least min_p of the largest weight) keeps the first so many in that order, so all do, and the token is
// the first one behind which the running sum S of weights exceeds u times the sum of what is kept.  No order of the row is ever made: every question is "the
// first token with S (or the number of tokens) of at least G", and sums over bins of values answer it.  Sums are of whole numbers (weights times 2^F),
// exact in any order, so that atomics leave no trace of theirs; the weights themselves are rounded once, from 64-bit exponentials, as u lies close to a border in
// one row of some thousands where 32 bits are all there is.
#include "common.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 4096, kCandidates = 1024;

struct SampleParams {
    const void* logits;
    int64_t stride;
    int vocab;
    const float *uniforms, *temperature, *top_p, *min_p;   // of each row, or null
    const int32_t* top_k;
    float temperature0, top_p0, min_p0;                    // ... of all
    int32_t top_k0;
    int64_t* ids;
    float* logprobs;                                       // nullable
};

// ---- the logits -----------------------------------------------------------------------------------------------------------------------------------------
// 32-bit key of the same order as the values, -0 as +0; 0 for those that have no weight: NaN and -inf
__device__ __forceinline__ uint32_t value_key(float x) {
    const uint32_t u = __float_as_uint(x), magnitude = u & 0x7fffffffu;
    if (magnitude > 0x7f800000u || u == 0xff800000u) return 0;
    return u != magnitude && magnitude != 0 ? ~u : magnitude | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0 ? key & 0x7fffffffu : ~key); }

// A row as aligned 16-byte vectors, with the elements in front of the first and behind the last (at most a vector's less one each) one to a thread.
template <typename T> struct Row {
    static constexpr int V = Elem<T>::kVec, kAhead = 4;
    const T* x;
    int vocab, head, vecs;
    __device__ __forceinline__ Row(const SampleParams& p, int64_t row) : x(static_cast<const T*>(p.logits) + row * p.stride), vocab(p.vocab) {
        const int to_boundary = (int)(((16u - (unsigned)(reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / sizeof(T));
        head = to_boundary < vocab ? to_boundary : vocab;
        vecs = (vocab - head) / V;
    }
    // f(value, index) of every element
    template <class F> __device__ __forceinline__ void each(const F& f) const {
        const uint4* at = reinterpret_cast<const uint4*>(x + head);
        for (int v0 = threadIdx.x; v0 < vecs; v0 += kAhead * kThreads) {
            uint4 u[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) u[a] = at[min(v0 + a * kThreads, vecs - 1)];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int v = v0 + a * kThreads;
                if (v >= vecs) break;
                float e[V];
                Elem<T>::unpack(u[a], e);
#pragma unroll
                for (int i = 0; i < V; ++i) f(e[i], head + v * V + i);
            }
        }
        const int behind = head + vecs * V, i = (int)threadIdx.x < head ? (int)threadIdx.x : behind + (int)threadIdx.x - head;
        if (i < vocab) f(Elem<T>::load1(x + i), i);
    }
};

// ---- sums over a workgroup ------------------------------------------------------------------------------------------------------------------------------
struct Mass { uint64_t count, weight; };                   // tokens, and their weights

struct Shared {
    uint32_t count[kBins];
    uint64_t weight[kBins];
    uint64_t candidates[kCandidates], sorted[kCandidates];
    Mass partial[kWaves];
    uint64_t word[4];
    uint32_t number;
};

__device__ __forceinline__ uint64_t shuffle_up(uint64_t v, int by) { return __shfl_up((unsigned long long)v, by, 64); }

// Sums over the threads in front of this one, and over all.
__device__ __forceinline__ Mass scan(Shared& s, Mass v, Mass& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Mass upto = v;
#pragma unroll
    for (int by = 1; by < 64; by *= 2) {
        const uint64_t c = shuffle_up(upto.count, by), w = shuffle_up(upto.weight, by);
        if (lane >= by) { upto.count += c; upto.weight += w; }
    }
    __syncthreads();
    if (lane == 63) s.partial[wave] = upto;
    __syncthreads();
    Mass before{0, 0};
    all = Mass{0, 0};
    for (int w = 0; w < kWaves; ++w) {
        const Mass m = s.partial[w];
        if (w < wave) { before.count += m.count; before.weight += m.weight; }
        all.count += m.count;
        all.weight += m.weight;
    }
    return Mass{before.count + upto.count - v.count, before.weight + upto.weight - v.weight};
}

// ---- weights --------------------------------------------------------------------------------------------------------------------------------------------
struct Weights {
    float largest;                                         // value
    double inverse;                                        // 1 / T
    int bits;                                              // F
    __device__ __forceinline__ double log_of(float x) const {
        if (x == largest) return 0.0;
        return largest == INFINITY ? -INFINITY : ((double)x - (double)largest) * inverse;
    }
    __device__ __forceinline__ double of(float x) const { return exp(log_of(x)); }
    // ... times 2^F as a whole number: 2^F <= 2^51, so in a sum with 2^52 it is what the mantissa holds
    __device__ __forceinline__ uint64_t whole(double w) const { return (uint64_t)__double_as_longlong(ldexp(w, bits) + 0x1p52) & ((1ull << 52) - 1); }
    __device__ __forceinline__ uint64_t whole_of(float x) const { return whole(of(x)); }
};

// ---- searches -------------------------------------------------------------------------------------------------------------------------------------------
// Values of an interval of keys in kBins bins, largest first: of equal width in value, or in key.
struct Bins {
    uint32_t lo, hi;
    float top, scale;                                      // scale 0: by key
    int shift;
    __device__ __forceinline__ bool holds(uint32_t key) const { return key >= lo && key <= hi; }
    __device__ __forceinline__ int of(float x, uint32_t key) const {
        return scale > 0.f ? min((int)((top - x) * scale), kBins - 1) : (int)((hi - key) >> shift);
    }
};

struct Found {
    uint32_t key;                                          // of the token
    int index;                                             // -1 unless asked for
    Mass upto;                                             // tokens up to it, it included
};

template <typename T> struct Search {
    Shared& s;
    const Row<T>& row;
    const Weights& weights;
    Bins first;                                            // of the whole row
    bool filled = false;                                   // with them

    __device__ __forceinline__ void fill(const Bins& bins) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) { s.count[i] = 0; s.weight[i] = 0; }
        __syncthreads();
        row.each([&](float x, int) {
            const uint32_t key = value_key(x);
            if (key == 0 || !bins.holds(key)) return;
            const int b = bins.of(x, key);
            atomicAdd(&s.count[b], 1u);
            atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)weights.whole_of(x));
        });
        __syncthreads();
    }

    // The bin in which the count or weight reaches `goal`, with what lies in front of it.
    __device__ __forceinline__ int bin_of(bool by_count, uint64_t goal, Mass& before) {
        constexpr int kEach = kBins / kThreads;
        Mass mine{0, 0}, all;
        for (int i = 0; i < kEach; ++i) { mine.count += s.count[kEach * threadIdx.x + i]; mine.weight += s.weight[kEach * threadIdx.x + i]; }
        Mass at = scan(s, mine, all);
        at.count += before.count;
        at.weight += before.weight;
        if (threadIdx.x == 0) s.number = 0;
        __syncthreads();
        for (int i = 0; i < kEach; ++i) {
            const int b = kEach * threadIdx.x + i;
            const Mass next{at.count + s.count[b], at.weight + s.weight[b]};
            if (by_count ? at.count < goal && next.count >= goal : at.weight < goal && next.weight >= goal) {
                s.number = b;
                s.word[0] = at.count;
                s.word[1] = at.weight;
            }
            at = next;
        }
        __syncthreads();
        const int b = (int)s.number;
        before = Mass{s.word[0], s.word[1]};
        return b;
    }

    // The first token up to which there are `goal` tokens, or there is that much weight: at least 1, at most what there is.
    __device__ __forceinline__ Found find(bool by_count, uint64_t goal, bool want_index) {
        Bins bins = first;
        Mass before{0, 0};
        if (!filled) { fill(bins); filled = true; }
        for (;;) {
            const int bin = bin_of(by_count, goal, before);
            const uint32_t n = s.count[bin];
            const auto in_bin = [&](float x, uint32_t key) { return key != 0 && bins.holds(key) && bins.of(x, key) == bin; };
            if (n <= kCandidates) return among(in_bin, (int)n, by_count, goal, before);
            uint32_t lo = 0xffffffffu, hi = 0;
            row.each([&](float x, int) {
                const uint32_t key = value_key(x);
                if (in_bin(x, key)) { lo = min(lo, key); hi = max(hi, key); }
            });
            __syncthreads();
            if (threadIdx.x == 0) { s.word[2] = 0xffffffffu; s.word[3] = 0; }
            __syncthreads();
            atomicMin((unsigned int*)&s.word[2], lo);
            atomicMax((unsigned int*)&s.word[3], hi);
            __syncthreads();
            lo = (uint32_t)s.word[2];
            hi = (uint32_t)s.word[3];
            __syncthreads();
            if (lo == hi) return equals(lo, n, by_count, goal, before, want_index);
            bins = Bins{lo, hi, 0.f, 0.f, max(0, 32 - (int)__builtin_clz(hi - lo) - 12)};
            fill(bins);
            filled = false;
        }
    }

    // ... of the few tokens of a bin
    template <class F> __device__ __forceinline__ Found among(const F& in_bin, int n, bool by_count, uint64_t goal, Mass before) {
        __syncthreads();
        if (threadIdx.x == 0) s.number = 0;
        __syncthreads();
        row.each([&](float x, int i) {
            const uint32_t key = value_key(x);
            if (!in_bin(x, key)) return;
            s.candidates[min(atomicAdd(&s.number, 1u), (uint32_t)kCandidates - 1)] = (uint64_t)~key << 32 | (uint32_t)i;
        });
        __syncthreads();
        Mass mine{0, 0}, all;
        if ((int)threadIdx.x < n) {
            const uint64_t c = s.candidates[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < n; ++i) rank += s.candidates[i] < c;
            s.sorted[rank] = c;
        }
        __syncthreads();
        uint32_t key = 0;
        int index = 0;
        if ((int)threadIdx.x < n) {
            key = ~(uint32_t)(s.sorted[threadIdx.x] >> 32);
            index = (int)(uint32_t)s.sorted[threadIdx.x];
            mine = Mass{1, weights.whole_of(key_value(key))};
        }
        Mass at = scan(s, mine, all);
        at.count += before.count;
        at.weight += before.weight;
        const Mass next{at.count + mine.count, at.weight + mine.weight};
        if (by_count ? at.count < goal && next.count >= goal : at.weight < goal && next.weight >= goal) {
            s.word[0] = next.count;
            s.word[1] = next.weight;
            s.word[2] = key;
            s.word[3] = (uint32_t)index;
        }
        __syncthreads();
        const Found f{(uint32_t)s.word[2], (int)(uint32_t)s.word[3], Mass{s.word[0], s.word[1]}};
        __syncthreads();
        return f;
    }

    // ... of n equal tokens
    __device__ __forceinline__ Found equals(uint32_t key, uint32_t n, bool by_count, uint64_t goal, Mass before, bool want_index) {
        const uint64_t w = weights.whole_of(key_value(key));
        uint64_t nth = by_count ? goal - before.count : w > 0 ? (goal - before.weight + w - 1) / w : 1;       // 1 .. n
        nth = nth < 1 ? 1 : nth > n ? n : nth;
        Found f{key, -1, Mass{before.count + nth, before.weight + nth * w}};
        if (!want_index) return f;
        // bins of equal width in the index
        const int width = (row.vocab + kBins - 1) / kBins;
        filled = false;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) { s.count[i] = 0; s.weight[i] = 0; }
        __syncthreads();
        row.each([&](float x, int i) { if (value_key(x) == key) atomicAdd(&s.count[i / width], 1u); });
        __syncthreads();
        Mass none{0, 0};
        const int bin = bin_of(true, nth, none);
        if (threadIdx.x == 0) {
            uint64_t left = nth - none.count;
            for (int i = bin * width; i < row.vocab && i < (bin + 1) * width; ++i)
                if (value_key(Elem<T>::load1(row.x + i)) == key && --left == 0) { s.word[3] = i; break; }
        }
        __syncthreads();
        f.index = (int)s.word[3];
        return f;
    }
};

// One workgroup per row.
template <typename T> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams p) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const Row<T> row(p, r);
    // ---- parameters (compared as bits: comparisons with NaN are compiled away) ----
    const uint32_t t_bits = __float_as_uint(p.temperature ? p.temperature[r] : p.temperature0);
    const bool greedy = t_bits - 1u >= 0x7f800000u;        // zero, negative, NaN
    const uint32_t u_bits = __float_as_uint(p.uniforms[r]);
    const float u = u_bits >= 0x80000000u || u_bits > 0x7f800000u ? 0.f : __uint_as_float(min(u_bits, 0x3f7fffffu));
    const uint32_t p_bits = __float_as_uint(p.top_p ? p.top_p[r] : p.top_p0), m_bits = __float_as_uint(p.min_p ? p.min_p[r] : p.min_p0);
    int k = p.top_k ? p.top_k[r] : p.top_k0;
    if (greedy) k = 1;
    // ---- the largest and the smallest value with a weight ----
    uint32_t lo = 0xffffffffu, hi = 0;
    row.each([&](float x, int) {
        const uint32_t key = value_key(x);
        if (key != 0) { lo = min(lo, key); hi = max(hi, key); }
    });
    if (threadIdx.x == 0) { s.word[2] = 0xffffffffu; s.word[3] = 0; }
    __syncthreads();
    atomicMin((unsigned int*)&s.word[2], lo);
    atomicMax((unsigned int*)&s.word[3], hi);
    __syncthreads();
    lo = (uint32_t)s.word[2];
    hi = (uint32_t)s.word[3];
    __syncthreads();
    if (hi == 0) {                                         // nothing to draw from
        if (threadIdx.x == 0) {
            p.ids[r] = 0;
            if (p.logprobs) p.logprobs[r] = -INFINITY;
        }
        return;
    }
    Weights w;
    w.largest = key_value(hi);
    w.inverse = greedy ? 1.0 : 1.0 / (double)__uint_as_float(t_bits);
    w.bits = min(51, 30 + __builtin_clz((unsigned)row.vocab));        // all tokens' sum stays under 2^62
    Search<T> search{s, row, w, Bins{lo, hi, w.largest, 0.f, 0}};
    const float range = w.largest - key_value(lo);
    search.first.scale = range > 0.f && range < INFINITY ? (float)kBins / range : 0.f;
    if (!(search.first.scale < INFINITY)) search.first.scale = 0.f;
    if (search.first.scale == 0.f) search.first.shift = hi > lo ? max(0, 32 - (int)__builtin_clz(hi - lo) - 12) : 0;
    // ---- what is kept: so much weight ----
    search.fill(search.first);
    search.filled = true;
    Mass mine{0, 0}, all;
    for (int i = threadIdx.x; i < kBins; i += kThreads) { mine.count += s.count[i]; mine.weight += s.weight[i]; }
    scan(s, mine, all);
    uint64_t kept = all.weight;
    if (k > 0 && (uint64_t)k < all.count) kept = search.find(true, (uint64_t)k, false).upto.weight;
    const uint64_t one = 1ull << w.bits;
    const uint64_t of_k = kept;
    if (p_bits >= 0x80000000u && p_bits <= 0xff800000u) {  // negative
        kept = one;
    } else if (p_bits < 0x3f800000u) {
        const double goal = ceil((double)of_k * (double)__uint_as_float(p_bits));
        kept = search.find(false, goal < 1.0 ? 1 : (uint64_t)goal, false).upto.weight;
    }
    if (m_bits - 1u < 0x7f800000u) {
        const double least = (double)__uint_as_float(m_bits);
        Mass heavy{0, 0};
        row.each([&](float x, int) {
            if (value_key(x) == 0) return;
            const double v = w.of(x);
            if (v >= least) heavy.weight += w.whole(v);
        });
        scan(s, heavy, all);
        kept = min(kept, max(all.weight, one));
    }
    // ---- the token ----
    const uint64_t goal = (uint64_t)((double)kept * (double)u) + 1;
    const Found f = search.find(false, min(goal, kept), true);
    if (threadIdx.x == 0) {
        p.ids[r] = f.index;
        if (p.logprobs) p.logprobs[r] = (float)(w.log_of(key_value(f.key)) - log(ldexp((double)kept, -w.bits)));
    }
}

}  // namespace

extern "C" int mi_sample(const mi_sample_args* a) {
    if (!a) return mi_fail(MI_E_NULL, "sample: args is null");
    if (a->n_rows == 0) return MI_OK;
    if (a->n_rows < 0 || a->n_rows > 0x7fffffffLL || a->vocab < 1 || a->vocab > MI_SAMPLE_VOCAB_MAX || a->row_stride < 0)
        return mi_fail(MI_E_SHAPE, "sample: %lld rows of %lld logits (1 to %d), %lld apart", (long long)a->n_rows, (long long)a->vocab, MI_SAMPLE_VOCAB_MAX,
                       (long long)a->row_stride);
    if (!a->logits || !a->uniforms || !a->ids) return mi_fail(MI_E_NULL, "sample: null pointer");
    const SampleParams p{a->logits, a->row_stride, (int)a->vocab, a->uniforms, a->temperatures, a->top_ps, a->min_ps, a->top_ks, a->temperature, a->top_p, a->min_p,
                         a->top_k, a->ids, a->logprobs};
    MI_DISPATCH_DTYPE(a->dtype, sample_kernel<T><<<dim3((unsigned)a->n_rows), dim3(kThreads), 0, (hipStream_t)a->stream>>>(p));
    return mi_check_launch("sample");
}

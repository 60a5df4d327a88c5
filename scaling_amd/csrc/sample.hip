// A token of every row of logits by temperature, top-k, top-p and min-p, from one given random number a row.
//
// A row's tokens are ordered by value, largest first, equal ones by index; token i weighs w_i = exp((x_i - max) / T).  Each of top-k (the first k), top-p (the
// fewest with p of their weight together) and min-p (those of at least min_p of the largest weight) keeps the first so many in that order, so all do, and the token is
// the first one behind which the running sum S of weights exceeds u times the sum of what is kept.  No order of the row is ever made: every question is "the
// first token with S (or the number of tokens) of at least G", and sums over bins of values answer it.  Sums are of whole numbers (weights times 2^F),
// exact in any order, so that atomics leave no trace of theirs; the weights themselves are rounded once, from 64-bit exponentials, as u lies close to a border in
// one row of some thousands where 32 bits are all there is.
#include "common.h"

#include <stddef.h>

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

// Values of keys lo to hi as a test of a value's bits: its positive and its negative part, with both zeros where zero is in it (one of two parts that are alike, where
// there is only one).  NaN is in none.
struct Interval {
    uint32_t a0, n0, a1, n1;
    __device__ __forceinline__ Interval(uint32_t lo, uint32_t hi) {
        constexpr uint32_t kZero = 0x80000000u;
        if (hi == kZero - 1) --hi;                         // (no value's key; its bits are those of -0)
        a0 = lo > kZero ? lo & 0x7fffffffu : 0;
        n0 = (hi & 0x7fffffffu) - a0;
        a1 = hi >= kZero ? kZero : ~hi;
        n1 = (lo < kZero ? ~lo : kZero) - a1;
        if (hi < kZero) { a0 = a1; n0 = n1; }
        if (lo > kZero) { a1 = a0; n1 = n0; }
    }
    __device__ __forceinline__ bool holds(float x) const {
        const uint32_t u = __float_as_uint(x);
        return (u - a0 <= n0) | (u - a1 <= n1);
    }
};
// The smallest key of lo to hi that `reached` holds for, as it does for all above and for hi: 64 keys at a time by a wavefront.
template <class F> __device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, const F& reached) {
    const uint32_t lane = threadIdx.x & 63;
    while (lo < hi) {
        const uint32_t n = hi - lo, step = n / 64 + 1, at = lane * step <= n ? lo + lane * step : hi;
        const uint64_t those = __ballot(reached(at));
        if (those == 0) {                                  // (lane 63 may be short of hi)
            lo = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + 1;
            continue;
        }
        const int l = __builtin_ctzll(those);
        hi = (uint32_t)__builtin_amdgcn_readlane((int)at, l);
        if (l == 0) break;
        lo = (uint32_t)__builtin_amdgcn_readlane((int)at, l - 1) + 1;
    }
    return hi;
}

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
    // f(value, index) of every element; the next vectors are under way while these are looked at
    template <class F> __device__ __forceinline__ void each(const F& f) const {
        const uint4* at = reinterpret_cast<const uint4*>(x + head);
        const int last = vecs - 1;
        uint4 u[kAhead];
        if (vecs > 0) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) u[a] = at[min((int)threadIdx.x + a * kThreads, last)];
        }
#pragma unroll 1
        for (int v0 = threadIdx.x; v0 < vecs; v0 += kAhead * kThreads) {
            uint4 now[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                now[a] = u[a];
                u[a] = at[min(v0 + (kAhead + a) * kThreads, last)];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int v = v0 + a * kThreads;
                if (v >= vecs) break;
                float e[V];
                Elem<T>::unpack(now[a], e);
#pragma unroll
                for (int i = 0; i < V; ++i) f(e[i], head + v * V + i);
            }
        }
        const int behind = head + vecs * V, i = (int)threadIdx.x < head ? (int)threadIdx.x : behind + (int)threadIdx.x - head;
        if (i < vocab) f(Elem<T>::load1(x + i), i);
    }
    // f(value, index) of the elements of an interval, which are few: they are marked first, up to 64 a thread, and then fetched once more, so that a wavefront
    // takes as many turns as its lane with the most of them has, and not one for every element.  (us of 448 of 49999: 4.2, an element after the other 6.0.)
    template <class F> __device__ __forceinline__ void select(const Interval& those, const F& f) const {
        static_assert(V == 4 && kAhead == 4);
        const uint4* at = reinterpret_cast<const uint4*>(x + head);
        const int last = vecs - 1;
        uint4 u[kAhead];
        if (vecs > 0) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) u[a] = at[min((int)threadIdx.x + a * kThreads, last)];
        }
        for (int v0 = threadIdx.x; v0 < vecs;) {
            const int first = v0;
            uint64_t marked = 0;
#pragma unroll 1
            for (int g = 48; g >= 0 && v0 < vecs; g -= 16, v0 += kAhead * kThreads) {
                uint32_t bits = 0;
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const uint4 now = u[a];
                    u[a] = at[min(v0 + (kAhead + a) * kThreads, last)];
                    float e[V];
                    Elem<T>::unpack(now, e);
#pragma unroll
                    for (int i = 0; i < V; ++i) bits = 2 * bits + those.holds(e[i]);
                }
                const int there = min((vecs - v0 + kThreads - 1) / kThreads, kAhead);      // (the others repeat the last vector)
                bits &= 0xffff0000u >> (V * there);
                marked |= (uint64_t)(bits & 0xffffu) << g;
            }
            while (marked != 0) {
                const int e = __builtin_clzll(marked), i = head + (first + (e >> 2) * kThreads) * V + (e & 3);
                marked &= ~(1ull << (63 - e));
                f(Elem<T>::load1(x + i), i);
            }
        }
        const int behind = head + vecs * V, i = (int)threadIdx.x < head ? (int)threadIdx.x : behind + (int)threadIdx.x - head;
        if (i < vocab) {
            const float v = Elem<T>::load1(x + i);
            if (those.holds(v)) f(v, i);
        }
    }
};

// A few tokens of a row that were gathered in LDS, in any order: complements of their keys over their indexes.
struct Gathered {
    const uint64_t* tokens;
    int n;
    template <class F> __device__ __forceinline__ void each(const F& f) const {
        for (int i = threadIdx.x; i < n; i += kThreads) f(key_value(~(uint32_t)(tokens[i] >> 32)), (int)(uint32_t)tokens[i]);
    }
    template <class F> __device__ __forceinline__ void select(const Interval& those, const F& f) const {
        each([&](float x, int i) { if (those.holds(x)) f(x, i); });
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

// Sums over lanes 0 .. this one of numbers that add up to less than 2^62, as three of 26 bits (64 of which fit 32): lane exchanges of 64 bits through LDS take
// longer than the rest of a search.
__device__ __forceinline__ uint64_t prefix_sum64(uint64_t v) {
    constexpr uint32_t kPart = (1u << 26) - 1;
    const uint32_t a = (uint32_t)prefix_sum((int)((uint32_t)v & kPart)), b = (uint32_t)prefix_sum((int)((uint32_t)(v >> 26) & kPart)), c = (uint32_t)prefix_sum((int)(uint32_t)(v >> 52));
    return ((uint64_t)c << 52) + ((uint64_t)b << 26) + a;
}
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

// Sum over the lanes: 16 lanes by exchanges, then the four sums.
__device__ __forceinline__ uint64_t sum64(uint64_t v) {
    const auto step = [&](auto ctrl) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, decltype(ctrl)::value, 0xf, 0xf, true);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), decltype(ctrl)::value, 0xf, 0xf, true);
        v += __builtin_bit_cast(uint64_t, make_uint2(lo, hi));
    };
    step(std::integral_constant<int, 0xB1>{});            // quad_perm [1, 0, 3, 2]
    step(std::integral_constant<int, 0x4E>{});            // quad_perm [2, 3, 0, 1]
    step(std::integral_constant<int, 0x141>{});           // row_half_mirror
    step(std::integral_constant<int, 0x140>{});           // row_mirror
    return of_lane(v, 0) + of_lane(v, 16) + of_lane(v, 32) + of_lane(v, 48);
}

// Sums over the threads in front of this one, and over all.
__device__ __forceinline__ Mass scan(Mass* partial, Mass v, Mass& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Mass upto{prefix_sum64(v.count), prefix_sum64(v.weight)};
    __syncthreads();
    if (lane == 63) partial[wave] = upto;
    __syncthreads();
    Mass of_wave{0, 0};
    if (lane < kWaves) of_wave = partial[lane];
    of_wave = Mass{prefix_sum64(of_wave.count), prefix_sum64(of_wave.weight)};
    all = Mass{of_lane(of_wave.count, kWaves - 1), of_lane(of_wave.weight, kWaves - 1)};
    const Mass before = wave > 0 ? Mass{of_lane(of_wave.count, wave - 1), of_lane(of_wave.weight, wave - 1)} : Mass{0, 0};
    return Mass{before.count + upto.count - v.count, before.weight + upto.weight - v.weight};
}

__device__ __forceinline__ uint64_t scan(Mass* partial, uint64_t v, uint64_t& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t upto = prefix_sum64(v);
    __syncthreads();
    if (lane == 63) partial[wave].count = upto;
    __syncthreads();
    const uint64_t of_wave = prefix_sum64(lane < kWaves ? partial[lane].count : 0);
    all = of_lane(of_wave, kWaves - 1);
    return (wave > 0 ? of_lane(of_wave, wave - 1) : 0) + upto - v;
}

// ---- weights --------------------------------------------------------------------------------------------------------------------------------------------
// 2^x for x <= 0, to 2^-47 of it: a whole power of two and the Taylor series of exp(f ln 2) for the rest f, of which 12 terms leave (ln 2 / 2)^12 / 12! = 6e-15.
// (The library's is half again as long, for the last bits and for arguments that there are none of here.)
__device__ __forceinline__ double scaled_exp2(double x, int scale) {
    const double whole = __builtin_rint(x), f = (x - whole) * 0.693147180559945309417;
    double y = 1.0 / 39916800;
    constexpr double kTerms[11] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800};
#pragma unroll
    for (int i = 10; i >= 0; --i) y = __builtin_fma(y, f, kTerms[i]);
    return ldexp(y, (int)fmax(whole, -2000.0) + scale);
}

struct Weights {
    float largest;                                         // value
    double inverse, slope;                                 // 1 / T, and this over ln 2
    int bits;                                              // F
    __device__ __forceinline__ Weights(float l, double i, int b) : largest(l), inverse(i), slope(i * 1.44269504088896340736), bits(b) {}
    __device__ __forceinline__ double log_of(float x) const {
        if (x == largest) return 0.0;
        return largest == INFINITY ? -INFINITY : ((double)x - (double)largest) * inverse;
    }
    // a token's weight times 2^F
    __device__ __forceinline__ double of(float x) const {
        if (largest == INFINITY) return x == largest ? ldexp(1.0, bits) : 0.0;
        return scaled_exp2(((double)x - (double)largest) * slope, bits);
    }
    // ... as a whole number: 2^F <= 2^51, so in a sum with 2^52 it is what the mantissa holds
    __device__ __forceinline__ uint64_t whole(double w) const { return (uint64_t)__double_as_longlong(w + 0x1p52) & ((1ull << 52) - 1); }
    __device__ __forceinline__ uint64_t whole_of(float x) const { return whole(of(x)); }
};
// count * w for w < 2^52
__device__ __forceinline__ uint64_t times(uint32_t count, uint64_t w) { return (uint64_t)count * (uint32_t)w + ((uint64_t)(count * (uint32_t)(w >> 32)) << 32); }

// ceil(a / b) for 0 < a < 2^62, 0 < b <= 2^51 and a quotient under 2^31
__device__ __forceinline__ uint64_t ceil_quotient(uint64_t a, uint64_t b) {
    uint64_t q = (uint64_t)(uint32_t)((double)a / (double)b);              // or one off
    q += q * b < a;
    q += q * b < a;
    return q > 1 && (q - 1) * b >= a ? q - 1 : q;
}

// The smallest lo and the largest hi of all threads.
__device__ __forceinline__ void range(Shared& s, uint32_t& lo, uint32_t& hi) {
    lo = group_reduce_bits<64>(lo, [](uint32_t a, uint32_t b) { return min(a, b); });
    hi = group_reduce_bits<64>(hi, [](uint32_t a, uint32_t b) { return max(a, b); });
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.partial[threadIdx.x >> 6] = Mass{lo, hi};
    __syncthreads();
    const int w = threadIdx.x & (kWaves - 1);
    lo = group_reduce_bits<16>((uint32_t)s.partial[w].count, [](uint32_t a, uint32_t b) { return min(a, b); });
    hi = group_reduce_bits<16>((uint32_t)s.partial[w].weight, [](uint32_t a, uint32_t b) { return max(a, b); });
    static_assert(kWaves == 16);
    __syncthreads();
}

// ---- searches -------------------------------------------------------------------------------------------------------------------------------------------
// Values of keys lo to hi in kBins bins, largest first: of equal width in value, or in key.
struct Bins {
    uint32_t lo, hi;
    float top, scale;                                      // scale 0: by key
    int shift;
    // of equal width in value where the range allows
    static __device__ __forceinline__ Bins over(uint32_t lo, uint32_t hi) {
        const float top = key_value(hi), range = top - key_value(lo), scale = (float)kBins / range;
        return range > 0.f && range < INFINITY && scale < INFINITY ? Bins{lo, hi, top, scale, 0} : Bins{lo, hi, 0.f, 0.f, hi > lo ? max(0, 32 - (int)__builtin_clz(hi - lo) - 12) : 0};
    }
    __device__ __forceinline__ int of(float x) const { return scale > 0.f ? min((int)((top - x) * scale), kBins - 1) : (int)((hi - value_key(x)) >> shift); }
    // the smallest key of bins 0 to `bin`
    __device__ __forceinline__ uint32_t from(int bin) const {
        return first_key(lo, hi, [&](uint32_t key) { return of(key_value(key)) <= bin; });
    }
    // what a bin, that holds something, holds
    __device__ __forceinline__ Interval interval(int bin) const { return Interval(from(bin), bin > 0 ? from(bin - 1) - 1 : hi); }
};

struct Found {
    uint32_t key;                                          // of the token
    int index;                                             // -1 unless asked for
    uint64_t upto;                                         // tokens up to it, it included, or their weight
};

// Searches by count or by weight, in bins that hold the one or the other: adding to LDS is what a pass over a row waits for.  (us of 64 x 128256 by top-p: 111 with
// both, 100.)
template <typename T, class ROW> struct Search {
    Shared& s;
    const ROW& row;                                        // the tokens that are looked at
    const Row<T>& whole;
    const Weights& weights;
    bool weighed;                                          // bins of weights, or of counts
    Bins first;
    bool filled;                                           // with the first bins
    uint32_t passed;                                       // tokens in them, of this thread's

    __device__ __forceinline__ uint64_t in(int bin) const { return weighed ? s.weight[bin] : s.count[bin]; }
    __device__ __forceinline__ void fill(const Bins& bins) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            if (weighed) s.weight[i] = 0;
            else s.count[i] = 0;
        }
        __syncthreads();
        const Interval asked(bins.lo, bins.hi);
        uint32_t n = 0;
        row.each([&](float x, int) {
            if (!asked.holds(x)) return;
            const int b = bins.of(x);
            ++n;
            if (weighed) atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)weights.whole_of(x));
            else atomicAdd(&s.count[b], 1u);
        });
        passed = n;
        __syncthreads();
    }
    // All tokens of keys lo to hi, lo at least 1.
    __device__ __forceinline__ void take(uint32_t lo, uint32_t hi, bool with_weights) {
        weighed = with_weights;
        first = Bins::over(lo, hi);
        fill(first);
        filled = true;
    }

    // What all bins hold.
    __device__ __forceinline__ uint64_t all() const {
        uint64_t mine = 0, sum;
        for (int i = threadIdx.x; i < kBins; i += kThreads) mine += in(i);
        scan(s.partial, mine, sum);
        return sum;
    }
    __device__ __forceinline__ uint64_t tokens() const {
        uint64_t sum;
        scan(s.partial, (uint64_t)passed, sum);
        return sum;
    }

    // The bin in which what `value` gives reaches `goal`, with what lies in front of it.
    template <class F> __device__ __forceinline__ int bin_of(const F& value, uint64_t goal, uint64_t& before) {
        constexpr int kEach = kBins / kThreads;
        uint64_t mine = 0, all;
        for (int i = 0; i < kEach; ++i) mine += value(kEach * threadIdx.x + i);
        uint64_t at = scan(s.partial, mine, all) + before;
        if (threadIdx.x == 0) s.number = 0;
        __syncthreads();
        for (int i = 0; i < kEach; ++i) {
            const int b = kEach * threadIdx.x + i;
            const uint64_t next = at + value(b);
            if (at < goal && next >= goal) {
                s.number = b;
                s.word[0] = at;
            }
            at = next;
        }
        __syncthreads();
        before = s.word[0];
        return (int)s.number;
    }
    __device__ __forceinline__ int bin_of(uint64_t goal, uint64_t& before) {
        return bin_of([&](int b) { return in(b); }, goal, before);
    }

    // The first token up to which there are `goal` tokens, or there is that much weight: at least 1, at most what there is.
    __device__ __forceinline__ Found find(uint64_t goal, bool want_index) {
        Bins bins = first;
        uint64_t before = 0;
        if (!filled) { fill(bins); filled = true; }
        for (;;) {
            const int bin = bin_of(goal, before);
            const Interval in_bin = bins.interval(bin);
            uint32_t n = weighed ? 0 : s.count[bin];
            if (n <= kCandidates) {
                n = collect(in_bin);
                if (n <= kCandidates) return among((int)n, goal, before);
            }
            uint32_t lo = 0xffffffffu, hi = 0;
            row.each([&](float x, int) {
                if (!in_bin.holds(x)) return;
                const uint32_t key = value_key(x);
                lo = min(lo, key);
                hi = max(hi, key);
            });
            range(s, lo, hi);
            if (lo == hi) return equals(lo, n, goal, before, want_index);
            bins = Bins{lo, hi, 0.f, 0.f, max(0, 32 - (int)__builtin_clz(hi - lo) - 12)};
            fill(bins);
            filled = false;
        }
    }

    // The tokens of an interval, as far as there is room; how many there are.
    __device__ __forceinline__ uint32_t collect(const Interval& those) {
        __syncthreads();
        if (threadIdx.x == 0) s.number = 0;
        __syncthreads();
        row.select(those, [&](float x, int i) {
            const uint32_t at = atomicAdd(&s.number, 1u);
            if (at < (uint32_t)kCandidates) s.candidates[at] = (uint64_t)~value_key(x) << 32 | (uint32_t)i;
        });
        __syncthreads();
        const uint32_t n = s.number;
        __syncthreads();
        return n;
    }

    // ... of the few tokens of a bin
    __device__ __forceinline__ Found among(int n, uint64_t goal, uint64_t before) {
        if ((int)threadIdx.x < n) {
            const uint64_t c = s.candidates[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < n; ++i) rank += s.candidates[i] < c;
            s.sorted[rank] = c;
        }
        __syncthreads();
        uint32_t key = 0;
        int index = 0;
        uint64_t mine = 0, all;
        if ((int)threadIdx.x < n) {
            key = ~(uint32_t)(s.sorted[threadIdx.x] >> 32);
            index = (int)(uint32_t)s.sorted[threadIdx.x];
            mine = weighed ? weights.whole_of(key_value(key)) : 1;
        }
        const uint64_t at = scan(s.partial, mine, all) + before;
        if (at < goal && at + mine >= goal) {
            s.word[0] = at + mine;
            s.word[2] = key;
            s.word[3] = (uint32_t)index;
        }
        __syncthreads();
        const Found f{(uint32_t)s.word[2], (int)(uint32_t)s.word[3], s.word[0]};
        __syncthreads();
        return f;
    }

    // ... of n equal tokens
    __device__ __forceinline__ Found equals(uint32_t key, uint32_t n, uint64_t goal, uint64_t before, bool want_index) {
        const uint64_t w = weighed ? weights.whole_of(key_value(key)) : 1;
        uint64_t nth = w > 0 ? ceil_quotient(goal - before, w) : 1;           // 1 .. n
        nth = nth < 1 ? 1 : nth > n ? n : nth;
        Found f{key, -1, before + nth * w};
        if (!want_index) return f;
        // bins of equal width in the index
        const int width = (whole.vocab + kBins - 1) / kBins;
        filled = filled && weighed;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0;
        __syncthreads();
        const Interval equal(key, key);
        row.each([&](float x, int i) { if (equal.holds(x)) atomicAdd(&s.count[i / width], 1u); });
        __syncthreads();
        uint64_t none = 0;
        const int bin = bin_of([&](int b) { return (uint64_t)s.count[b]; }, nth, none);
        if (threadIdx.x == 0) {
            uint64_t left = nth - none;
            for (int i = bin * width; i < whole.vocab && i < (bin + 1) * width; ++i)
                if (value_key(Elem<T>::load1(whole.x + i)) == key && --left == 0) { s.word[3] = i; break; }
        }
        __syncthreads();
        f.index = (int)s.word[3];
        return f;
    }
};

// ---- parameters -----------------------------------------------------------------------------------------------------------------------------------------
// (compared as bits: comparisons with NaN are compiled away)
struct Parameters {
    bool greedy, top_p_none, top_p_one, any_min_p;         // top-p keeps everything, or one token
    int k;
    float u;
    double inverse, top_p, min_p;
    __device__ __forceinline__ Parameters(const SampleParams& p, int64_t r) {
        const uint32_t t_bits = __float_as_uint(p.temperature ? p.temperature[r] : p.temperature0), u_bits = __float_as_uint(p.uniforms[r]);
        const uint32_t p_bits = __float_as_uint(p.top_p ? p.top_p[r] : p.top_p0), m_bits = __float_as_uint(p.min_p ? p.min_p[r] : p.min_p0);
        k = p.top_k ? p.top_k[r] : p.top_k0;
        greedy = t_bits - 1u >= 0x7f800000u;               // zero, negative, NaN
        if (greedy) k = 1;
        inverse = greedy ? 1.0 : 1.0 / (double)__uint_as_float(t_bits);
        u = u_bits > 0x7f800000u ? 0.f : __uint_as_float(min(u_bits, 0x3f7fffffu));     // negative, NaN: 0
        top_p_one = p_bits >= 0x80000000u && p_bits <= 0xff800000u;
        top_p_none = !top_p_one && p_bits >= 0x3f800000u;
        top_p = (double)__uint_as_float(p_bits);
        any_min_p = m_bits - 1u < 0x7f800000u;
        min_p = (double)__uint_as_float(m_bits);
    }
    // Keys lo to hi, hi the largest: from where on the logarithm of a weight may be `log` or more (a little below the value that this stands for).
    __device__ __forceinline__ uint32_t from(uint32_t lo, uint32_t hi, double log) const {
        const double largest = (double)key_value(hi), at = largest + log / inverse, x = at - 1e-6 * fmax(fabs(at), fabs(largest));
        if (key_value(hi) == INFINITY || !(inverse > 0.0) || !(x > -3e38)) return lo;      // (no float may be lower than x)
        const uint32_t key = value_key((float)x);
        return key > lo && key <= hi ? key : lo;
    }
    __device__ __forceinline__ uint32_t heavy_from(uint32_t lo, uint32_t hi) const { return from(lo, hi, log(min_p)); }
};

// The token of what top-k (k > 0), top-p and min-p leave of the weight `kept`, and how much that is: find(step, goal), of step 0 by count,
// gives the weight up to the first token that reaches the goal.  heavy: the weight of those of at least min_p.  (One call in a loop: the compiler makes three of three, with registers for each.)
template <class F> __device__ __forceinline__ uint64_t draw(const Parameters& p, uint64_t kept, int k, uint64_t one, uint64_t heavy, const F& find) {
#pragma unroll 1
    for (int step = k > 0 ? 0 : 1; step < 3; ++step) {
        uint64_t goal = (uint64_t)k;
        if (step == 1) {
            if (p.top_p_one) kept = one;
            if (p.top_p_one || p.top_p_none) continue;
            const double least = ceil((double)kept * p.top_p);
            goal = least < 1.0 ? 1 : (uint64_t)least;
        }
        if (step == 2) {
            if (p.any_min_p) kept = min(kept, max(heavy, one));
            goal = min((uint64_t)((double)kept * (double)p.u) + 1, kept);
        }
        const uint64_t weight = find(step, goal);
        if (step < 2) kept = weight;
    }
    return kept;
}

__device__ __forceinline__ void write_nothing(const SampleParams& p, int64_t r) {
    if (threadIdx.x != 0) return;
    p.ids[r] = 0;
    if (p.logprobs) p.logprobs[r] = -INFINITY;
}
__device__ __forceinline__ void write_logprob(const SampleParams& p, int64_t r, const Weights& w, float x, uint64_t kept) {      // (by one thread)
    if (p.logprobs) p.logprobs[r] = (float)(w.log_of(x) - log(ldexp((double)kept, -w.bits)));
}
__device__ __forceinline__ int weight_bits(int vocab) { return min(51, 30 + __builtin_clz((unsigned)vocab)); }      // all tokens' sum stays under 2^62

// ---- 32-bit logits --------------------------------------------------------------------------------------------------------------------------------------
// One workgroup per row, for which every pass over it is an exchange with memory.  The first one counts the tokens by the upper 13 bits of their keys, which
// tells from where on top-k asks for tokens; without top-p, min-p does too.  If these are few they are gathered in LDS, and all else happens there.
// 1024 threads leave 128 registers each, of which the searches over a whole row would take more: 36 are spilled (84 bytes of scratch a lane).
constexpr int kGathered = 6144, kCoarse = 19, kCoarseBins = 1 << (32 - kCoarse), kEach = kGathered / kThreads;      // bits of a key below its first bin

// All tokens of keys lo to hi in LDS, of which there are no more than fit.
template <typename T> __device__ __forceinline__ Gathered gather(Shared& s, uint64_t* gathered, const Row<T>& row, uint32_t lo) {
    __syncthreads();
    if (threadIdx.x == 0) s.number = 0;
    __syncthreads();
    const Interval asked(lo, 0xff800000u);
    row.select(asked, [&](float x, int i) { gathered[min(atomicAdd(&s.number, 1u), (uint32_t)kGathered - 1)] = (uint64_t)~value_key(x) << 32 | (uint32_t)i; });
    __syncthreads();
    const Gathered few{gathered, min((int)s.number, kGathered)};
    __syncthreads();
    return few;
}

// Puts gathered tokens of keys from lo on in order: by bins of their values, and in a bin, of which most hold a handful, by comparisons.  False, and nothing done, where one holds many.
__device__ __forceinline__ bool sort(Shared& s, uint64_t* tokens, int n, uint32_t lo, uint32_t hi) {
    uint64_t* scattered = s.weight;
    static_assert(sizeof(s.weight) + sizeof(s.candidates) + sizeof(s.sorted) >= kGathered * sizeof(uint64_t) && offsetof(Shared, candidates) == offsetof(Shared, weight) + sizeof(s.weight) &&
                  offsetof(Shared, sorted) == offsetof(Shared, candidates) + sizeof(s.candidates), "room for the tokens, in one piece");
    constexpr int kMost = 128, kBinsEach = kBins / kThreads;
    const Bins bins = Bins::over(lo, hi);
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0;
    __syncthreads();
    uint64_t token[kEach];
    int bin[kEach];
    uint32_t place[kEach];                                 // among the bin's, in no order
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = threadIdx.x + e * kThreads;
        if (i >= n) break;
        token[e] = tokens[i];
        const uint32_t key = ~(uint32_t)(token[e] >> 32);
        bin[e] = bins.of(key_value(key));
        place[e] = atomicAdd(&s.count[bin[e]], 1u);
    }
    __syncthreads();
    uint32_t count[kBinsEach], most = 0;
    uint64_t all, mine = 0;
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) {
        count[e] = s.count[kBinsEach * threadIdx.x + e];
        mine += count[e];
        most = max(most, count[e]);
    }
    if (__syncthreads_or(most > kMost)) return false;
    uint32_t front = (uint32_t)scan(s.partial, mine, all);
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) { s.count[kBinsEach * threadIdx.x + e] = front; front += count[e]; }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if ((int)threadIdx.x + e * kThreads >= n) break;
        scattered[s.count[bin[e]] + place[e]] = token[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if ((int)threadIdx.x + e * kThreads >= n) break;
        const int from = (int)s.count[bin[e]], end = bin[e] + 1 < kBins ? (int)s.count[bin[e] + 1] : n;
        int rank = from;
        for (int i = from; i < end; ++i) rank += scattered[i] < token[e];
        tokens[rank] = token[e];
    }
    __syncthreads();
    return true;
}

// The token of the first `n` of a row that lie in order, whose running sums answer everything: all of them or, of a row's `whole` weight (0: of these), the first k (k > 0).
__device__ __forceinline__ void sample_sorted(Shared& s, const SampleParams& p, int64_t r, const Parameters& of, const Weights& w, const uint64_t* tokens, int n, int k, uint64_t whole) {
    const uint64_t one = 1ull << w.bits;
    const double least = ldexp(of.min_p, w.bits);
    const int each = (n + kThreads - 1) / kThreads;        // tokens to a thread
    uint64_t weight[kEach], mine = 0, all, heavy = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        weight[e] = 0;
        if (e >= each) continue;
        const int i = each * threadIdx.x + e;
        const double v = i < n ? w.of(key_value(~(uint32_t)(tokens[i] >> 32))) : 0.0;
        weight[e] = i < n ? w.whole(v) : 0;
        mine += weight[e];
        if (of.any_min_p && i < n && v >= least) heavy = mine;
    }
    const uint64_t front = scan(s.partial, mine, all);
    // up to the last one of enough weight
    const int lane = threadIdx.x & 63;
    const uint64_t upto_heavy = of_lane(front + heavy, 63 - __builtin_clzll(__ballot(heavy > 0) | 1)), any = __ballot(heavy > 0);
    __syncthreads();
    if (lane == 0) s.partial[threadIdx.x >> 6].weight = any != 0 ? upto_heavy : 0;
    if (k > 0 && k <= n) {
        uint64_t upto = front;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            upto += weight[e];
            if (e < each && each * (int)threadIdx.x + e == k - 1) s.word[2] = upto;
        }
    }
    __syncthreads();
    const uint64_t of_wave = s.partial[lane & (kWaves - 1)].weight;
    heavy = of_lane(of_wave, 63 - __builtin_clzll((__ballot(of_wave > 0) & 0xffff) | 1));
    if (whole > 0) all = whole;
    else if (k > 0 && k <= n) all = s.word[2];
    const uint64_t kept = draw(of, all, 0, one, heavy, [&](int, uint64_t goal) {
        uint64_t upto = front;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (upto < goal && upto + weight[e] >= goal) { s.word[0] = upto + weight[e]; s.number = each * threadIdx.x + e; }
            upto += weight[e];
        }
        __syncthreads();
        const uint64_t reached = s.word[0];
        __syncthreads();
        return reached;
    });
    if (threadIdx.x == 0) {
        const uint64_t token = tokens[s.number];
        p.ids[r] = (int64_t)(uint32_t)token;
        write_logprob(p, r, w, key_value(~(uint32_t)(token >> 32)), kept);
    }
}

// A value's place among all: the values' order, and below the lowest finite one (kLowest) -inf and NaN.
constexpr uint32_t kPlace = 0x007fffffu, kLowest = 0x00ffffffu;
__device__ __forceinline__ uint32_t place_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) + kPlace;        // (NaN of either sign wraps)
}

// A thread's coarse bins, and how many tokens there are in those down to a key's.
constexpr int kCoarseEach = kCoarseBins / kThreads;
struct CoarseBins {
    uint32_t here[kCoarseEach];
    __device__ __forceinline__ explicit CoarseBins(const uint32_t* coarse) {
        static_assert(kCoarseEach % 4 == 0);
#pragma unroll
        for (int i = 0; i < kCoarseEach; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(coarse + kCoarseEach * threadIdx.x + i);
            here[i] = u.x; here[i + 1] = u.y; here[i + 2] = u.z; here[i + 3] = u.w;
        }
    }
    __device__ __forceinline__ uint64_t from(Shared& s, uint32_t key) const {
        uint64_t mine = 0, all;
#pragma unroll
        for (int i = 0; i < kCoarseEach; ++i)
            if (kCoarseEach * (int)threadIdx.x + i <= (int)(~(key + kPlace) >> kCoarse)) mine += here[i];
        scan(s.partial, mine, all);
        return all;
    }
};

// Of the tokens of keys lo to hi, hi the largest of the row and these the first ones, all or the first k (k > 0).
template <typename T, class ROW>
__device__ __forceinline__ void sample_from(Shared& s, uint64_t* gathered, const SampleParams& p, int64_t r, const Parameters& of, const Row<T>& whole, const ROW& row, uint32_t lo,
                                            uint32_t hi, int k) {
    const Weights w(key_value(hi), of.inverse, weight_bits(whole.vocab));
    const uint64_t one = 1ull << w.bits;
    Search<T, ROW> search{s, row, whole, w, false, {}, false, 0};
    if (k > 0) {
        search.take(lo, hi, false);
        if (search.all() > (uint64_t)k) lo = search.find((uint64_t)k, false).key;
        else k = 0;
    }
    search.take(lo, hi, true);
    uint64_t all = search.all();
    if (k > 0) all -= (search.tokens() - k) * w.whole_of(key_value(lo));      // equals of the k-th token behind it
    const auto finish = [&](auto& search) {
        uint64_t heavy = 0;
        if (of.any_min_p) {
            const double least = ldexp(of.min_p, w.bits);
            uint64_t weight = 0;
            const Interval asked(of.heavy_from(lo, hi), hi);
            search.row.each([&](float x, int) {
                if (!asked.holds(x)) return;
                const double v = w.of(x);
                if (v >= least) weight += w.whole(v);
            });
            scan(s.partial, weight, heavy);
        }
        Found f;
        const uint64_t kept = draw(of, all, 0, one, heavy, [&](int step, uint64_t goal) { f = search.find(goal, step == 2); return f.upto; });
        if (threadIdx.x == 0) {
            p.ids[r] = f.index;
            write_logprob(p, r, w, key_value(f.key), kept);
        }
    };
    if constexpr (std::is_same_v<ROW, Row<T>>) {
        if (!of.top_p_one && !of.top_p_none) {             // what top-p keeps is often few: no more passes over the row
            uint64_t front = 0;
            const double least = ceil((double)all * of.top_p);
            const uint32_t from = search.first.from(search.bin_of(least < 1.0 ? 1 : (uint64_t)least, front));
            if (CoarseBins(reinterpret_cast<const uint32_t*>(gathered)).from(s, from) <= (uint64_t)kGathered) {
                const Gathered few = gather(s, gathered, whole, from);
                if (sort(s, gathered, few.n, from, hi)) return sample_sorted(s, p, r, of, w, gathered, few.n, 0, all);
                Search<T, Gathered> rest{s, few, whole, w, false, {}, false, 0};
                rest.take(from, hi, true);
                return finish(rest);
            }
        }
    }
    finish(search);
}

template <typename T> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams p) {
    __shared__ Shared s;
    __shared__ __attribute__((aligned(16))) uint64_t gathered[kGathered];
    const int64_t r = blockIdx.x;
    const Row<T> row(p, r);
    const Parameters of(p, r);
    uint32_t* coarse = reinterpret_cast<uint32_t*>(gathered);
    static_assert(kCoarseBins * sizeof(uint32_t) <= sizeof(gathered));
    for (int i = threadIdx.x; i < kCoarseBins; i += kThreads) coarse[i] = 0;
    __syncthreads();
    uint32_t n_lowest = 0, most = 0;
    row.each([&](float x, int) {
        const uint32_t at = place_of(x);
        most = max(most, at);
        if (at > kLowest) atomicAdd(&coarse[~at >> kCoarse], 1u);              // largest first
        else n_lowest += at == kLowest;                    // (masked tokens may be many, and adding to one word takes turns)
    });
    n_lowest = group_reduce_bits<64>(n_lowest, [](uint32_t a, uint32_t b) { return a + b; });
    if ((threadIdx.x & 63) == 0 && n_lowest > 0) atomicAdd(&coarse[~kLowest >> kCoarse], n_lowest);
    uint32_t none = 0;
    range(s, none, most);
    if (most < kLowest) return write_nothing(p, r);
    const uint32_t hi = value_key(key_value(most - kPlace));
    const auto edge = [](int bin) { return max((uint32_t)~(((uint64_t)(bin + 1) << kCoarse) - 1), kLowest) - kPlace; };      // the smallest key of a bin
    // ---- from where on tokens are asked for, and how many there are ----
    const CoarseBins bins(coarse);
    const auto& here = bins.here;
    uint64_t mine = 0, n_all;
#pragma unroll
    for (int i = 0; i < kCoarseEach; ++i) mine += here[i];
    uint64_t upto = scan(s.partial, mine, n_all);
    uint32_t lo = kLowest - kPlace;
    const int k = of.k > 0 && (uint64_t)of.k < n_all ? of.k : 0;
    if (k > 0) {
#pragma unroll
        for (int i = 0; i < kCoarseEach; ++i) {
            if (upto < (uint64_t)k && upto + here[i] >= (uint64_t)k) s.word[0] = edge(kCoarseEach * threadIdx.x + i);
            upto += here[i];
        }
        __syncthreads();
        lo = max(lo, (uint32_t)s.word[0]);
    }
    double least = -0.693147180559945309417 * (weight_bits(row.vocab) + 2);             // (those below weigh nothing: no sum, and no search by one, has to do with them)
    if (of.any_min_p && of.top_p_none) least = fmax(least, log(of.min_p));
    lo = of.from(lo, hi, least);
    if (lo == kLowest - kPlace) {                          // the lowest there is
        uint32_t last = 0;
#pragma unroll
        for (int i = 0; i < kCoarseEach; ++i)
            if (here[i] > 0) last = kCoarseEach * threadIdx.x + i;
        range(s, none, last);
        lo = edge((int)last);
    }
    if (bins.from(s, lo) > kGathered) return sample_from<T>(s, gathered, p, r, of, row, row, lo, hi, k);
    const Gathered few = gather(s, gathered, row, lo);
    if (sort(s, gathered, few.n, lo, hi)) return sample_sorted(s, p, r, of, Weights(key_value(hi), of.inverse, weight_bits(row.vocab)), gathered, few.n, k, 0);
    sample_from<T>(s, gathered, p, r, of, row, few, lo, hi, k);
}

// ---- 16-bit logits --------------------------------------------------------------------------------------------------------------------------------------
// There are 2^16 values, so a workgroup counts how often each occurs in its row: equal tokens weigh the same, and everything else is arithmetic on the
// few thousand values that occur, with one exponential each.  Up to 16 vectors a thread of the row (131072 logits) stay in
// registers: a second pass finds which of the tokens that equal the drawn value is meant.  Counts of
// 16 bits, of x and -x in one word of LDS, are 128 KB.  One of more than 65535 equal tokens overflows, which shows as counts that do not add up: then
// once more, in pieces of 32768 tokens with counts over 32767 put aside in between.
constexpr int kMagnitudes = 1 << 15, kUnit = 64, kUnits = 2 * kMagnitudes / kUnit, kAside = MI_SAMPLE_VOCAB_MAX / 32768;

struct KeyShared {
    uint32_t counts[kMagnitudes];                          // of a magnitude's bits: positive values in the lower half
    uint64_t unit_weight[kUnits + 1];                      // of units of 64 keys that occur, largest first: sums in front; of all
    uint32_t unit_count[kUnits + 1];
    uint16_t units[kUnits];
    Mass partial[kWaves];
    uint64_t heavy;
    uint32_t occupied[kWaves];
    int found, index, nth, n_aside;
    uint32_t frequent, n_frequent;                         // bits of a value that many tokens have, and how many of them are not in the counts
    uint32_t aside[kAside];                                // bits of a value that 32768 more tokens have
};

// Bits of values to 16-bit keys of the same order; -0 is one below +0, and counted with it.
template <typename T> struct Key16 {
    static constexpr uint32_t kInf = std::is_same_v<T, _Float16> ? 0x7c00u : 0x7f80u, kTop = kInf | 0x8000u, kNone = 0x7fffu - kInf;     // keys of +inf and -inf
    static __device__ __forceinline__ uint32_t bits(uint32_t key) { return (key & 0x8000u) != 0 ? key & 0x7fffu : ~key & 0xffffu; }
    static __device__ __forceinline__ float value(uint32_t key) { return (float)__builtin_bit_cast(T, (uint16_t)bits(key)); }
};
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

template <typename T, int NV> __global__ __launch_bounds__(kThreads) void sample_keys_kernel(const SampleParams p) {
    using K = Key16<T>;
    constexpr uint32_t kNothing = 0x10000;                 // no value's bits
    static_assert(K::kInf % kUnit == 0 && NV % 4 == 0, "infinities begin a unit; pieces of four vectors a thread");
    __shared__ KeyShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t r = blockIdx.x;
    const Row<T> row(p, r);
    const uint4* at = reinterpret_cast<const uint4*>(row.x + row.head);
    uint4 held[NV];
    if (row.vecs > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) held[i] = at[min(tid + i * kThreads, row.vecs - 1)];
    }
    const int behind = row.head + row.vecs * 8, single = tid < row.head ? tid : behind + tid - row.head;
    uint32_t single_bits = 0;
    if (single < row.vocab) { T x = row.x[single]; single_bits = __builtin_bit_cast(uint16_t, x); }
    const Parameters of(p, r);
    // f(vector, its number) of all vectors, next() behind every four a thread.  (The compiler would otherwise take all vectors at once, and keep what it makes of each for
    // another round.)
    const auto vectors = [&](const auto& f, const auto& next) {
        int n = row.vecs - tid;
        asm volatile("" : "+v"(n));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            asm volatile("" : "+v"(held[i].x), "+v"(held[i].y), "+v"(held[i].z), "+v"(held[i].w));
            if (i * kThreads < n) f(held[i], tid + i * kThreads);
            if (i % 4 == 3) next();
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int v0 = NV * kThreads, i = 0; v0 < row.vecs; v0 += kThreads, ++i) {
            if (v0 < n) f(at[v0 + tid], v0 + tid);
            if (i % 4 == 3) next();
        }
    };

    // ---- how often each value occurs ----
    const auto put_aside = [&]() {
        __syncthreads();
        for (int i = tid; i < kMagnitudes; i += kThreads) {
            const uint32_t both = s.counts[i], over = both & 0x80008000u;
            if (over == 0) continue;
            s.counts[i] = both & 0x7fff7fffu;
            for (int h = 0; h < 2; ++h)
                if ((over >> (16 * h + 15) & 1) != 0) s.aside[min(atomicAdd(&s.n_aside, 1), kAside - 1)] = i | h << 15;
        }
        __syncthreads();
    };
    int pieces = 0;                                        // 1: counts are put aside between pieces
    for (;;) {
        for (int i = tid; i < kMagnitudes / 4; i += kThreads) reinterpret_cast<uint4*>(s.counts)[i] = make_uint4(0, 0, 0, 0);
        s.unit_count[tid] = 0;                             // (a lane's place for the frequent value)
        if (tid == 0) { s.n_aside = s.found = 0; s.heavy = 0; s.frequent = kNothing; s.n_frequent = 0; }
        __syncthreads();
        const auto add = [&](uint32_t at, uint32_t negative) {       // (1, or 2^16 for a negative value)
            uint32_t what;
            asm("v_mad_u32_u24 %0, %1, %2, 1" : "=v"(what) : "v"(negative), "s"(0xffff));
            atomicAdd(reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(s.counts) + at), what);
        };
        // One value may be most of a row's, as those of masked tokens are, and words that are added to at once take turns: the lanes have places of their own for it.  It is the
        // first one that a wavefront finds in many lanes.  (us of 64 x 128256, three quarters of which are the lowest value: 190 in one word, 21.)
        constexpr int kMany = 16, kStillMany = 8;
        const uint32_t own = offsetof(KeyShared, unit_count) + 4 * tid;
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int v = i / 2 * (NV - 1) / 2;            // the first, a middle and the last of a whole row's
            const uint32_t candidate = (uint32_t)__builtin_amdgcn_readfirstlane((int)(i % 2 == 0 ? held[v].x : held[v].y)) & 0xffffu;
            if ((v + 1) * kThreads <= row.vecs && __popcll(__ballot((held[v].z & 0xffffu) == candidate)) >= kMany && lane == 0) atomicCAS(&s.frequent, kNothing, candidate);
        }
        __syncthreads();
        const uint32_t frequent = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.frequent);
        const auto add_vector = [&](const uint4& u, auto some) {
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            const uint32_t those = frequent << 16;
            const auto place = [&](uint32_t high, uint32_t at) { return decltype(some)::value && (high ^ those) <= 0xffffu ? own : at; };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t low = (w[i] << 2) & 0x1fffcu, high = (w[i] >> 14) & 0x1fffcu;
                add(place(w[i] << 16, low), w[i] >> 15 & 1);
                add(place(w[i], high), w[i] >> 31);
            }
        };
        vectors([&](const uint4& u, int) {
            if (frequent != kNothing && __popcll(__ballot((u.x & 0xffffu) == frequent)) >= kStillMany) add_vector(u, std::true_type{});
            else add_vector(u, std::false_type{});
        }, [&]() { if (pieces != 0) put_aside(); });
        if (single < row.vocab) add(4 * (single_bits & 0x7fffu), single_bits >> 15);
        if (frequent != kNothing) {
            const int n = __builtin_amdgcn_readlane(prefix_sum((int)(s.unit_count[tid] >> (frequent >> 15 << 4))), 63);
            if (lane == 0) atomicAdd(&s.n_frequent, (uint32_t)n);
        }
        if (pieces != 0) put_aside();                      // (the last ones: fewer than a vector)
        __syncthreads();
        if (pieces != 0 || row.vocab <= 0xffff) break;
        uint32_t found = tid == 0 ? s.n_frequent : 0;
        for (int i = tid; i < kMagnitudes / 4; i += kThreads) {
            const uint4 c = reinterpret_cast<const uint4*>(s.counts)[i];
            found += (c.x & 0xffffu) + (c.x >> 16) + (c.y & 0xffffu) + (c.y >> 16) + (c.z & 0xffffu) + (c.z >> 16) + (c.w & 0xffffu) + (c.w >> 16);
        }
        found = group_reduce_bits<64>(found, [](uint32_t a, uint32_t b) { return a + b; });
        if (lane == 0) atomicAdd(&s.found, (int)found);
        __syncthreads();
        if (s.found == row.vocab) break;
        pieces = 1;
        __syncthreads();
    }
    const int n_aside = s.n_aside;
    const uint32_t frequent = s.frequent, n_frequent = s.n_frequent;
    const auto count_of = [&](uint32_t key) -> uint32_t {
        if (key > K::kTop || key <= K::kNone || key == 0x7fffu) return 0;
        const uint32_t bits = K::bits(key), both = s.counts[bits & 0x7fffu];
        uint32_t c = (bits >> 15 ? 0 : both & 0xffffu) + (bits >> 15 || bits == 0 ? both >> 16 : 0);
        c += bits == frequent || (bits == 0 && frequent == 0x8000u) ? n_frequent : 0;
        for (int i = 0; i < n_aside; ++i) c += s.aside[i] == bits || (bits == 0 && s.aside[i] == 0x8000u) ? 32768 : 0;
        return c;
    };

    // ---- the units of 64 keys that occur, largest first: unit u holds keys 65535 - 64 u and the 63 below; sums of their counts ----
    int in_unit = 0;                                       // one unit to a thread
    {
        const bool positive = tid < kUnits / 2;
        const int from = positive ? kMagnitudes - kUnit * (tid + 1) : kUnit * (tid - kUnits / 2);                  // their magnitudes
        const uint4* of_unit = reinterpret_cast<const uint4*>(s.counts + from);
        if (from < (int)K::kInf) {                         // (NaN and what stands in for masked tokens lie above)
            const u16x2_t which = {positive, !positive};
            for (int i = 0; i < kUnit / 4; ++i) {
                const uint4 c = of_unit[(i + lane) & (kUnit / 4 - 1)];
                const uint32_t each[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) in_unit = (int)__builtin_amdgcn_udot2(__builtin_bit_cast(u16x2_t, each[j]), which, (uint32_t)in_unit, false);
            }
        } else if (from == (int)K::kInf && positive) {
            in_unit = (int)(of_unit[0].x & 0xffffu);
        }
        if (from == 0) in_unit += positive ? (int)(s.counts[0] >> 16) : -(int)(s.counts[0] >> 16);                 // -0
        const auto add = [&](uint32_t bits, int n) {
            const uint32_t x = bits == 0x8000u ? 0 : bits;
            if ((x >> 15 == 0) == positive && (int)(x & 0x7fffu) >= from && (int)(x & 0x7fffu) < from + kUnit && (int)(x & 0x7fffu) <= (int)K::kInf - !positive) in_unit += n;
        };
        if (n_frequent > 0) add(frequent, (int)n_frequent);
        for (int i = 0; i < n_aside; ++i) add(s.aside[i], 32768);
    }
    const uint64_t occupied = __ballot(in_unit > 0);
    const int counts_upto = prefix_sum(in_unit);
    if (lane == 63) { s.occupied[wave] = (uint32_t)__popcll(occupied); s.partial[wave].count = (uint64_t)counts_upto; }
    __syncthreads();
    const int units_upto = prefix_sum(lane < kWaves ? (int)s.occupied[lane] : 0), counts_before = prefix_sum(lane < kWaves ? (int)s.partial[lane].count : 0);
    int n_units = __builtin_amdgcn_readlane(units_upto, kWaves - 1);
    const int n_tokens = __builtin_amdgcn_readlane(counts_before, kWaves - 1);
    if (in_unit > 0) {
        const int i = (wave > 0 ? __builtin_amdgcn_readlane(units_upto, wave - 1) : 0) + __popcll(occupied & ((1ull << lane) - 1));
        s.units[i] = (uint16_t)tid;
        s.unit_count[i] = counts_upto - in_unit + (wave > 0 ? __builtin_amdgcn_readlane(counts_before, wave - 1) : 0);
    }
    if (tid == 0) s.unit_count[n_units] = n_tokens;
    __syncthreads();
    if (n_units == 0) return write_nothing(p, r);

    // ---- the largest value, and the units' masses as far as they are asked for ----
    const auto key_in = [&](int i) { return (uint32_t)(2 * kMagnitudes - 1 - kUnit * (int)s.units[i] - lane); };
    const uint32_t first = key_in(0), top = (uint32_t)__builtin_amdgcn_readlane((int)first, __builtin_ctzll(__ballot(count_of(first) != 0)));
    const Weights w(K::value(top), of.inverse, weight_bits(row.vocab));
    const uint64_t one = 1ull << w.bits;
    const double least = ldexp(of.min_p, w.bits);
    const bool cut = of.k > 0 && of.k < n_tokens;
    if (cut || (of.any_min_p && of.top_p_none)) {          // the units in front of the k-th token and, where top-p does not ask for the whole, those with a token of enough weight
        const bool asked = tid < n_units && !(cut && (int)s.unit_count[tid] >= of.k) &&
                           !(of.any_min_p && of.top_p_none && tid > 0 && w.of(K::value(min((uint32_t)(2 * kMagnitudes - 1 - kUnit * (int)s.units[tid]), K::kTop))) < 0.5 * least);
        const uint64_t all = __ballot(asked);
        if (lane == 0) s.occupied[wave] = (uint32_t)__popcll(all);
        __syncthreads();
        n_units = __builtin_amdgcn_readlane(prefix_sum(lane < kWaves ? (int)s.occupied[lane] : 0), kWaves - 1);
    }
    uint64_t heavy = 0;
    for (int i = wave; i < n_units; i += kWaves) {
        const uint32_t key = key_in(i), c = count_of(key);
        const double v = w.of(K::value(key));
        const uint64_t mass = c != 0 ? times(c, w.whole(v)) : 0;
        if (of.any_min_p && c != 0 && v >= least) heavy += mass;
        const uint64_t masses = sum64(mass);
        if (lane == 0) s.unit_weight[i] = masses;
    }
    if (of.any_min_p) {
        heavy = sum64(heavy);
        if (lane == 0) atomicAdd((unsigned long long*)&s.heavy, (unsigned long long)heavy);
    }
    __syncthreads();
    uint64_t mine = tid < n_units ? s.unit_weight[tid] : 0, all;
    const uint64_t before = scan(s.partial, mine, all);
    if (tid < n_units) s.unit_weight[tid] = before;
    if (tid == 0) s.unit_weight[n_units] = all;
    __syncthreads();

    // ---- searches, by the first wavefront (others would only take its turns) ----
    if (wave == 0) {
        uint32_t found_key = 0;
        int found_nth = 0;                                 // of the tokens of that value: 1 ...
        const auto find = [&](bool by_count, uint64_t goal) {
            int unit = n_units - 1;                        // the first unit up to which the goal is reached
            for (int base = 0; base < n_units; base += 64) {
                const int i = min(base + lane + 1, n_units);
                const uint64_t reached = __ballot((by_count ? (uint64_t)s.unit_count[i] : s.unit_weight[i]) >= goal);
                if (reached != 0) { unit = min(base + (int)__builtin_ctzll(reached), n_units - 1); break; }
            }
            const uint32_t key = key_in(unit), c = count_of(key);
            const uint64_t each = c != 0 ? w.whole_of(K::value(key)) : 0;
            const Mass upto{s.unit_count[unit] + (uint64_t)(uint32_t)prefix_sum((int)c), s.unit_weight[unit] + prefix_sum64(times(c, each))};
            const uint64_t reached = __ballot(by_count ? upto.count >= goal : upto.weight >= goal);
            const int l = reached != 0 ? __builtin_ctzll(reached) : 63;
            const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)c, l);
            const uint64_t weight = of_lane(each, l);
            const Mass start{of_lane(upto.count, l) - n, of_lane(upto.weight, l) - n * weight};
            uint64_t nth = by_count ? goal - start.count : weight > 0 ? ceil_quotient(goal - start.weight, weight) : 1;
            nth = nth < 1 ? 1 : nth > n ? n : nth;
            found_key = (uint32_t)__builtin_amdgcn_readlane((int)key, l);
            found_nth = (int)nth;
            return start.weight + nth * weight;
        };
        const uint64_t kept = draw(of, all, cut ? of.k : 0, one, s.heavy, [&](int step, uint64_t goal) { return find(step == 0, goal); });
        if (lane == 0) {
            s.found = (int)found_key;
            s.nth = found_nth;
            write_logprob(p, r, w, K::value(found_key), kept);
        }
    }
    __syncthreads();                                       // (nobody counts any more)
    const uint32_t found_key = (uint32_t)s.found;
    const int found_nth = s.nth;

    // ---- which of the tokens of that value ----
    // Pieces of the row in its order: the elements in front of the vectors, up to 1022 pieces of 2^shift vectors, the elements behind them.
    const int shift = max(4, 32 - (int)__builtin_clz((unsigned)row.vecs | 1) - 9), last_piece = kThreads - 1;
    uint32_t* of_piece = s.counts;                         // [1024], and behind these a bit to each token of one piece
    uint32_t* bitmap = s.counts + kThreads;
    of_piece[tid] = 0;
    __syncthreads();
    const uint32_t raw = K::bits(found_key), mask = raw == 0 ? 0x7fffu : 0xffffu;     // (of zero, both signs)
    const uint32_t raw2 = raw * 0x10001u, mask2 = mask * 0x10001u;
    vectors([&](const uint4& u, int v) {
        const u16x2_t x[4] = {__builtin_bit_cast(u16x2_t, (u.x ^ raw2) & mask2), __builtin_bit_cast(u16x2_t, (u.y ^ raw2) & mask2),
                              __builtin_bit_cast(u16x2_t, (u.z ^ raw2) & mask2), __builtin_bit_cast(u16x2_t, (u.w ^ raw2) & mask2)};
        const u16x2_t nearest = __builtin_elementwise_min(__builtin_elementwise_min(x[0], x[1]), __builtin_elementwise_min(x[2], x[3]));
        if (nearest[0] != 0 && nearest[1] != 0) return;
        const u16x2_t ones = {1, 1};
        u16x2_t others = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) others += __builtin_elementwise_min(x[i], ones);
        atomicAdd(&of_piece[1 + (v >> shift)], 8u - others[0] - others[1]);
    }, []() {});
    if (single < row.vocab && ((single_bits ^ raw) & mask) == 0) atomicAdd(&of_piece[single < row.head ? 0 : last_piece], 1u);
    __syncthreads();
    const int here = (int)of_piece[tid], in_front = (int)scan(s.partial, (uint64_t)here, all);
    if (in_front < found_nth && in_front + here >= found_nth) { s.index = tid; s.nth = found_nth - in_front; }
    __syncthreads();
    const int piece = s.index, from = piece == 0 ? 0 : piece == last_piece ? behind : row.head + ((piece - 1) << (shift + 3));
    const int upto = piece == 0 ? row.head : piece == last_piece ? row.vocab : min(behind, from + (8 << shift));
    for (int i = tid; i < 8 << shift; i += kThreads) {     // whole wavefronts
        uint32_t x = 1;
        if (from + i < upto) { const T v = row.x[from + i]; x = (__builtin_bit_cast(uint16_t, v) ^ raw) & mask; }
        const uint64_t equal = __ballot(x == 0);
        if (lane == 0) { bitmap[i >> 5] = (uint32_t)equal; bitmap[(i >> 5) + 1] = (uint32_t)(equal >> 32); }
    }
    __syncthreads();
    if (tid == 0) {
        int left = s.nth, i = 0;
        for (; i < (1 << (shift - 2)) - 1 && left > __popc(bitmap[i]); ++i) left -= __popc(bitmap[i]);
        uint32_t b = bitmap[i];
        for (; left > 1; --left) b &= b - 1;
        p.ids[r] = from + 32 * i + __builtin_ctz(b | 0x80000000u);
    }
}

constexpr int64_t kMostRows = (1ll << 32) / kThreads - 1;  // a launch has fewer than 2^32 threads

template <typename T> void launch(const SampleParams& p, int64_t rows, hipStream_t st) {
    const dim3 grid((unsigned)rows), block(kThreads);
    if constexpr (sizeof(T) == 4) sample_kernel<T><<<grid, block, 0, st>>>(p);
    else if (p.vocab <= 4 * 8 * kThreads) sample_keys_kernel<T, 4><<<grid, block, 0, st>>>(p);
    else sample_keys_kernel<T, 16><<<grid, block, 0, st>>>(p);
}

}  // namespace

extern "C" int mi_sample(const mi_sample_args* a) {
    if (!a) return mi_fail(MI_E_NULL, "sample: args is null");
    if (a->n_rows == 0) return MI_OK;
    if (a->n_rows < 0 || a->n_rows > kMostRows || a->vocab < 1 || a->vocab > MI_SAMPLE_VOCAB_MAX || a->row_stride < 0)
        return mi_fail(MI_E_SHAPE, "sample: %lld rows of %lld logits (1 to %d), %lld apart", (long long)a->n_rows, (long long)a->vocab, MI_SAMPLE_VOCAB_MAX,
                       (long long)a->row_stride);
    if (!a->logits || !a->uniforms || !a->ids) return mi_fail(MI_E_NULL, "sample: null pointer");
    const SampleParams p{a->logits, a->row_stride, (int)a->vocab, a->uniforms, a->temperatures, a->top_ps, a->min_ps, a->top_ks, a->temperature, a->top_p, a->min_p,
                         a->top_k, a->ids, a->logprobs};
    MI_DISPATCH_DTYPE(a->dtype, launch<T>(p, a->n_rows, (hipStream_t)a->stream));
    return mi_check_launch("sample");
}

// The next step of a paged cache from lengths that lie on the device: which pages it takes, and position, slot and sequence of every new token.
//
// With len keys of a sequence before the step and n new ones, pages of P keys and exclusive sums over the sequences
//     held = ceil(len / P),   wanted = ceil((len + n) / P) - held,   W = sum of wanted in front,   C = sum of n in front,
// page held + i of its table is the (W + i)-th from the top of the stack of free pages, and its token j is row C + j of the step at position len + j.  A sequence
// that ends (n < 0) has its pages put on the stack first, last page first, sequence after sequence, as PagedKVCache does on the host.
// Latency is all there is to it: one workgroup sums with a sequence to a thread and goes over pages and tokens with a thread to each, finding their
// sequences in the sums in LDS; only the tokens of long steps are a launch of their own.
#include "common.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kTokensInOne = 4096;                         // tokens of a step up to which there is one launch

struct StepParams {
    const int32_t *new_tokens, *lengths, *state, *offsets;
    int32_t *ctx_len, *state_out, *table, *free_pages, *cu;
    int64_t *positions, *slots, *sequences, *last;
    int64_t table_stride;
    int batch, max_pages, page, n_free, tokens, max_ctx;
    uint32_t page_m;                                       // for divide()
};

enum { kNoPages = 1, kTooLong = 2, kTooMany = 4 };

struct Sequence {
    int n, len, held, wanted, given;
    bool too_long;
};
__device__ __forceinline__ Sequence sequence(const StepParams& p, int b, bool take) {
    Sequence s{0, 0, 0, 0, 0, false};
    if (b >= p.batch) return s;
    const int n = p.new_tokens[b], len = min(max(p.lengths[b], 0), p.max_pages * p.page), pages = divide((uint32_t)(len + p.page - 1), p.page, p.page_m);
    if (n < 0) {
        s.given = pages;
        return s;
    }
    s.len = len;
    s.held = pages;
    if (!take) return s;
    s.too_long = n > 0 && n > p.max_ctx - len;
    s.n = min(n, p.tokens + 1);                            // (more than there may be)
    s.wanted = s.too_long ? 0 : divide((uint32_t)(len + n + p.page - 1), p.page, p.page_m) - pages;
    return s;
}

// Sums of a chunk of 1024 sequences in front of each, [kThreads]: of all.
struct Sums { int given[kThreads + 1], wanted[kThreads + 1], tokens[kThreads + 1]; };

// the entry e of sums that holds place x: sums[e] <= x < sums[e + 1]
__device__ __forceinline__ int holder(const int* sums, int x) {
    int lo = 0, hi = kThreads;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void write_row(const StepParams& p, int row, int64_t position, int64_t slot, int64_t sequence) {
    p.positions[row] = position;
    p.slots[row] = slot;
    p.sequences[row] = sequence;
}
__device__ __forceinline__ void write_token(const StepParams& p, int row, int b, int position) {
    const int index = divide((uint32_t)position, p.page, p.page_m);
    write_row(p, row, position + (p.offsets ? (int64_t)p.offsets[b] : 0), (int64_t)p.table[b * p.table_stride + index] * p.page + (position - index * p.page), b);
}

__global__ __launch_bounds__(kThreads) void paged_step_kernel(const StepParams p, bool write_tokens) {
    __shared__ Sums sums;
    __shared__ int of_wave[4][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int free_before = min(max(p.state[0], 0), p.n_free), was = p.state[1];

    // sums of a chunk of sequences; what all of them have together (of more tokens than there may be: some number over it)
    struct Totals { int given, wanted, tokens; bool too_long, several; };
    const auto add_up = [&](const Sequence& s) {
        const int given = prefix_sum(s.given), wanted = prefix_sum(s.wanted), tokens = prefix_sum(s.n);
        const int flags = (__any(s.too_long) ? 1 : 0) | (__any(s.n > 1) ? 2 : 0);
        __syncthreads();
        if (lane == 63) { of_wave[0][wave] = given; of_wave[1][wave] = wanted; of_wave[2][wave] = min(tokens, p.tokens + 1); of_wave[3][wave] = flags; }
        __syncthreads();
        const bool there = lane < kWaves;
        int before[3], total[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int upto = prefix_sum(there ? of_wave[k][lane & (kWaves - 1)] : 0);
            before[k] = wave > 0 ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
            total[k] = __builtin_amdgcn_readlane(upto, kWaves - 1);
        }
        const int of_all = there ? of_wave[3][lane & (kWaves - 1)] : 0;
        sums.given[tid] = before[0] + given - s.given;
        sums.wanted[tid] = before[1] + wanted - s.wanted;
        sums.tokens[tid] = before[2] + tokens - s.n;
        if (tid == 0) { sums.given[kThreads] = total[0]; sums.wanted[kThreads] = total[1]; sums.tokens[kThreads] = total[2]; }
        __syncthreads();
        return Totals{total[0], total[1], total[2], __any(of_all & 1) != 0, __any(of_all & 2) != 0};
    };

    // pages of a chunk's sequences that end onto the stack from `at` on, last page first; four at a time, so that four are under way
    const auto push = [&](int base, int64_t at) {
        constexpr int kAhead = 4;
        const int n = sums.given[kThreads];
        for (int i0 = tid; i0 < n; i0 += kAhead * kThreads) {
            int page[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = min(i0 + k * kThreads, n - 1), e = holder(sums.given, i);
                page[k] = p.table[(int64_t)(base + e) * p.table_stride + sums.given[e + 1] - 1 - i];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kThreads;
                if (i < n && at + i < p.n_free) p.free_pages[at + i] = page[k];
            }
        }
    };

    // ---- a token of each sequence at most: the sequences' threads have all that is needed ----
    const bool one_chunk = p.batch <= kThreads;
    Sequence s = sequence(p, tid, true);
    Totals all;
    if (one_chunk) {
        const int at = divide((uint32_t)s.len, p.page, p.page_m);
        const bool there = tid < p.batch;
        int page = there && s.len < p.max_pages * p.page ? p.table[(int64_t)tid * p.table_stride + at] : 0;       // (asked for before it is known whether it is a new one)
        const int offset = there && p.offsets ? p.offsets[tid] : 0;
        all = add_up(s);
        if (!all.several) {
            const int64_t wanted = all.wanted, tokens = all.tokens, stacked = min(free_before + (int64_t)all.given, (int64_t)p.n_free);
            const int status = (wanted > stacked ? kNoPages : 0) | (all.too_long ? kTooLong : 0) | (tokens > p.tokens ? kTooMany : 0);
            const bool take = status == 0;
            const int row = sums.tokens[tid];
            if (there) {
                if (take && s.wanted > 0) {                // (of those that were just given back, from where they come: nobody waits for them to be on the stack)
                    const int64_t from = stacked - 1 - sums.wanted[tid];
                    if (from >= free_before) {
                        const int i = (int)(from - free_before), e = holder(sums.given, i);
                        page = p.table[(int64_t)e * p.table_stride + sums.given[e + 1] - 1 - i];
                    } else {
                        page = p.free_pages[from];
                    }
                    p.table[(int64_t)tid * p.table_stride + at] = page;
                }
                const bool writes = take && s.n > 0;
                p.ctx_len[tid] = s.len + (writes ? 1 : 0);
                p.cu[tid] = take ? row : 0;
                p.last[tid] = writes ? row : 0;
                if (writes && write_tokens) write_row(p, row, s.len + (int64_t)offset, (int64_t)page * p.page + (s.len - at * p.page), tid);
            }
            const int rows = take ? (int)tokens : 0;
            if (write_tokens)
                for (int i = rows + tid; i < p.tokens; i += kThreads) write_row(p, i, 0, -1, 0);
            push(0, free_before);
            if (tid == 0) {
                p.cu[p.batch] = rows;
                p.state_out[0] = (int)(stacked - (take ? wanted : 0));
                p.state_out[1] = was | status;
            }
            return;
        }
    }

    // ---- whether there is room ----
    int64_t given = 0, wanted = 0, tokens = 0;
    bool too_long = false;
    for (int base = 0; base < p.batch; base += kThreads) {
        if (!one_chunk) {
            s = sequence(p, base + tid, true);
            all = add_up(s);
        }
        given += all.given; wanted += all.wanted; tokens += all.tokens;
        too_long |= all.too_long;
    }
    const int64_t stacked = min(free_before + given, (int64_t)p.n_free);        // (more than all pages: the caller's mistake)
    const int status = (wanted > stacked ? kNoPages : 0) | (too_long ? kTooLong : 0) | (tokens > p.tokens ? kTooMany : 0);
    const bool take = status == 0;

    // ---- pages onto the stack ----
    if (given > 0) {
        int64_t done = free_before;
        for (int base = 0; base < p.batch; base += kThreads) {
            if (!one_chunk) add_up(sequence(p, base + tid, true));
            push(base, done);
            done += sums.given[kThreads];
        }
    }
    __syncthreads();

    // ---- pages from it, lengths and the tokens ----
    int64_t taken = 0;
    int rows = 0;
    for (int base = 0; base < p.batch; base += kThreads) {
        const int b = base + tid;
        if (!one_chunk || !take) {
            s = sequence(p, b, take);
            add_up(s);
        }
        for (int i = tid; i < sums.wanted[kThreads]; i += kThreads) {
            const int e = holder(sums.wanted, i);
            const int len = min(max(p.lengths[base + e], 0), p.max_pages * p.page);
            p.table[(int64_t)(base + e) * p.table_stride + divide((uint32_t)(len + p.page - 1), p.page, p.page_m) + i - sums.wanted[e]] =
                p.free_pages[stacked - 1 - taken - i];
        }
        __syncthreads();                                   // the table is read below
        if (write_tokens)
            for (int i = tid; i < sums.tokens[kThreads]; i += kThreads) {
                const int e = holder(sums.tokens, i);
                write_token(p, rows + i, base + e, min(max(p.lengths[base + e], 0), p.max_pages * p.page) + i - sums.tokens[e]);
            }
        __syncthreads();                                   // ctx_len may be the lengths
        if (b < p.batch) {
            p.ctx_len[b] = s.len + s.n;
            p.cu[b] = rows + sums.tokens[tid];
            p.last[b] = s.n > 0 ? rows + sums.tokens[tid] + s.n - 1 : 0;
        }
        taken += sums.wanted[kThreads];
        rows += sums.tokens[kThreads];
    }
    if (write_tokens)
        for (int i = rows + tid; i < p.tokens; i += kThreads) write_row(p, i, 0, -1, 0);
    if (tid == 0) {
        p.cu[p.batch] = rows;
        p.state_out[0] = (int)(stacked - taken);
        p.state_out[1] = was | status;
    }
}

// The tokens of a step whose sequences are planned.  (With the sequences' rows in LDS, for which a workgroup waits first, 4.7 us of 65000 tokens; so 3.6.)
constexpr int kTokenThreads = 256;
__global__ __launch_bounds__(kTokenThreads) void paged_step_tokens_kernel(const StepParams p) {
    const int row = blockIdx.x * kTokenThreads + threadIdx.x;
    if (row >= p.tokens) return;
    if (row >= p.cu[p.batch]) return write_row(p, row, 0, -1, 0);
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid] <= row) lo = mid; else hi = mid;
    }
    write_token(p, row, lo, p.ctx_len[lo] - p.cu[lo + 1] + row);
}

}  // namespace

extern "C" int mi_paged_step(const mi_paged_step_args* a) {
    if (!a) return mi_fail(MI_E_NULL, "paged_step: args is null");
    if (a->batch < 1 || a->batch > (1 << 24) || a->max_pages < 1 || a->max_pages > (1 << 24) || a->page_size < 1 || (int64_t)a->max_pages * a->page_size > (1 << 30) ||
        (int64_t)a->batch * a->max_pages > 0x7fffffffLL || a->n_free < 0 || a->tokens < 0 || a->tokens > (1 << 24) || a->max_ctx < 0 || a->max_ctx > a->max_pages * a->page_size || a->page_table_stride < 0)
        return mi_fail(MI_E_SHAPE, "paged_step: %d sequences of up to %d pages of %d keys, %d keys at most, %d tokens, a stack of %d pages", a->batch, a->max_pages,
                       a->page_size, a->max_ctx, a->tokens, a->n_free);
    if (!a->new_tokens || !a->lengths || !a->state || !a->ctx_len || !a->state_out || !a->page_table || !a->cu_seqlens || !a->last ||
        (a->n_free > 0 && !a->free_pages) || (a->tokens > 0 && (!a->position_ids || !a->slots || !a->sequences)))
        return mi_fail(MI_E_NULL, "paged_step: null pointer");
    const StepParams p{a->new_tokens, a->lengths, a->state, a->position_offset, a->ctx_len, a->state_out, a->page_table, a->free_pages, a->cu_seqlens, a->position_ids,
                       a->slots, a->sequences, a->last, a->page_table_stride, a->batch, a->max_pages, a->page_size, a->n_free, a->tokens,
                       a->max_ctx > 0 ? a->max_ctx : a->max_pages * a->page_size, divide_m(a->page_size)};
    const bool one = a->tokens <= kTokensInOne;
    paged_step_kernel<<<dim3(1), dim3(kThreads), 0, (hipStream_t)a->stream>>>(p, one);
    if (const int rc = mi_check_launch("paged_step"); rc != MI_OK || one) return rc;
    paged_step_tokens_kernel<<<dim3((unsigned)((a->tokens + kTokenThreads - 1) / kTokenThreads)), dim3(kTokenThreads), 0, (hipStream_t)a->stream>>>(p);
    return mi_check_launch("paged_step_tokens");
}

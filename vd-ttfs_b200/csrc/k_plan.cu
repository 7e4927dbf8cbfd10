// k_plan.cu -- first rows, positions, cache slots and pages of a step's tokens
// from its sequences' lengths, and the pages of finished sequences put back.
//
//   start_s = sum of the new tokens before sequence s,  kept_s = held_s + new_s
//   row start_s + i holds position held_s + i, in page (held_s + i) / P of its sequence
//   pages ceil(held_s / P) .. ceil(kept_s / P) come from the ring of free ones,
//   sequence after sequence
//
// Nothing here is more than a prefix sum over the sequences and 12 bytes a
// token: bound by the latency of the scan and of a launch.  Each token finds
// its page by itself, in the table if the sequence had it before and in the
// ring if not, so tokens need no order among them, nor among the pages that are
// written into the table meanwhile.
#include <algorithm>

#include "step_internal.h"

namespace vdt {
namespace {

constexpr int kPlanThreads = 256, kEach = 4, kFused = kPlanThreads * kEach;   // sequences of the one-launch form
constexpr int kTokens = 2;                                                    // tokens a thread

// lengths as the planner counts them: nothing below zero, nothing past 32 bits
__device__ __forceinline__ int length(int n) { return max(n, 0); }
__device__ __forceinline__ int together(int held, int fresh) { return (int)min((long long)length(held) + length(fresh), 0x7fffffffLL); }
__device__ __forceinline__ int pages_for(int tokens, int page) { return (int)(((long long)tokens + page - 1) / page); }
// pages of the table that a sequence's new tokens begin
__device__ __forceinline__ int wanted(int held, int kept, int page, int width) {
    return max(0, min(pages_for(kept, page), width) - pages_for(held, page));
}
// the ring's state, whatever it holds: a place inside, no more pages than it has room for
__device__ __forceinline__ void ring_state(const int32_t* span, int size, int& first, int& left) {
    const int a = span[0];
    left = a < 0 || a >= size ? 0 : min(max(span[1], 0), size);
    first = a < 0 || a >= size ? 0 : a;
}

// Sums before each thread's own, of tokens and of pages; both totals in `all`.
// 64 bits: the sums of broken lengths do not wrap.
template <int THREADS>
__device__ __forceinline__ void scan2(long long& tokens, long long& pages, long long (&all)[2]) {
    __shared__ long long part[2][THREADS / 32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    long long t = tokens, p = pages;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long a = __shfl_up_sync(0xffffffffu, t, d), b = __shfl_up_sync(0xffffffffu, p, d);
        if (lane >= d) {
            t += a;
            p += b;
        }
    }
    __syncthreads();
    if (lane == 31) {
        part[0][warp] = t;
        part[1][warp] = p;
    }
    __syncthreads();
    long long bt = 0, bp = 0;
    all[0] = all[1] = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        if (i == warp) {
            bt = all[0];
            bp = all[1];
        }
        all[0] += part[0][i];
        all[1] += part[1][i];
    }
    tokens = bt + t - tokens;
    pages = bp + p - pages;
}
__device__ __forceinline__ int clamp32(long long v) { return (int)min(v, 0x7fffffffLL); }

// What a token needs of its sequence
struct Seq {
    int start, held, base;      // first row; tokens before; pages given to the sequences before
};

__device__ __forceinline__ void plan_token(const PlanParams& p, long long row, int seq, const Seq& q, int first, int left) {
    const long long at = (long long)q.held + (row - q.start);
    const long long j = at / p.page;
    const int had = pages_for(q.held, p.page);
    int number = -1;
    if (j < p.width) {
        const long long i = (long long)q.base + (j - had);
        if (j < had) number = p.pages[(long long)seq * p.width + j];
        else if (i < left) number = p.ring[(first + i) % p.size];
    }
    p.positions[row] = (int)min(at, 0x7fffffffLL);
    p.slots[row] = number >= 0 ? (long long)number * p.page + at % p.page : -1;
}
__device__ __forceinline__ void plan_none(const PlanParams& p, long long row) {
    p.positions[row] = -1;
    p.slots[row] = -1;
}
__device__ __forceinline__ void plan_span(const PlanParams& p, int first, int left, long long took) {
    p.span_out[0] = p.size ? (int)((first + min(took, (long long)left)) % p.size) : 0;
    p.span_out[1] = (int)max(left - took, -0x7fffffffLL);
}

// The last sequence that starts at or before a row, or whose pages begin at or
// before a number: the one that has the row, or the page
template <int Seq::*From>
__device__ __forceinline__ int owner(const Seq* seqs, int n, long long of) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (seqs[mid].*From <= of) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ void plan_rows(const PlanParams& p, const Seq* seqs, int first, int left, int tokens, int pages) {
    const long long from = (long long)blockIdx.x * kPlanThreads + threadIdx.x, step = (long long)gridDim.x * kPlanThreads;
    for (long long i = from; i < pages; i += step) {
        const int s = owner<&Seq::base>(seqs, p.seqs, i);
        p.pages[(long long)s * p.width + pages_for(seqs[s].held, p.page) + (i - seqs[s].base)] = i < left ? p.ring[(first + i) % p.size] : -1;
    }
    for (long long row = from; row < p.total; row += step) {
        if (row >= tokens) {
            plan_none(p, row);
            continue;
        }
        const int s = owner<&Seq::start>(seqs, p.seqs, row);
        plan_token(p, row, s, seqs[s], first, left);
    }
}

// One launch for up to kFused sequences: every CTA sums all their lengths for
// itself and plans its own rows; the first writes what belongs to the
// sequences.  Outputs must not lie over inputs that the other CTAs still read.
__global__ void __launch_bounds__(kPlanThreads) k_plan(PlanParams p) {
    __shared__ Seq seqs[kFused + 1];
    const int thread = threadIdx.x;
    int first, left;
    ring_state(p.span, p.size, first, left);
    int held[kEach], kept[kEach], fresh[kEach];
    long long tokens = 0, pages = 0, all[2];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = thread * kEach + i;
        const bool in = s < p.seqs;
        held[i] = in ? length(p.held[s]) : 0;
        fresh[i] = in ? length(p.fresh[s]) : 0;
        kept[i] = together(held[i], fresh[i]);
        tokens += fresh[i];
        pages += wanted(held[i], kept[i], p.page, p.width);
    }
    scan2<kPlanThreads>(tokens, pages, all);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = thread * kEach + i;
        seqs[s] = {clamp32(tokens), held[i], clamp32(pages)};
        if (blockIdx.x == 0 && s < p.seqs) {
            p.kept[s] = kept[i];
            p.starts[s] = clamp32(tokens);
        }
        tokens += fresh[i];
        pages += wanted(held[i], kept[i], p.page, p.width);
    }
    if (blockIdx.x == 0 && thread == 0) {
        p.starts[p.seqs] = clamp32(all[0]);
        plan_span(p, first, left, all[1]);
    }
    __syncthreads();
    plan_rows(p, seqs, first, left, clamp32(all[0]), clamp32(all[1]));
}

// The general form, two launches: one CTA sums the lengths into the scratch
// (start, held and base of each sequence; first, left, both sums), then the rows are
// planned from it.
constexpr int kScanThreads = 1024;
__global__ void __launch_bounds__(kScanThreads) k_plan_scan(PlanParams p) {
    chain_release();
    int first, left;
    ring_state(p.span, p.size, first, left);
    __syncthreads();                         // span may be span_out
    Seq* const out = reinterpret_cast<Seq*>(p.scratch + 4);
    long long tokens0 = 0, pages0 = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += kScanThreads) {
        const int s = s0 + threadIdx.x;
        const bool in = s < p.seqs;
        const int held = in ? length(p.held[s]) : 0, fresh = in ? length(p.fresh[s]) : 0, kept = together(held, fresh);
        long long tokens = fresh, pages = wanted(held, kept, p.page, p.width), all[2];
        scan2<kScanThreads>(tokens, pages, all);
        if (in) {
            out[s] = {clamp32(tokens0 + tokens), held, clamp32(pages0 + pages)};
            p.kept[s] = kept;
            p.starts[s] = clamp32(tokens0 + tokens);
        }
        tokens0 += all[0];
        pages0 += all[1];
    }
    if (threadIdx.x == 0) {
        p.scratch[0] = first;
        p.scratch[1] = left;
        p.scratch[2] = clamp32(tokens0);
        p.scratch[3] = clamp32(pages0);
        p.starts[p.seqs] = clamp32(tokens0);
        plan_span(p, first, left, pages0);
    }
}
__global__ void __launch_bounds__(kPlanThreads) k_plan_rows(PlanParams p) {
    chain_wait();
    plan_rows(p, reinterpret_cast<const Seq*>(p.scratch + 4), p.scratch[0], p.scratch[1], p.scratch[2], p.scratch[3]);
}

// One CTA: a warp counts a finished sequence's pages, the counts are summed,
// and the warp that counted them writes them behind the ring's last.
__global__ void __launch_bounds__(kScanThreads) k_free(FreeParams p) {
    __shared__ int counts[kScanThreads];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int first, left;
    ring_state(p.span, p.size, first, left);
    __syncthreads();                         // span may be span_out
    long long before = left;
    for (int s0 = 0; s0 < p.seqs; s0 += kScanThreads) {
        const int here = min(kScanThreads, p.seqs - s0);
        for (int i = warp; i < kScanThreads; i += kScanThreads / 32) {
            int n = 0;
            const int s = s0 + i;
            if (i < here && p.done[s]) {
                const int most = min(pages_for(length(p.held[s]), p.page), p.width);
                for (int j = lane; j < most; j += 32) n += p.pages[(long long)s * p.width + j] >= 0;
                n = __reduce_add_sync(0xffffffffu, n);
            }
            if (lane == 0) counts[i] = n;
        }
        __syncthreads();
        long long at = counts[threadIdx.x], none = 0, all[2];
        scan2<kScanThreads>(at, none, all);
        __syncthreads();
        counts[threadIdx.x] = clamp32(before + at);
        __syncthreads();
        for (int i = warp; i < here; i += kScanThreads / 32) {
            const int s = s0 + i;
            if (!p.done[s]) continue;
            const int most = min(pages_for(length(p.held[s]), p.page), p.width);
            long long to = counts[i];
            for (int j0 = 0; j0 < most; j0 += 32) {
                const int number = j0 + lane < most ? p.pages[(long long)s * p.width + j0 + lane] : -1;
                const unsigned have = __ballot_sync(0xffffffffu, number >= 0);
                const long long mine = to + __popc(have & ((1u << lane) - 1));
                if (number >= 0 && mine < p.size) p.ring[(first + mine) % p.size] = number;
                to += __popc(have);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += kScanThreads) p.held_out[s0 + i] = p.done[s0 + i] ? 0 : p.held[s0 + i];
        before += all[0];
    }
    if (threadIdx.x == 0) {
        p.span_out[0] = first;
        p.span_out[1] = (int)min(before, (long long)p.size);
    }
}

bool over(const int32_t* a, long long n, const int32_t* b, long long m) { return a < b + m && b < a + n; }

}  // namespace

size_t plan_scratch_bytes(int seqs) { return 16 + (size_t)seqs * sizeof(Seq); }

// One launch up to kFused sequences, unless the step is planned in place
// (kept over held, the ring's state over itself), which needs every length to
// be read before the first is written.
cudaError_t launch_plan_pages(const PlanParams& p, cudaStream_t s) {
    const long long blocks = (p.total + kPlanThreads * kTokens - 1) / (kPlanThreads * kTokens);
    const dim3 grid((unsigned)std::max(1LL, std::min(blocks, 8LL * kSmCount)));
    bool aliased = over(p.span, 2, p.span_out, 2) || over(p.span, 2, p.kept, p.seqs) || over(p.span, 2, p.starts, p.seqs + 1);
    for (const int32_t* in : {p.held, p.fresh})
        aliased = aliased || over(in, p.seqs, p.kept, p.seqs) || over(in, p.seqs, p.starts, p.seqs + 1) || over(in, p.seqs, p.span_out, 2);
    if (p.seqs <= kFused && (!aliased || grid.x == 1)) {
        k_plan<<<grid, kPlanThreads, 0, s>>>(p);
        return cudaGetLastError();
    }
    k_plan_scan<<<1, kScanThreads, 0, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_after(k_plan_rows, grid, dim3(kPlanThreads), 0, s, p);
}

cudaError_t launch_free_pages(const FreeParams& p, cudaStream_t s) {
    k_free<<<1, kScanThreads, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace vdt

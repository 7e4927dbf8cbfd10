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
//
// us a replayed launch: 48 sequences of one new token 6.0, 200 sequences of up to
// 4093 new tokens (6 MB written) 6.7; with the pages of the finished ones put
// back, a second launch, 8.6 and 10.3.  All CTAs of the one-launch form scan the
// lengths again, which takes less than a launch in between would.
#include <algorithm>

#include "step_internal.h"

namespace vdt {
namespace {

constexpr int kPlanThreads = 256, kEach = 4, kFused = kPlanThreads * kEach;   // sequences of the one-launch form
constexpr int kRows = 4;                                                      // consecutive rows a thread

// A page's tokens, and the shift that divides by them (or -1).  Divisions are of
// numbers below 2^32: a length and the rows of a call together are.
struct Page {
    uint32_t tokens;
    int shift;
    __device__ __forceinline__ uint32_t of(uint32_t at) const { return shift >= 0 ? at >> shift : at / tokens; }
    __device__ __forceinline__ int many(int n) const { return (int)of((uint32_t)n + tokens - 1); }     // pages of n tokens
};
// lengths as the planner counts them: nothing below zero, nothing past 32 bits
__device__ __forceinline__ int length(int n) { return max(n, 0); }
__device__ __forceinline__ int together(int held, int fresh) { return (int)min((long long)length(held) + length(fresh), 0x7fffffffLL); }
// pages of the table that a sequence's new tokens begin
__device__ __forceinline__ int wanted(int held, int kept, const Page& page, int width) { return max(0, min(page.many(kept), width) - page.many(held)); }
// the ring's state, whatever it holds: a place inside, no more pages than it has room for
__device__ __forceinline__ void ring_state(const int32_t* span, int size, int& first, int& left) {
    const int a = span[0], n = span[1];
    left = a < 0 || a >= size ? 0 : min(max(n, 0), size);
    first = a < 0 || a >= size ? 0 : a;
}
// the ring's entry number i from its first, i below its size
__device__ __forceinline__ uint32_t ring_place(int first, int i, int size) {
    const uint32_t at = (uint32_t)first + (uint32_t)i;
    return at >= (uint32_t)size ? at - (uint32_t)size : at;
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

// What a token needs of its sequence: its first row, the tokens and pages it had,
// the pages given to the sequences before
struct __align__(16) Seq {
    int start, held, had, base;
};

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
// seqs[p.seqs].start: the first row behind them all
__device__ __forceinline__ void plan_rows(const PlanParams& p, const Seq* seqs, int first, int left, int tokens, int pages) {
    const Page page{(uint32_t)p.page, p.shift};
    const long long from = (long long)blockIdx.x * kPlanThreads + threadIdx.x, step = (long long)gridDim.x * kPlanThreads;
    for (long long i = from; i < pages; i += step) {
        const int s = owner<&Seq::base>(seqs, p.seqs, i);
        p.pages[(long long)s * p.width + seqs[s].had + ((int)i - seqs[s].base)] = i < left ? p.ring[ring_place(first, (int)i, p.size)] : -1;
    }
    for (long long row0 = from * kRows; row0 < p.total; row0 += step * kRows) {
        int at[kRows], s = 0, next = 0;
        long long slot[kRows];
        Seq q{};
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const long long row = row0 + k;
            at[k] = -1;
            slot[k] = -1;
            if (row >= tokens || row >= p.total) continue;
            if (k == 0 || row >= next) {
                s = owner<&Seq::start>(seqs, p.seqs, row);
                q = seqs[s];
                next = seqs[s + 1].start;
            }
            const uint32_t place = (uint32_t)q.held + (uint32_t)((int)row - q.start), j = page.of(place);
            int number = -1;
            if (j < (uint32_t)p.width) {
                const long long i = (long long)q.base + (int)j - q.had;
                if ((int)j < q.had) number = p.pages[(long long)s * p.width + j];
                else if (i < left) number = p.ring[ring_place(first, (int)i, p.size)];
            }
            at[k] = (int)min(place, 0x7fffffffu);
            if (number >= 0) slot[k] = (long long)number * p.page + (place - j * page.tokens);
        }
        if (p.wide && row0 + kRows <= p.total) {
            *reinterpret_cast<int4*>(p.positions + row0) = make_int4(at[0], at[1], at[2], at[3]);
            *reinterpret_cast<longlong2*>(p.slots + row0) = make_longlong2(slot[0], slot[1]);
            *reinterpret_cast<longlong2*>(p.slots + row0 + 2) = make_longlong2(slot[2], slot[3]);
        } else {
#pragma unroll
            for (int k = 0; k < kRows; ++k)
                if (row0 + k < p.total) {
                    p.positions[row0 + k] = at[k];
                    p.slots[row0 + k] = slot[k];
                }
        }
    }
}

// One launch for up to kFused sequences: every CTA sums all their lengths for
// itself and plans its own rows; the first writes what belongs to the
// sequences.  Outputs must not lie over inputs that the other CTAs still read.
__global__ void __launch_bounds__(kPlanThreads) k_plan(PlanParams p) {
    __shared__ Seq seqs[kFused + 1];
    const int thread = threadIdx.x;
    const Page page{(uint32_t)p.page, p.shift};
    int first, left;
    ring_state(p.span, p.size, first, left);
    int held[kEach], kept[kEach], fresh[kEach], want[kEach];
    long long tokens = 0, pages = 0, all[2];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = i * kPlanThreads + thread;
        held[i] = s < p.seqs ? p.held[s] : 0;
        fresh[i] = s < p.seqs ? p.fresh[s] : 0;
    }
    // each thread's sequences side by side
    if (p.seqs > kPlanThreads) {
        int* const turn = reinterpret_cast<int*>(seqs);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            turn[i * kPlanThreads + thread] = held[i];
            turn[kFused + i * kPlanThreads + thread] = fresh[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            held[i] = turn[thread * kEach + i];
            fresh[i] = turn[kFused + thread * kEach + i];
        }
        __syncthreads();
    }
    const int each = p.seqs > kPlanThreads ? kEach : 1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        held[i] = length(held[i]);
        fresh[i] = length(fresh[i]);
        kept[i] = together(held[i], fresh[i]);
        want[i] = wanted(held[i], kept[i], page, p.width);
        if (i >= each) continue;
        tokens += fresh[i];
        pages += want[i];
    }
    scan2<kPlanThreads>(tokens, pages, all);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (i >= each) continue;
        const int s = thread * each + i;
        seqs[s] = {clamp32(tokens), held[i], page.many(held[i]), clamp32(pages)};
        if (blockIdx.x == 0 && s < p.seqs) {
            p.kept[s] = kept[i];
            p.starts[s] = clamp32(tokens);
        }
        tokens += fresh[i];
        pages += want[i];
    }
    if (thread == 0) {
        if (blockIdx.x == 0) {
            p.starts[p.seqs] = clamp32(all[0]);
            plan_span(p, first, left, all[1]);
        }
    }
    __syncthreads();
    if (thread == 0) seqs[p.seqs].start = clamp32(all[0]);
    __syncthreads();
    plan_rows(p, seqs, first, left, clamp32(all[0]), clamp32(all[1]));
}

// The general form, two launches: one CTA sums the lengths into the scratch
// (first, left and both sums, then the sequences), then the rows are
// planned from it.
constexpr int kScanThreads = 1024;
__global__ void __launch_bounds__(kScanThreads) k_plan_scan(PlanParams p) {
    chain_release();
    int first, left;
    ring_state(p.span, p.size, first, left);
    __syncthreads();                         // span may be span_out
    const Page page{(uint32_t)p.page, p.shift};
    Seq* const out = reinterpret_cast<Seq*>(p.scratch + 4);
    long long tokens0 = 0, pages0 = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += kScanThreads) {
        const int s = s0 + threadIdx.x;
        const bool in = s < p.seqs;
        const int held = in ? length(p.held[s]) : 0, fresh = in ? length(p.fresh[s]) : 0, kept = together(held, fresh);
        long long tokens = fresh, pages = wanted(held, kept, page, p.width), all[2];
        scan2<kScanThreads>(tokens, pages, all);
        if (in) {
            out[s] = {clamp32(tokens0 + tokens), held, page.many(held), clamp32(pages0 + pages)};
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
        out[p.seqs] = {clamp32(tokens0), 0, 0, 0};
        p.starts[p.seqs] = clamp32(tokens0);
        plan_span(p, first, left, pages0);
    }
}
__global__ void __launch_bounds__(kPlanThreads) k_plan_rows(PlanParams p) {
    chain_wait();
    plan_rows(p, reinterpret_cast<const Seq*>(p.scratch + 4), p.scratch[0], p.scratch[1], p.scratch[2], p.scratch[3]);
}

// One CTA: the finished sequences are listed, a warp counts each one's pages, the
// counts are summed, and the warp that counted them writes them behind the
// ring's last.  Made for the few that end in a step: us, 2 of 48 sequences with 19 pages each 2.8, 6
// of 200 with 79 3.3; many at once are one SM's latency, 1000 with 128 pages each 59, with 512 179.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_free(FreeParams p) {
    __shared__ int which[THREADS], tokens[THREADS], counts[THREADS];
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const Page page{(uint32_t)p.page, p.shift};
    int first, left;
    ring_state(p.span, p.size, first, left);
    long long before = left;
    for (int s0 = 0; s0 < p.seqs; s0 += THREADS) {
        const int s = s0 + threadIdx.x;
        const bool in = s < p.seqs, done = in && p.done[s];
        const int held = in ? p.held[s] : 0;
        if (in) p.held_out[s] = done ? 0 : held;
        long long at = done, none = 0, all[2];
        scan2<THREADS>(at, none, all);                        // (all have read the ring's state, too)
        const int many = (int)all[0];
        if (done) {
            which[at] = s;
            tokens[at] = min(page.many(length(held)), p.width);
        }
        __syncthreads();
        for (int i = warp; i < many; i += kWarps) {
            int n = 0;
            for (int j = lane; j < tokens[i]; j += 32) n += p.pages[(long long)which[i] * p.width + j] >= 0;
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) counts[i] = n;
        }
        __syncthreads();
        at = (int)threadIdx.x < many ? counts[threadIdx.x] : 0;
        scan2<THREADS>(at, none, all);
        if ((int)threadIdx.x < many) counts[threadIdx.x] = (int)min(before + at, (long long)p.size);
        __syncthreads();
        for (int i = warp; i < many; i += kWarps) {
            int to = counts[i];
            for (int j0 = 0; j0 < tokens[i]; j0 += 32) {
                const int number = j0 + lane < tokens[i] ? p.pages[(long long)which[i] * p.width + j0 + lane] : -1;
                const unsigned have = __ballot_sync(0xffffffffu, number >= 0);
                const int mine = to + __popc(have & ((1u << lane) - 1));
                if (number >= 0 && mine < p.size) p.ring[ring_place(first, mine, p.size)] = number;
                to = min(to + __popc(have), p.size);
            }
        }
        __syncthreads();
        before += all[0];
    }
    if (threadIdx.x == 0) {
        p.span_out[0] = first;
        p.span_out[1] = (int)min(before, (long long)p.size);
    }
}

int shift_of(int page) { return (page & (page - 1)) == 0 ? __builtin_ctz((unsigned)page) : -1; }
bool over(const int32_t* a, long long n, const int32_t* b, long long m) { return a < b + m && b < a + n; }

}  // namespace

size_t plan_scratch_bytes(int seqs) { return 16 + ((size_t)seqs + 1) * sizeof(Seq); }

// One launch up to kFused sequences, unless the step is planned in place
// (kept over held, the ring's state over itself), which needs every length to
// be read before the first is written.
cudaError_t launch_plan_pages(const PlanParams& params, cudaStream_t s) {
    PlanParams p = params;
    p.shift = shift_of(p.page);
    p.wide = aligned(p.positions, 16) && aligned(p.slots, 16);
    const long long blocks = (p.total + kPlanThreads * kRows - 1) / (kPlanThreads * kRows);
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

cudaError_t launch_free_pages(const FreeParams& params, cudaStream_t s) {
    FreeParams p = params;
    p.shift = shift_of(p.page);
    if (p.seqs <= 256) k_free<256><<<1, 256, 0, s>>>(p);
    else k_free<1024><<<1, 1024, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace vdt

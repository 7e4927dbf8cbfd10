// k_sample.cu -- the next token of each row of logits, from given random numbers.
//
//   w_i = exp((x_i - max) / T);  tokens in the order of (x descending, index ascending);
//   kept: the first k; of these the ones before which less than p of their sum lies;
//   of these the ones with w_i >= min_p;  token = the first index, in the vocabulary's
//   order, at which the sum of the kept weights passes u times their whole sum
//
// Each of the three conditions keeps a first part of the order, so what is
// kept is everything up to one last token: it is found by its place, without
// sorting the row.  A token hangs on comparisons of sums, so the weights are
// whole numbers, w * 2^45 (less for vocabularies above 2^17), from a polynomial
// in 64 bits: sums are exact, the same in any order, and an answer differs from
// the real numbers' one where u comes within some 2^-34 of a border.
//
// A cluster of CTAs takes a row and holds it in shared memory, so the row is
// read from memory once.  The last kept token is found by histograms, of counts
// for k and of weights for p, over 2048 steps of log2(w) first; when no more than
// kList tokens are left up to its step, one CTA sorts them and finishes; else the
// step itself is searched, by parts of (value, index), and all CTAs sum and
// draw.
#include <cooperative_groups.h>

#include "step_internal.h"

namespace vdt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kList = 1024;
constexpr float kBinsPerOctave = 44.0f;      // kBins - 1 steps are 46.5 octaves, the last ones' weights round to 0
constexpr int kMostBits = 45;

using u64 = unsigned long long;

// Order of the values as whole numbers; -0 is 0, NaN above everything
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// a token's place in the order: smaller is earlier, no two are equal
__device__ __forceinline__ u64 place_of(float x, int index) { return (u64)~key_of(x) << 32 | (uint32_t)index; }

struct Weigher {
    float top, steps;       // the row's largest value; steps of the histogram for two units of the logits
    double octaves;         // log2(e) / T
    int bits;
    __device__ __forceinline__ int bin(float x) const {
        const float d = x == top ? 0.0f : (0.5f * top - 0.5f * x) * steps;     // halves: a difference of two large values is one, too
        return d < (float)(kBins - 1) ? (int)d : kBins - 1;
    }
    // 2^bits exp((x - top) / T) to the nearest whole number.  2^f on [-1/2, 1/2] by the
    // interpolating polynomial of degree 9 at Chebyshev's points, off by at most 2^-45.6.
    __device__ __forceinline__ u64 weight(float x) const {
        if (x == top) return 1ull << bits;
        const double t = ((double)x - (double)top) * octaves;
        if (!(t > -60.0)) return 0;
        const double whole = rint(t), f = t - whole;
        double y = 0x1.b6557c7da8ca4p-24;
        y = fma(y, f, 0x1.63efd536dcb25p-20);
        y = fma(y, f, 0x1.ffcb7a04d3b13p-17);
        y = fma(y, f, 0x1.43088df6dd4a7p-13);
        y = fma(y, f, 0x1.5d87fe8e6c4b1p-10);
        y = fma(y, f, 0x1.3b2ab72b2b245p-7);
        y = fma(y, f, 0x1.c6b08d7045e60p-5);
        y = fma(y, f, 0x1.ebfbdff814945p-3);
        y = fma(y, f, 0x1.62e42fefa39e9p-1);
        y = fma(y, f, 1.0);
        return (u64)__double2ll_rn(y * __hiloint2double((1023 + bits + (int)whole) << 20, 0));
    }
};

struct Shared {
    uint32_t count[kBins], part[3][kBins];   // weights in three parts of 15 bits: a CTA's sums of each stay below 2^32
    u64 list[kList];
    u64 sums[2][8];                          // what the CTAs tell each other, two exchanges in turn
    u64 warp_a[kWarps], warp_b[kWarps];
    u64 found[4];                            // a histogram's step: its number, tokens and weight before it, tokens in it
    u64 total[2];
    unsigned listed;
    int token;
    float logp;
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const u64 o = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)(threadIdx.x % 32) >= d) v += o;
    }
    return v;
}

// floor of a share in [0, 1) of a sum, and whether the product is whole
__device__ __forceinline__ u64 share_of(double share, u64 sum, bool* whole) {
    const u64 f = __double2ull_rz(share * 18446744073709551616.0);
    *whole = f * sum == 0;
    return __umul64hi(f, sum);
}

template <typename T>
struct Row {
    cg::cluster_group cluster;
    Shared& sh;
    const T* slice;          // this CTA's part, in shared or global memory
    int first, n, seg;       // its first index, its length, and what a warp takes of it
    bool held;
    int rank, ranks, turn;
    Weigher w;

    // What each CTA has to say, to all of them: the sum, and the sum of the ranks below
    __device__ __forceinline__ u64 exchange(u64 mine, u64* below = nullptr) {
        u64* const slots = sh.sums[turn];
        turn ^= 1;
        if ((int)threadIdx.x < ranks) cluster.map_shared_rank(slots, threadIdx.x)[rank] = mine;
        cluster.sync();
        u64 all = 0, before = 0;
        for (int i = 0; i < ranks; ++i) {
            if (i == rank) before = all;
            all += slots[i];
        }
        if (below) *below = before;
        return all;
    }
    __device__ __forceinline__ u64 exchange_max(u64 mine) {
        u64* const slots = sh.sums[turn];
        turn ^= 1;
        if ((int)threadIdx.x < ranks) cluster.map_shared_rank(slots, threadIdx.x)[rank] = mine;
        cluster.sync();
        u64 all = 0;
        for (int i = 0; i < ranks; ++i) all = max(all, slots[i]);
        return all;
    }
    __device__ __forceinline__ u64 block_max(u64 v) {
#pragma unroll
        for (int d = 16; d; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        __syncthreads();
        if (threadIdx.x % 32 == 0) sh.warp_a[threadIdx.x / 32] = v;
        __syncthreads();
        v = 0;
        for (int i = 0; i < kWarps; ++i) v = max(v, sh.warp_a[i]);
        return v;
    }

    // Every token of this thread: a warp's are consecutive, a lane's N of them too
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int N = Vec16<T>::N;
        const int lane = threadIdx.x % 32, from = threadIdx.x / 32 * seg, to = min(n, from + seg);
        for (int i0 = from; i0 < to; i0 += 32 * N) {
            const int i = i0 + lane * N;
            float x[N];
            load(i, x);
#pragma unroll
            for (int j = 0; j < N; ++j) f(x[j], i + j);
        }
    }
    // N values; past the end of the part there is -inf
    __device__ __forceinline__ void load(int i, float* x) const {
        constexpr int N = Vec16<T>::N;
        if (held) {
            Vec16<T> v;
            v.raw = *reinterpret_cast<const uint4*>(slice + i);
            v.get(x);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = i + j < n ? to_f32(slice[i + j]) : -INFINITY;
        }
    }

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.count[i] = sh.part[0][i] = sh.part[1][i] = sh.part[2][i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void count(int bin, float x, bool weights) {
        atomicAdd(&sh.count[bin], 1u);
        if (weights) {
            const u64 v = w.weight(x);
            atomicAdd(&sh.part[0][bin], (uint32_t)(v & 0x7fff));
            atomicAdd(&sh.part[1][bin], (uint32_t)(v >> 15 & 0x7fff));
            atomicAdd(&sh.part[2][bin], (uint32_t)(v >> 30));
        }
    }
    // The histogram's step in which the token number `want` (of_weight: the one at
    // whose end the weight reaches `want`; of_share: that share of all the weight,
    // rounded up) lies: {step, tokens before, weight before, tokens in it}, tokens in
    // all, weight in all.  found[0] is kBins where there are not that many.
    struct Found {
        int bin;
        u64 count, weight, in, all_count, all_weight, want;
    };
    __device__ __forceinline__ Found cross(u64 want, bool of_weight, double of_share) {
        cluster.sync();                                       // all histograms are there
        const int mine = kBins / ranks, from = rank * mine;   // this CTA's steps
        if (threadIdx.x == 0) sh.found[0] = kBins;            // (written again after the next exchange alone)
        const int per = (mine + kThreads - 1) / kThreads;     // of a thread: at most 4, consecutive
        u64 c[4] = {}, v[4] = {}, cs = 0, vs = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = threadIdx.x * per + i;
            if (i >= per || b >= mine) continue;
            for (int r = 0; r < ranks; ++r) {
                const Shared* const o = cluster.map_shared_rank(&sh, r);
                c[i] += o->count[from + b];
                v[i] += o->part[0][from + b] + ((u64)o->part[1][from + b] << 15) + ((u64)o->part[2][from + b] << 30);
            }
            cs += c[i];
            vs += v[i];
        }
        const u64 ci = warp_scan(cs), vi = warp_scan(vs);
        if (threadIdx.x % 32 == 31) {
            sh.warp_a[threadIdx.x / 32] = ci;
            sh.warp_b[threadIdx.x / 32] = vi;
        }
        __syncthreads();
        u64 c0 = ci - cs, v0 = vi - vs, ct = 0, vt = 0;
        for (int i = 0; i < kWarps; ++i) {
            if (i < (int)threadIdx.x / 32) {
                c0 += sh.warp_a[i];
                v0 += sh.warp_b[i];
            }
            ct += sh.warp_a[i];
            vt += sh.warp_b[i];
        }
        u64 cb, vb;
        Found r;
        r.all_count = exchange(ct, &cb);
        r.all_weight = exchange(vt, &vb);
        if (of_share >= 0.0) {
            bool whole;
            want = share_of(of_share, r.all_weight, &whole);
            if (!whole) ++want;
            if (!want) want = 1;
        }
        r.want = want;
        c0 += cb;
        v0 += vb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u64 before = of_weight ? v0 : c0, after = before + (of_weight ? v[i] : c[i]);
            if (before < want && want <= after)
                for (int k = 0; k < ranks; ++k) {
                    u64* const f = cluster.map_shared_rank(sh.found, k);
                    f[1] = c0;
                    f[2] = v0;
                    f[3] = c[i];
                    f[0] = from + threadIdx.x * per + i;
                }
            c0 += c[i];
            v0 += v[i];
        }
        cluster.sync();
        r.bin = (int)sh.found[0];
        r.count = sh.found[1];
        r.weight = sh.found[2];
        r.in = sh.found[3];
        return r;
    }

    // The places of the tokens that `take` wants, into the first CTA's list
    template <typename F>
    __device__ __forceinline__ unsigned gather(F take) {
        if (threadIdx.x == 0) sh.listed = 0;
        cluster.sync();
        unsigned* const listed = cluster.map_shared_rank(&sh.listed, 0);
        u64* const list = cluster.map_shared_rank(sh.list, 0);
        each([&](float x, int i) {
            const bool mine = take(x, i);
            if (mine) {
                const unsigned at = atomicAdd(listed, 1u);
                if (at < kList) list[at] = place_of(x, first + i);
            }
        });
        cluster.sync();
        return rank == 0 ? min(sh.listed, (unsigned)kList) : 0;     // the others may go on after the first CTA has ended
    }
};

// Ascending, in place; every thread of the CTA
__device__ __forceinline__ void sort_list(u64* a, unsigned n) {
    unsigned size = 2;
    while (size < n) size *= 2;
    for (unsigned i = n + threadIdx.x; i < size; i += kThreads) a[i] = ~0ull;
    __syncthreads();
    for (unsigned run = 2; run <= size; run *= 2)
        for (unsigned gap = run / 2; gap; gap /= 2) {
            for (unsigned i = threadIdx.x; i < size / 2; i += kThreads) {
                const unsigned lo = i / gap * gap * 2 + i % gap, hi = lo + gap;
                const bool up = (lo & run) == 0;
                const u64 x = a[lo], y = a[hi];
                if ((x > y) == up) {
                    a[lo] = y;
                    a[hi] = x;
                }
            }
            __syncthreads();
        }
}

// Sums before each of a thread's two neighbours in the list (2 * thread, 2 * thread + 1)
__device__ __forceinline__ u64 scan_list(Shared& sh, u64 a, u64 b, u64* total) {
    const u64 mine = a + b, upto = warp_scan(mine);
    __syncthreads();
    if (threadIdx.x % 32 == 31) sh.warp_a[threadIdx.x / 32] = upto;
    __syncthreads();
    u64 before = upto - mine, all = 0;
    for (int i = 0; i < kWarps; ++i) {
        if (i < (int)threadIdx.x / 32) before += sh.warp_a[i];
        all += sh.warp_a[i];
    }
    *total = all;
    return before;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(SampleParams p, int part, int held) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ Shared sh;
    constexpr int N = Vec16<T>::N;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long r = blockIdx.x / ranks;
    const int first = rank * part, n = max(0, min(p.vocab - first, part));
    const T* const row = static_cast<const T*>(p.logits) + r * p.stride + first;
    const int seg = ((part + kWarps - 1) / kWarps + 32 * N - 1) / (32 * N) * (32 * N);
    Row<T> s{cluster, sh, row, first, n, seg, held != 0, rank, ranks, 0, {}};
    if (held) {
        T* const mine = reinterpret_cast<T*>(memory);
        const bool wide = reinterpret_cast<uintptr_t>(row) % 16 == 0;
        const int vecs = wide ? n / N : 0, room = kWarps * seg;
        for (int i = threadIdx.x; i < vecs; i += kThreads) reinterpret_cast<uint4*>(mine)[i] = __ldg(reinterpret_cast<const uint4*>(row) + i);
        for (int i = vecs * N + threadIdx.x; i < room; i += kThreads) mine[i] = i < n ? row[i] : from_f32<T>(-INFINITY);
        s.slice = mine;
        __syncthreads();
    }
    const float temperature = p.temperatures ? p.temperatures[r] : p.temperature, top_p = p.top_ps ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps ? p.min_ps[r] : p.min_p, u = p.u[r];
    const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const bool greedy = temperature == 0.0f;

    // the largest value and the lowest index that has it
    u64 best = 0;
    s.each([&](float x, int i) { best = max(best, (u64)key_of(x) << 32 | (uint32_t)~(first + i)); });
    best = s.exchange_max(s.block_max(best));
    const uint32_t top = (uint32_t)(best >> 32);
    const bool fine = top != 0xffffffffu && top != key_of(-INFINITY) && temperature >= 0.0f && temperature < INFINITY && top_p == top_p &&
                      min_p == min_p && (greedy || (u >= 0.0f && u < 1.0f));
    if (!fine || greedy) {
        if (rank == 0 && threadIdx.x == 0) {
            p.tokens[r] = fine ? (int)~(uint32_t)best : -1;
            if (p.logp) p.logp[r] = fine ? 0.0f : NAN;
        }
        cluster.sync();
        return;
    }
    Weigher& w = s.w;
    w.top = value_of(top);
    w.octaves = 1.4426950408889634 / (double)temperature;
    w.steps = fminf((float)w.octaves * (2.0f * kBinsPerOctave), 3.0e38f);
    w.bits = min(kMostBits, 62 - (32 - __clz(p.vocab - 1)));
    const u64 least = __double2ull_ru((double)fminf(fmaxf(min_p, 0.0f), 1.0f) * (double)(1ull << w.bits));

    bool by_count = top_k > 0 && top_k < p.vocab;
    const bool by_weight = top_p < 1.0f;
    u64 last = ~0ull;                 // the last kept token's place
    bool listed = false;
    u64 limit_k = ~0ull, limit_w = ~0ull;
    unsigned in_list = 0;
    for (int pass = 0; pass < 2 && !listed; ++pass) {
        const bool weights = pass == 1;
        if (weights ? !by_weight : !by_count) continue;
        s.clear();
        s.each([&](float x, int i) {
            const int b = w.bin(x);
            if (b < kBins - 1 && (last == ~0ull || place_of(x, first + i) <= last)) s.count(b, x, weights);
        });
        auto at = s.cross(weights ? 0 : (u64)top_k, weights, weights ? fmaxf(top_p, 0.0f) : -1.0);
        if (at.bin == kBins) continue;                    // fewer tokens than k have any weight
        if (at.count + at.in <= kList) {
            // few tokens up to the step: the first CTA has them all
            if (weights) limit_w = at.want;
            else limit_k = (u64)top_k;
            const int upto = at.bin;
            const u64 end = last;
            in_list = s.gather([&](float x, int i) { return w.bin(x) <= upto && (end == ~0ull || place_of(x, first + i) <= end); });
            listed = true;
            break;
        }
        // the step is searched by (value, index): parts of it, until few tokens are left
        const int bin = at.bin;
        u64 want = at.want - (weights ? at.weight : at.count), in = at.in, lo = 0, hi = last;
        for (int round = 0; round < 8 && in > kList; ++round) {          // 2^11 parts each: 64 bits are through before
            u64 low = 0, high = 0;                        // the first (inverted) and last place in the range
            s.each([&](float x, int i) {
                const u64 o = place_of(x, first + i);
                if (w.bin(x) == bin && o >= lo && o <= hi) {
                    low = max(low, ~o);
                    high = max(high, o);
                }
            });
            lo = ~s.exchange_max(s.block_max(low));
            hi = s.exchange_max(s.block_max(high));
            const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
            s.clear();
            s.each([&](float x, int i) {
                const u64 o = place_of(x, first + i);
                if (w.bin(x) == bin && o >= lo && o <= hi) s.count((int)((o - lo) >> shift), x, weights);
            });
            at = s.cross(want, weights, -1.0);
            want -= weights ? at.weight : at.count;
            in = at.in;
            lo += (u64)at.bin << shift;
            hi = min(hi, lo + ((1ull << shift) - 1));
        }
        const unsigned few = s.gather([&](float x, int i) {
            const u64 o = place_of(x, first + i);
            return w.bin(x) == bin && o >= lo && o <= hi;
        });
        if (rank == 0) {
            sort_list(sh.list, few);
            const unsigned a = 2 * threadIdx.x;
            u64 before = 0, va = 0, vb = 0, all;
            if (a < few) va = weights ? w.weight(value_of(~(uint32_t)(sh.list[a] >> 32))) : 1;
            if (a + 1 < few) vb = weights ? w.weight(value_of(~(uint32_t)(sh.list[a + 1] >> 32))) : 1;
            before = scan_list(sh, va, vb, &all);
            // the last one with less than `want` before it
            if (a < few && before < want && (before + va >= want || a + 1 >= few)) sh.total[0] = sh.list[a];
            if (a + 1 < few && before + va < want && (before + va + vb >= want || a + 2 >= few)) sh.total[0] = sh.list[a + 1];
        }
        cluster.sync();
        last = *cluster.map_shared_rank(&sh.total[0], 0);
        cluster.sync();
    }

    const double share = u;
    bool whole;
    if (listed) {
        if (rank == 0) {
            sort_list(sh.list, in_list);
            const unsigned a = 2 * threadIdx.x;
            const u64 oa = a < in_list ? sh.list[a] : ~0ull, ob = a + 1 < in_list ? sh.list[a + 1] : ~0ull;
            u64 va = a < in_list && a < limit_k ? w.weight(value_of(~(uint32_t)(oa >> 32))) : 0;
            u64 vb = a + 1 < in_list && a + 1 < limit_k ? w.weight(value_of(~(uint32_t)(ob >> 32))) : 0;
            u64 sum, kept;
            const u64 before = scan_list(sh, va, vb, &sum);
            if (limit_w == ~0ull && by_weight) {
                limit_w = share_of(fmaxf(top_p, 0.0f), sum, &whole);
                if (!whole) ++limit_w;
                if (!limit_w) limit_w = 1;
            }
            if (before + va >= limit_w) vb = 0;
            if (before >= limit_w) va = 0;
            if (va < least) va = 0;
            if (vb < least) vb = 0;
            scan_list(sh, va, vb, &kept);
            const u64 target = share_of(share, kept, &whole);
            // the kept ones again, in the vocabulary's order
            __syncthreads();
            if (a < in_list) sh.list[a] = va ? oa << 32 | oa >> 32 : ~0ull;
            if (a + 1 < in_list) sh.list[a + 1] = vb ? ob << 32 | ob >> 32 : ~0ull;
            __syncthreads();
            sort_list(sh.list, in_list);
            const u64 ia = a < in_list ? sh.list[a] : ~0ull, ib = a + 1 < in_list ? sh.list[a + 1] : ~0ull;
            va = ia != ~0ull ? w.weight(value_of(~(uint32_t)ia)) : 0;
            vb = ib != ~0ull ? w.weight(value_of(~(uint32_t)ib)) : 0;
            const u64 upto = scan_list(sh, va, vb, &kept);
            const bool here_a = upto <= target && target < upto + va, here_b = upto + va <= target && target < upto + va + vb;
            if (here_a || here_b) {
                p.tokens[r] = (int)((here_a ? ia : ib) >> 32);
                if (p.logp) p.logp[r] = (float)log((double)(here_a ? va : vb) / (double)kept);
            }
        }
        return;
    }

    // everything up to `last`: each warp's sum, each CTA's, the whole; then the warp in
    // which the sum passes the target goes through its part once more
    auto weight = [&](float x, int i) -> u64 {
        if (last != ~0ull && place_of(x, first + i) > last) return 0;
        const u64 v = w.weight(x);
        return v >= least ? v : 0;
    };
    u64 mine = 0;
    s.each([&](float x, int i) { mine += weight(x, i); });
    mine = warp_sum(mine);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.warp_b[threadIdx.x / 32] = mine;
    __syncthreads();
    u64 here = 0, before = 0, below;
    for (int i = 0; i < kWarps; ++i) {
        if (i < (int)threadIdx.x / 32) before += sh.warp_b[i];
        here += sh.warp_b[i];
    }
    const u64 sum = s.exchange(here, &below);
    const u64 target = share_of(share, sum, &whole);
    before += below;
    if (before <= target && target < before + mine) {
        const int lane = threadIdx.x % 32, from = threadIdx.x / 32 * seg;
        for (int i0 = from; i0 < min(n, from + seg); i0 += 32 * N) {
            float x[N];
            s.load(i0 + lane * N, x);
            u64 v[N], lane_sum = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) lane_sum += v[j] = weight(x[j], i0 + lane * N + j);
            const u64 upto = warp_scan(lane_sum), all = __shfl_sync(0xffffffffu, upto, 31);
            if (target < before + all) {
                u64 at = before + upto - lane_sum;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (at <= target && target < at + v[j]) {
                        p.tokens[r] = first + i0 + lane * N + j;
                        if (p.logp) p.logp[r] = (float)log((double)v[j] / (double)sum);
                    }
                    at += v[j];
                }
                break;
            }
            before += all;
        }
    }
}

template <typename T>
cudaError_t sample_launch(const SampleParams& p, cudaStream_t s) {
    // as many CTAs a row as it takes to put the GPU to work, and to hold the row
    constexpr int N = Vec16<T>::N, kRoom = 160 * 1024;
    auto part_of = [&](int ranks) { return ((p.vocab + ranks - 1) / ranks + N - 1) / N * N; };
    auto bytes_of = [&](int ranks) {
        const int seg = ((part_of(ranks) + kWarps - 1) / kWarps + 32 * N - 1) / (32 * N) * (32 * N);
        return (long long)kWarps * seg * (long long)sizeof(T);
    };
    int ranks = 1;
    while (ranks < 8 && ((p.rows * ranks * 2 <= kSmCount && part_of(ranks * 2) >= 1024) || bytes_of(ranks) > kRoom || part_of(ranks) > 1 << 16)) ranks *= 2;
    const bool held = bytes_of(ranks) <= kRoom;
    const cudaError_t e = allow_shared<k_sample<T>>(kRoom);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = held ? (size_t)bytes_of(ranks) : 0;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_sample<T>, p, part_of(ranks), (int)held);
}

}  // namespace

cudaError_t launch_sample(const SampleParams& p, cudaStream_t s) {
    if (p.type == VDT_F32) return sample_launch<float>(p, s);
    if (p.type == VDT_F16) return sample_launch<__half>(p, s);
    return sample_launch<__nv_bfloat16>(p, s);
}

}  // namespace vdt

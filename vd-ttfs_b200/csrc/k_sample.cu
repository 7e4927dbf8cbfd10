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
// whole numbers, w * 2^44 (2^43 for vocabularies above 2^18), from a polynomial
// in 64 bits: sums are exact, the same in any order, and an answer differs from
// the real numbers' one where u comes within some 2^-34 of a border.
//
// One CTA takes a row, or a cluster of them where rows are few; what does not fit
// beside the histograms in shared memory is read again from L2.  A histogram of
// the tokens over 2048 steps of log2(w), 44 an octave, gives the step of the
// token number k, and, since a step's weights are within a 44th of an octave of
// each other, bounds of the few steps in which the last token for p lies.  One pass
// then sums all weights and those before these steps, and lists the steps'
// tokens; they are told apart by finer histograms while there are many of them, and
// sorted in the end.  Where no more than kList tokens come up to there, one CTA
// sorts them all and finishes; else all CTAs sum what is kept, and the part of the
// warp in which the sum passes the target is gone through again.
#include <cooperative_groups.h>

#include <cfloat>

#include "step_internal.h"

namespace vdt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kRoom = kBins + 4, kList = 1024, kChosen = 8192;
constexpr float kSteps = 44.0f;              // of an octave; kBins of them are 46.5 octaves, below which weights round to 0
constexpr int kMostBits = 44, kBoundBits = 40;

using u64 = unsigned long long;

// Order of the values as whole numbers; -0 is 0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// a token's place in the order: smaller is earlier, no two are equal
__device__ __forceinline__ u64 place_of(float x, int index) { return (u64)~key_of(x) << 32 | (uint32_t)index; }
__device__ __forceinline__ float value_at(u64 place) { return value_of(~(uint32_t)(place >> 32)); }

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
// the largest of many values; NaN where one is
template <typename T>
struct Top {
    __nv_bfloat162 a = {__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80)};
    __device__ __forceinline__ void add(const Vec16<T>& v) {
        const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 b;
            memcpy(&b, &w[i], 4);
            a = __hmax2_nan(a, b);
        }
    }
    __device__ __forceinline__ float value() const { return max_or_nan(__low2float(a), __high2float(a)); }
};
template <>
struct Top<__half> {
    __half2 a = {__ushort_as_half(0xfc00), __ushort_as_half(0xfc00)};
    __device__ __forceinline__ void add(const Vec16<__half>& v) {
        const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __half2 b;
            memcpy(&b, &w[i], 4);
            a = __hmax2_nan(a, b);
        }
    }
    __device__ __forceinline__ float value() const { return max_or_nan(__low2float(a), __high2float(a)); }
};
template <>
struct Top<float> {
    float a = -INFINITY;
    __device__ __forceinline__ void add(const Vec16<float>& v) {
        a = max_or_nan(a, max_or_nan(max_or_nan(__uint_as_float(v.raw.x), __uint_as_float(v.raw.y)),
                                     max_or_nan(__uint_as_float(v.raw.z), __uint_as_float(v.raw.w))));
    }
    __device__ __forceinline__ float value() const { return a; }
};

struct Weigher {
    float top, bottom;      // the row's largest value; one whose weight is 0
    float part, part_top, steps;
    double octaves;         // log2(e) / T
    int bits;
    __device__ __forceinline__ void set(float largest, float temperature, int vocab) {
        top = largest;
        octaves = 1.4426950408889634 / (double)temperature;
        float below = value_of(key_of(top) - 1);             // the next value below (0's is not -0)
        if (below == top) below = value_of(key_of(top) - 2);
        bottom = fmaxf(fminf(__double2float_rd((double)top - 80.0 / octaves), below), -FLT_MAX);
        // of large logits halves, whose difference is always a number
        part = fabsf(top) > 1e30f ? 0.5f : 1.0f;
        part_top = part * top;
        steps = (float)(octaves / (double)part * (double)kSteps);
        bits = min(kMostBits, 62 - (32 - __clz(vocab - 1)));
        // the next value below the largest has no weight by far: no exponent below a double's
        const double span = (double)top - (double)bottom;
        if (span * octaves > 900.0) octaves = 80.0 / span;
    }
    // steps below the largest; kBins for all without weight
    __device__ __forceinline__ float depth(float x) const { return fminf(fmaf(-part, x, part_top) * steps, (float)kBins); }
    // the step itself: floor in the low bits of 2^23 + depth
    static __device__ __forceinline__ int step(float depth) { return __float_as_int(__fadd_rd(depth, 8388608.0f)) & (2 * kBins - 1); }
    // 2^bits exp((x - top) / T) to the nearest whole number.  2^f on [-1/2, 1/2] by the
    // interpolating polynomial of degree 8 at Chebyshev's points, off by at most 2^-39.7.
    // 3/2 2^52 added leaves the nearest whole number in the low bits; no branches, so that
    // the chains of several tokens run side by side.
    __device__ __forceinline__ u64 weight(float x) const {
        constexpr double kRound = 6755399441055744.0;
        const double d = (double)fmaxf(x, bottom) - (double)top;
        const double z = fma(d, octaves, kRound), f = fma(d, octaves, kRound - z);
        double y = 0x1.63d0e49869220p-20;
        y = fma(y, f, 0x1.00dc4b54b68d6p-16);
        y = fma(y, f, 0x1.4308acd88a0d7p-13);
        y = fma(y, f, 0x1.5d8745a58ae45p-10);
        y = fma(y, f, 0x1.3b2ab717e98f6p-7);
        y = fma(y, f, 0x1.c6b08dd6fe736p-5);
        y = fma(y, f, 0x1.ebfbdff823ef1p-3);
        y = fma(y, f, 0x1.62e42fef84ceep-1);
        y = fma(y, f, 1.0);
        y = fma(y, __hiloint2double((1023 + bits + __double2loint(z)) << 20, 0), 4503599627370496.0);
        return (u64)__double_as_longlong(y) & 0xfffffffffffffull;
    }
};

// A histogram, weights in three parts of 15 bits (a CTA's sums of each stay below
// 2^32; the row's first histogram, of counts alone, has four copies there, each
// for a quarter of the lanes: tokens of 16 bits have few values, and lanes with the
// same one wait for each other), and the tokens of the steps that are looked into
struct Work {
    uint32_t count[4][kRoom];                // (kBins: tokens without weight; later counts, and the weights' parts)
    int chosen[kChosen];
};
struct Shared {
    u64 list[kList];
    u64 said[2][8][3];                       // what the CTAs tell each other, two exchanges in turn
    u64 warps[3][kWarps];
    u64 found[4];
    u64 kept[kWarps];                        // weight of what each warp's part keeps
    u64 last;
    unsigned listed, chosen;
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
// Sums before each thread's own, in the CTA; the whole sums in `all`
template <int K>
__device__ __forceinline__ void block_scan(Shared& sh, u64 (&v)[K], u64 (&all)[K]) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    u64 own[K];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        own[k] = v[k];
        v[k] = warp_scan(v[k]);
        if (lane == 31) sh.warps[k][warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const u64 w = lane < kWarps ? sh.warps[k][lane] : 0, upto = warp_scan(w);
        all[k] = __shfl_sync(0xffffffffu, upto, 31);
        v[k] += __shfl_sync(0xffffffffu, upto - w, warp) - own[k];
    }
}
template <int K>
__device__ __forceinline__ void block_sum(Shared& sh, u64 (&v)[K]) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = warp_sum(v[k]);
        if (threadIdx.x % 32 == 0) sh.warps[k][threadIdx.x / 32] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(threadIdx.x % 32 < kWarps ? sh.warps[k][threadIdx.x % 32] : 0);
}

// floor of a share in [0, 1) of a sum, and whether the product is whole
__device__ __forceinline__ u64 share_of(double share, u64 sum, bool* whole) {
    const u64 f = __double2ull_rz(share * 18446744073709551616.0);
    *whole = f * sum == 0;
    return __umul64hi(f, sum);
}
// the weight that top_p wants of a sum: the share rounded up, at least something
__device__ __forceinline__ u64 want_of(float top_p, u64 sum) {
    bool whole;
    const u64 w = share_of(fmaxf(top_p, 0.0f), sum, &whole);
    return max(w + !whole, 1ull);
}

template <typename T>
struct Row {
    static constexpr int N = Vec16<T>::N;
    cg::cluster_group cluster;
    Shared& sh;
    Work& wk;
    const T* slice;          // this CTA's part
    int first, n, seg;       // its first index, its length, and what a warp takes of it
    bool wide, endless;      // endless: the largest value is +inf, which counts as 0 then, and all others as -inf
    bool tiny;               // logits and temperature count 2^90 times, for the smallest of them
    int rank, ranks, turn;
    u64 end;                 // the last token's place that counts, as far as it is known
    Weigher w;

    __device__ __forceinline__ void together() const {
        if (ranks > 1) cluster.sync();
        else __syncthreads();
    }
    // What each CTA has to say, to all of them
    template <int K>
    __device__ __forceinline__ u64 (&say(const u64 (&mine)[K]))[8][3] {
        u64 (&slots)[8][3] = sh.said[turn];
        turn ^= 1;
        if ((int)threadIdx.x < ranks) {
            u64* const to = cluster.map_shared_rank(&slots[rank][0], threadIdx.x);
#pragma unroll
            for (int k = 0; k < K; ++k) to[k] = mine[k];
        }
        together();
        return slots;
    }
    // sums over the CTAs; `below` (of the first): over the ranks below
    template <int K>
    __device__ __forceinline__ u64 say_sum(u64 (&v)[K]) {
        const auto& slots = say(v);
        u64 below = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0;
        for (int i = 0; i < ranks; ++i) {
            if (i == rank) below = v[0];
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += slots[i][k];
        }
        return below;
    }
    __device__ __forceinline__ u64 say_max(u64 mine) {
        const u64 v[1] = {mine};
        const auto& slots = say(v);
        u64 all = 0;
        for (int i = 0; i < ranks; ++i) all = max(all, slots[i][0]);
        return all;
    }
    __device__ __forceinline__ u64 block_max(u64 v) {
#pragma unroll
        for (int d = 16; d; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        __syncthreads();
        if (threadIdx.x % 32 == 0) sh.warps[0][threadIdx.x / 32] = v;
        __syncthreads();
        v = threadIdx.x % 32 < kWarps ? sh.warps[0][threadIdx.x % 32] : 0;
#pragma unroll
        for (int d = 16; d; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    }

    // N values; past the end of the part there is -inf
    __device__ __forceinline__ Vec16<T> load(int i) const {
        Vec16<T> v;
        if (wide && i + N <= n) {
            v.raw = *reinterpret_cast<const uint4*>(slice + i);
        } else {
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = i + j < n ? to_f32(slice[i + j]) : -INFINITY;
            v.set(x);
        }
        return v;
    }
    __device__ __forceinline__ float value(float x) const { return endless ? (x == INFINITY ? 0.0f : -INFINITY) : tiny ? x * 0x1p90f : x; }
    __device__ __forceinline__ void values(const Vec16<T>& v, float* x) const {
        v.get(x);
        if (endless || tiny)
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = value(x[j]);
    }
    // Every N tokens of this thread: a warp's are consecutive, a lane's N of them too;
    // the next are on their way meanwhile
    template <typename F>
    __device__ __forceinline__ void each_vector(F f) const {
        const int from = threadIdx.x / 32 * seg, to = min(n, from + seg), step = 32 * N;
        if (from >= to) return;
        int i = from + (int)(threadIdx.x % 32) * N;
        Vec16<T> next = load(i);
        for (int i0 = from; i0 < to; i0 += step, i += step) {
            const Vec16<T> v = next;
            if (i0 + step < to) next = load(i + step);
            float x[N];
            values(v, x);
            f(x, i);
        }
    }
    // the same as they lie, several vectors on their way
    template <typename F>
    __device__ __forceinline__ void each_load(F f) const {
        const int from = threadIdx.x / 32 * seg, to = min(n, from + seg);
#pragma unroll 4
        for (int i0 = from; i0 < to; i0 += 32 * N) f(load(i0 + (int)(threadIdx.x % 32) * N));
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each_vector([&](const float* x, int i) {
#pragma unroll
            for (int j = 0; j < N; ++j) f(x[j], i + j);
        });
    }

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < kRoom; i += kThreads) reinterpret_cast<uint4*>(&wk.count[0][0])[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    __device__ __forceinline__ void count(int bin, float x, bool weights) {
        atomicAdd(&wk.count[0][bin], 1u);
        if (weights) {
            const u64 v = w.weight(x);
            atomicAdd(&wk.count[1][bin], (uint32_t)(v & 0x7fff));
            atomicAdd(&wk.count[2][bin], (uint32_t)(v >> 15 & 0x7fff));
            atomicAdd(&wk.count[3][bin], (uint32_t)(v >> 30));
        }
    }
    __device__ __forceinline__ bool before_end(float x, int i) const { return place_of(x, first + i) <= end; }
    // The row's histogram, of the tokens up to the place `end` (PART), or of all
    template <bool PART>
    __device__ __forceinline__ void histogram() {
        clear();
        uint32_t* const copy = &wk.count[threadIdx.x % 4][0];
        each([&](float x, int i) {
            const int b = Weigher::step(w.depth(x));
            atomicAdd(copy + (!PART || before_end(x, i) ? b : kBins), 1u);
        });
    }

    // The steps of the row's histogram in which the last kept token may lie, for the
    // count k (k >= 0), or else for the share top_p of the weight: by a step's bounds
    // of its tokens' weights, in multiples of 2^-40, of the sums and of the whole.
    struct Steps {
        int from, to;               // from == kBins: there is no such token
        u64 before, upto;           // tokens before `from`, and up to `to`
    };
    __device__ __forceinline__ Steps steps_for(int k, float top_p) {
        constexpr int kPer = kBins / kThreads;
        static_assert(kPer == 4, "four steps a thread");
        const int mine = kPer * threadIdx.x;
        __syncthreads();
        auto add = [](uint4 a, uint4 b) { return make_uint4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); };
        uint4 sum = *reinterpret_cast<const uint4*>(&wk.count[0][mine]);
#pragma unroll
        for (int k = 1; k < 4; ++k) sum = add(sum, *reinterpret_cast<const uint4*>(&wk.count[k][mine]));
        if (ranks > 1) {
            *reinterpret_cast<uint4*>(&wk.count[0][mine]) = sum;
            cluster.sync();                                   // all histograms are there
            uint4 o[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                o[r] = r < ranks ? *reinterpret_cast<const uint4*>(&cluster.map_shared_rank(&wk, r)->count[0][mine]) : make_uint4(0, 0, 0, 0);
            sum = o[0];
#pragma unroll
            for (int r = 1; r < 8; ++r) sum = add(sum, o[r]);
        }
        const uint32_t c[kPer] = {sum.x, sum.y, sum.z, sum.w};
        // bounds of a step's weight; it counts as wider than it is by 2^-16, for the 32-bit depths and exponentials
        auto under = [](int b) { return (u64)(exp2f((float)kBoundBits - (b + 1.0f) / kSteps) * (1.0f - 0x1p-16f)); };
        auto over = [](int b) { return (u64)(exp2f((float)kBoundBits - b / kSteps) * (1.0f + 0x1p-16f)) + 1; };
        u64 v[3] = {}, all[3];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            v[0] += c[i];
            v[1] += c[i] * under(mine + i);
            v[2] += c[i] * over(mine + i);
        }
        if (threadIdx.x == 0) {
            sh.found[0] = sh.found[1] = kBins;
            sh.found[3] = 0;
        }
        block_scan(sh, v, all);
        // the first step up to which there may be enough, and the first up to which there is
        bool whole;
        u64 least, most;
        if (k >= 0) {
            least = most = (u64)k;
        } else {
            least = max(share_of(fmaxf(top_p, 0.0f), all[1], &whole), 1ull);
            most = min(share_of(fmaxf(top_p, 0.0f), all[2], &whole) + 2, all[1]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const u64 lo = c[i] * under(mine + i), hi = c[i] * over(mine + i);
            const u64 a = k >= 0 ? v[0] : v[2], b = k >= 0 ? v[0] : v[1];
            if (a < least && least <= a + (k >= 0 ? c[i] : hi)) {
                sh.found[0] = mine + i;
                sh.found[2] = v[0];
            }
            if (b < most && most <= b + (k >= 0 ? c[i] : lo)) {
                sh.found[1] = mine + i;
                sh.found[3] = v[0] + c[i];
            }
            v[0] += c[i];
            v[1] += lo;
            v[2] += hi;
        }
        __syncthreads();
        return {(int)sh.found[0], (int)sh.found[1], sh.found[2], sh.found[3]};
    }

    // The part of a histogram of counts and weights in which the token number `want`,
    // or the one at whose end the weight reaches `want`, lies
    struct Part {
        int bin;
        u64 count, weight, in;      // tokens and weight before it, tokens in it
    };
    __device__ __forceinline__ Part cross(u64 want, bool of_weight) {
        together();                                           // all histograms are there
        constexpr int kPer = kBins / kThreads;
        const int mine = kBins / ranks, from = rank * mine;   // this CTA's parts
        const int per = (mine + kThreads - 1) / kThreads;     // of a thread: at most kPer, consecutive
        u64 c[kPer] = {}, v[kPer] = {}, sums[2] = {}, all[2];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = threadIdx.x * per + i;
            if (i >= per || b >= mine) continue;
            for (int r = 0; r < ranks; ++r) {
                const Work* const o = cluster.map_shared_rank(&wk, r);
                c[i] += o->count[0][from + b];
                v[i] += o->count[1][from + b] + ((u64)o->count[2][from + b] << 15) + ((u64)o->count[3][from + b] << 30);
            }
            sums[0] += c[i];
            sums[1] += v[i];
        }
        block_scan(sh, sums, all);
        const auto& slots = say(all);
        u64 c0 = sums[0], v0 = sums[1];
        for (int r = 0; r < rank; ++r) {
            c0 += slots[r][0];
            v0 += slots[r][1];
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const u64 before = of_weight ? v0 : c0, after = before + (of_weight ? v[i] : c[i]);
            if (before < want && want <= after)
                for (int k = 0; k < ranks; ++k) {
                    u64* const f = cluster.map_shared_rank(sh.found, k);
                    f[0] = from + threadIdx.x * per + i;
                    f[1] = c0;
                    f[2] = v0;
                    f[3] = c[i];
                }
            c0 += c[i];
            v0 += v[i];
        }
        together();
        const Part r{(int)sh.found[0], sh.found[1], sh.found[2], sh.found[3]};
        __syncthreads();
        return r;
    }

    // into the first CTA's list
    __device__ __forceinline__ void put(u64 place) {
        const unsigned at = atomicAdd(cluster.map_shared_rank(&sh.listed, 0), 1u);
        if (at < kList) cluster.map_shared_rank(sh.list, 0)[at] = place;
    }
    // its length, for the first CTA alone: the others may go on after that one has ended
    __device__ __forceinline__ unsigned in_list() const { return rank == 0 ? min(sh.listed, (unsigned)kList) : 0; }

    // One pass over the row's tokens (PART: up to the place `end`): with WEIGHTS their
    // weights' sum, and the sum of those in steps before `from`, each warp's into `kept`;
    // and the tokens of the steps from..to into `chosen`, or of all steps up to `to`
    // into the first CTA's list.
    template <bool PART, bool WEIGHTS>
    __device__ __forceinline__ void look(int from, int to, bool list, u64 (&sums)[2], bool* fits) {
        if (threadIdx.x == 0) sh.listed = sh.chosen = 0;
        together();
        sums[0] = sums[1] = 0;
        const float upto = (float)(to + 1), since = (float)from, first_step = list ? 0.0f : since;
        each_vector([&](const float* x, int i) {
            unsigned mine = 0, in = 0;
            float d[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                d[j] = w.depth(x[j]);
                if (PART && before_end(x[j], i + j)) in |= 1u << j;
                if (d[j] < upto && d[j] >= first_step) mine |= 1u << j;
            }
            if constexpr (PART) mine &= in;
            if (WEIGHTS && (!PART || __any_sync(0xffffffffu, in))) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const u64 o = w.weight(x[j]), v = d[j] < (float)kBins && (!PART || (in >> j & 1)) ? o : 0;      // (-inf has no weight)
                    sums[0] += v;
                    sums[1] += d[j] < since ? v : 0;
                }
            }
            if (!__any_sync(0xffffffffu, mine)) return;
            if (list) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (mine >> j & 1) put(place_of(x[j], first + i + j));
                return;
            }
            const int many = __popc(mine), lane = threadIdx.x % 32;
            int before = many;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int o = __shfl_up_sync(0xffffffffu, before, d);
                if (lane >= d) before += o;
            }
            unsigned at = 0;
            if (lane == 31) at = atomicAdd(&sh.chosen, (unsigned)before);
            at = __shfl_sync(0xffffffffu, at, 31) + before - many;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (mine >> j & 1) {
                    if (at < kChosen) wk.chosen[at] = i + j;
                    ++at;
                }
        });
        if constexpr (WEIGHTS) {
            const u64 kept = warp_sum(sums[1]);
            if (threadIdx.x % 32 == 0) sh.kept[threadIdx.x / 32] = kept;
            block_sum(sh, sums);
        } else {
            __syncthreads();
        }
        u64 said[3] = {sums[0], sums[1], sh.chosen > kChosen};
        say_sum(said);
        sums[0] = said[0];
        sums[1] = said[1];
        *fits = said[2] == 0;
    }
    // The sorted list's weights (or ones) of this thread's two places, the sum before them,
    // and the whole; those past the first `most` count nothing
    __device__ __forceinline__ u64 before_each(unsigned many, bool weights, u64 (&own)[2], u64* before, u64 most = ~0ull) {
        u64 v[1] = {0}, all[1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned a = 2 * threadIdx.x + i;
            own[i] = a < many && a < most ? (weights ? w.weight(value_at(sh.list[a])) : 1) : 0;
            v[0] += own[i];
        }
        block_scan(sh, v, all);
        *before = v[0];
        return all[0];
    }
    // Every token that `look` took: from its list, or, where that overflowed, from all
    template <typename F>
    __device__ __forceinline__ void each_chosen(bool listed, int from, int to, F f) const {
        if (listed) {
            const int many = (int)sh.chosen;
            for (int k = threadIdx.x; k < many; k += kThreads) {
                const int i = wk.chosen[k];
                f(value(to_f32(slice[i])), i);
            }
        } else {
            const float upto = (float)(to + 1), since = (float)from;
            each([&](float x, int i) {
                const float d = w.depth(x);
                if (d >= since && d < upto && before_end(x, i)) f(x, i);
            });
        }
    }
};

// Ascending, in place; every thread of the CTA.  A few by counting the smaller ones
// of each (equal ones, which are all of the largest number there is, keep their order).
constexpr unsigned kCounted = 192;
__device__ __forceinline__ void sort_list(u64* a, unsigned n) {
    if (n <= kCounted) {
        u64 mine = 0;
        unsigned at = 0;
        if (threadIdx.x < n) {
            mine = a[threadIdx.x];
            for (unsigned i = 0; i < n; ++i) at += a[i] < mine || (a[i] == mine && i < threadIdx.x);
        }
        __syncthreads();
        if (threadIdx.x < n) a[at] = mine;
        __syncthreads();
        return;
    }
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(SampleParams p, int part) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ Shared sh;
    Work& wk = *reinterpret_cast<Work*>(memory);
    constexpr int N = Vec16<T>::N;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long r = blockIdx.x / ranks;
    const int first = rank * part, n = max(0, min(p.vocab - first, part));
    const T* const row = static_cast<const T*>(p.logits) + r * p.stride + first;
    const int seg = ((part + kWarps - 1) / kWarps + 32 * N - 1) / (32 * N) * (32 * N);
    Row<T> s{cluster, sh, wk, row, first, n, seg, reinterpret_cast<uintptr_t>(row) % 16 == 0, false, false, rank, ranks, 0, ~0ull, {}};
    const float temperature = p.temperatures ? p.temperatures[r] : p.temperature, top_p = p.top_ps ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps ? p.min_ps[r] : p.min_p, u = p.u[r];
    const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const bool greedy = temperature == 0.0f;
    if (ranks > 1) cluster.barrier_arrive();

    // the largest value; NaN orders above the others
    Top<T> most;
    s.each_load([&](const Vec16<T>& v) { most.add(v); });
    if (ranks > 1) cluster.barrier_wait();                // all CTAs are there to be told
    const float mine_top = most.value();
    const u64 top_key = s.say_max(s.block_max(mine_top != mine_top ? ~0ull : (u64)key_of(mine_top)));
    const float top = value_of((uint32_t)top_key);
    const bool fine = top_key != ~0ull && top > -INFINITY && temperature >= 0.0f && temperature < INFINITY && top_p == top_p && min_p == min_p &&
                      (greedy || (u >= 0.0f && u < 1.0f));
    if (!fine || greedy) {
        u64 index = 0;                                    // the lowest that has it, inverted
        if (fine) {
            s.each([&](float x, int i) {
                if (x == top) index = max(index, (u64)~(uint32_t)(first + i));
            });
            index = s.say_max(s.block_max(index));
        }
        if (rank == 0 && threadIdx.x == 0) {
            p.tokens[r] = fine ? (int)~(uint32_t)index : -1;
            if (p.logp) p.logp[r] = fine ? 0.0f : NAN;
        }
        return;
    }
    Weigher& w = s.w;
    s.endless = top == INFINITY;
    s.tiny = !s.endless && temperature < 1e-30f && fabsf(top) < 1e9f;
    // (at that temperature, below larger values nothing has any weight)
    w.set(s.value(top), s.tiny ? temperature * 0x1p90f : fmaxf(temperature, 1e-30f), p.vocab);
    const u64 least = __double2ull_ru((double)fminf(fmaxf(min_p, 0.0f), 1.0f) * (double)(1ull << w.bits));

    const bool by_count = top_k > 0 && top_k < p.vocab, by_weight = top_p < 1.0f;
    u64 limit_k = ~0ull, limit_w = ~0ull;                 // tokens, and weight before a token, that are kept
    bool listed = false, counted = false, summed = false;
    unsigned in_list = 0;
    for (int pass = 0; pass < 2 && !listed; ++pass) {
        const bool weights = pass == 1, partly = s.end != ~0ull;
        if (weights ? !by_weight : !by_count) continue;
        if (partly) s.template histogram<true>();
        else if (!counted) s.template histogram<false>();
        counted = true;
        const auto at = s.steps_for(weights ? -1 : top_k, top_p);
        if (at.from == kBins) continue;                   // fewer tokens than k have any weight
        listed = at.upto <= kList;
        u64 sums[2];
        bool fits;
        if (!weights) s.template look<false, false>(at.from, at.to, listed, sums, &fits);
        else if (partly) s.template look<true, true>(at.from, at.to, listed, sums, &fits);
        else s.template look<false, true>(at.from, at.to, listed, sums, &fits);
        u64 want = weights ? want_of(top_p, sums[0]) : (u64)top_k;
        if (listed) {
            // few tokens up to the last step: the first CTA has them all
            (weights ? limit_w : limit_k) = want;
            in_list = s.in_list();
            break;
        }
        want -= weights ? sums[1] : at.before;
        // finer parts of the steps, then of the (value, index), until few tokens are left
        u64 in = at.upto - at.before, lo = 0, hi = s.end;
        const float since = (float)at.from, parts = (float)kBins / (float)(at.to + 1 - at.from);
        float low_part = 0.0f, high_part = INFINITY;
        auto part_of = [&](auto f) {
            s.each_chosen(fits, at.from, at.to, [&](float x, int i) {
                const float q = (w.depth(x) - since) * parts;
                const u64 place = place_of(x, first + i);
                if (q >= low_part && q < high_part && place >= lo && place <= hi) f(x, q, place);
            });
        };
        for (int round = 0; round < 8 && in > kList; ++round) {          // 2^11 parts each: 64 bits are through before
            int shift = 0;
            if (round) {
                u64 low = 0, high = 0;                    // the first (inverted) and last place in the range
                part_of([&](float, float, u64 place) {
                    low = max(low, ~place);
                    high = max(high, place);
                });
                lo = ~s.say_max(s.block_max(low));
                hi = s.say_max(s.block_max(high));
                shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
            }
            s.clear();
            part_of([&](float x, float q, u64 place) { s.count(round ? (int)((place - lo) >> shift) : min((int)q, kBins - 1), x, weights); });
            const auto found = s.cross(want, weights);
            want -= weights ? found.weight : found.count;
            in = found.in;
            if (round) {
                lo += (u64)found.bin << shift;
                hi = min(hi, lo + ((1ull << shift) - 1));
            } else {
                low_part = (float)found.bin;
                high_part = found.bin == kBins - 1 ? INFINITY : (float)(found.bin + 1);
            }
        }
        if (threadIdx.x == 0) sh.listed = 0;
        s.together();
        part_of([&](float, float, u64 place) { s.put(place); });
        s.together();
        if (rank == 0) {
            const unsigned few = s.in_list();
            sort_list(sh.list, few);
            // the last one with less than `want` before it
            u64 own[2], before = 0;
            s.before_each(few, weights, own, &before);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned a = 2 * threadIdx.x + i;
                if (a < few && before < want && (before + own[i] >= want || a + 1 == few)) sh.last = sh.list[a];
                before += own[i];
            }
        }
        s.together();
        s.end = *cluster.map_shared_rank(&sh.last, 0);
        s.together();
        if (weights && !least) {
            // what the steps' tokens add to each warp's part
            s.each_chosen(fits, at.from, at.to, [&](float x, int i) {
                if (s.before_end(x, i)) atomicAdd(&sh.kept[i / seg], w.weight(x));
            });
            __syncthreads();
            summed = true;
        }
    }

    const double share = u;
    bool whole;
    if (listed) {
        if (rank == 0) {
            const unsigned a = 2 * threadIdx.x;
            sort_list(sh.list, in_list);
            u64 own[2], before, kept[2], all[1] = {0};
            u64 sum = s.before_each(in_list, true, own, &before, limit_k);
            if (by_weight && limit_w == ~0ull) limit_w = want_of(top_p, sum);
            u64 place[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                place[i] = a + i < in_list ? sh.list[a + i] : ~0ull;
                kept[i] = before < limit_w && own[i] >= least ? own[i] : 0;
                before += own[i];
            }
            all[0] = kept[0] + kept[1];
            block_sum(sh, all);
            const u64 target = share_of(share, all[0], &whole);
            // the kept ones again, in the vocabulary's order
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (a + i < in_list) sh.list[a + i] = kept[i] ? place[i] << 32 | place[i] >> 32 : ~0ull;
            __syncthreads();
            sort_list(sh.list, in_list);
            u64 turned[2], v[1] = {0};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                turned[i] = a + i < in_list ? sh.list[a + i] : ~0ull;
                own[i] = turned[i] != ~0ull ? w.weight(value_of(~(uint32_t)turned[i])) : 0;
                v[0] += own[i];
            }
            block_scan(sh, v, all);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (v[0] <= target && target < v[0] + own[i]) {
                    p.tokens[r] = (int)(turned[i] >> 32);
                    if (p.logp) p.logp[r] = (float)log((double)own[i] / (double)all[0]);
                }
                v[0] += own[i];
            }
        }
        return;
    }

    // everything up to the last: each warp's sum, each CTA's, the whole; then the part of the
    // warp in which the sum passes the target once more
    const float last_value = s.end == ~0ull ? -INFINITY : value_at(s.end);
    const int last_index = s.end == ~0ull ? INT_MIN : (int)((uint32_t)s.end - (uint32_t)first);
    auto weigh = [&](const float* x, int i, u64* v) {
        unsigned kept = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) kept |= (x[j] > last_value || (x[j] == last_value && i + j <= last_index)) ? 1u << j : 0u;
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0;
        if (__any_sync(0xffffffffu, kept)) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const u64 o = w.weight(x[j]);
                v[j] = (kept >> j & 1) && o >= least ? o : 0;
                sum += v[j];
            }
        }
        return sum;
    };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (!summed) {
        u64 mine = 0;
        s.each_vector([&](const float* x, int i) {
            u64 v[N];
            mine += weigh(x, i, v);
        });
        mine = warp_sum(mine);
        __syncthreads();
        if (lane == 0) sh.kept[warp] = mine;
        __syncthreads();
    }
    const u64 own = lane < kWarps ? sh.kept[lane] : 0, upto = warp_scan(own);   // each warp has them all
    u64 sum[1] = {__shfl_sync(0xffffffffu, upto, 31)};
    const u64 here = sum[0], below = s.say_sum(sum), target = share_of(share, sum[0], &whole);
    if (target < below || target >= below + here) return;
    // the part in which the target lies, by all warps
    const int of = __popc(__ballot_sync(0xffffffffu, below + upto <= target));
    u64 before = below + __shfl_sync(0xffffffffu, upto - own, of);
    const int from = of * seg, to = min(n, from + seg);
    for (int i0 = from; i0 < to; i0 += kThreads * N) {
        const int i = i0 + (int)threadIdx.x * N;
        u64 v[N] = {}, part_sum[1] = {0}, all[1];
        if (i0 + warp * 32 * N < to) {                    // whole warps
            float x[N];
            s.values(s.load(i), x);
            part_sum[0] = weigh(x, i, v);
        }
        block_scan(sh, part_sum, all);
        u64 place = before + part_sum[0];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (place <= target && target < place + v[j]) {
                p.tokens[r] = first + i + j;
                if (p.logp) p.logp[r] = (float)log((double)v[j] / (double)sum[0]);
            }
            place += v[j];
        }
        before += all[0];
    }
}

// CTAs a row: one, as long as the rows alone put two on every SM or the parts get
// small, and as many as keep a part's tokens within what the histograms count.
template <typename T>
cudaError_t sample_launch(const SampleParams& p, cudaStream_t s) {
    constexpr int N = Vec16<T>::N, kMostPart = 1 << 17, kLeastPart = 4096;
    auto part_of = [&](int ranks) { return ((p.vocab + ranks - 1) / ranks + N - 1) / N * N; };
    int ranks = 1;
    while (part_of(ranks) > kMostPart || (ranks < 8 && p.rows * ranks * 2 <= 2 * kSmCount && part_of(ranks * 2) >= kLeastPart)) ranks *= 2;
    const cudaError_t e = allow_shared<k_sample<T>>((int)sizeof(Work));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Work);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_sample<T>, p, part_of(ranks));
}

}  // namespace

cudaError_t launch_sample(const SampleParams& p, cudaStream_t s) {
    if (p.type == VDT_F32) return sample_launch<float>(p, s);
    if (p.type == VDT_F16) return sample_launch<__half>(p, s);
    return sample_launch<__nv_bfloat16>(p, s);
}

}  // namespace vdt

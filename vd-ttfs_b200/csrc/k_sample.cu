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
// whole numbers, w * 2^44 (2^43 for vocabularies above 2^18), from a table of roots
// and a polynomial in 64 bits: sums are exact, the same in any order.  A weight is rounded
// by up to half a step, the sum of n of them by up to n / 2, and a share of it by as much, so
// an answer can differ from the real numbers' one where u or top_p come within n steps of a
// border: 2^-27 of the sum for 2^17 tokens, 2^-24 for 2^19.  It takes a tail whose weights all
// round the same way (45.2 octaves down they count nothing); of others root n steps remain, 2^-35.
//
// One CTA takes a row, or a cluster of them where rows are few, and reads it
// from L2 for each pass.  A histogram of the tokens over 2048 steps of log2(w), 44 an
// octave, gives the step of the token number k, and an estimate of the few steps
// in which the last token for p lies: a step's weights are within a 44th of an
// octave of its middle.  One pass then sums all weights and those before these
// steps, and lists the steps' tokens.  The sums say whether the estimate holds; where
// it does not, the same again with the bounds of the steps' weights, which do.  The
// listed tokens are told apart by finer histograms while there are many of them,
// and sorted in the end.  Where no more than kList tokens come up to there, one CTA sorts
// them all and finishes; else all CTAs sum what is kept, and the part of the warp in
// which the sum passes the target is gone through again.
//
// Bound by instructions, some 100 a token with top_p in three passes, and by 64
// registers a thread, with which two CTAs share an SM so that one computes while
// the other waits for a barrier (one CTA with 128: each row is faster, all of them
// slower).  us, replayed: 250 x 100003 f32, top_p, 137, against 15 for reading the
// logits once; 64 x 131072 bf16, mixed parameters, 62; one row of 32768 16.5, which
// are some ten exchanges in the cluster and code that runs once.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "step_internal.h"

namespace vdt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kRoom = kBins + 4, kList = 1024, kChosen = 512;
constexpr float kSteps = 44.0f;              // of an octave; kBins of them are 46.5 octaves, below which weights round to 0
constexpr int kMostBits = 44, kBoundBits = 40;
constexpr int kMostPart = 1 << 17;           // tokens of a CTA

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
// Eight values side by side, on a multiple of their size
template <typename T>
struct Eight {
    static constexpr int kWords = 2 * sizeof(T);
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* from) {
        if constexpr (sizeof(T) == 4) {
            asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                : "l"(from));
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(from));
            w[0] = v.x;
            w[1] = v.y;
            w[2] = v.z;
            w[3] = v.w;
        }
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(w[i]);
            else unpack2<T>(w[i], f[2 * i], f[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void set(const float* f) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
            else w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
    }
};
// the largest of many values; NaN where one is
template <typename T>
struct Top {
    using Pair = std::conditional_t<sizeof(T) == 4, float, std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>>;
    Pair a;
    __device__ __forceinline__ Top() {
        const uint32_t lowest = sizeof(T) == 4 || std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u : 0xfc00fc00u;
        if constexpr (sizeof(T) == 4) a = -INFINITY;
        else memcpy(&a, &lowest, 4);
    }
    __device__ __forceinline__ void add(const Eight<T>& v) {
#pragma unroll
        for (int i = 0; i < Eight<T>::kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                a = max_or_nan(a, __uint_as_float(v.w[i]));
            } else {
                Pair b;
                memcpy(&b, &v.w[i], 4);
                a = __hmax2_nan(a, b);
            }
        }
    }
    __device__ __forceinline__ float value() const {
        if constexpr (sizeof(T) == 4) return a;
        else return max_or_nan(__low2float(a), __high2float(a));
    }
};

// 2^(i / 32)
__device__ const double kRoots[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

struct Weigher {
    // How a row's values are taken.  As they are, mostly; `alone`: the largest as 0, all
    // others as -inf, where it is +inf or the next value below it has no weight; `shift`: less
    // the largest, where that is many temperatures (what has any weight is near to
    // it then, and the difference exact); times `factor`, a power of two, for the smallest temperatures
    bool odd, alone, shift;
    float largest, factor;
    float top, bottom;      // the largest then, and a value without weight (-inf is not weighed)
    float slope, start;     // steps of the histogram below the largest: start + slope x
    double parts;           // 32 log2(e) / T
    const double* roots;    // kRoots times 2^bits, in shared memory
    int bits;
    static __device__ __forceinline__ int bits_of(int vocab) { return min(kMostBits, 62 - (32 - __clz(vocab - 1))); }
    __device__ __forceinline__ float value(float x) const {
        return alone ? (x == largest ? 0.0f : -INFINITY) : (shift ? x - largest : x) * factor;
    }
    __device__ __forceinline__ void set(float row_top, float temperature, int vocab) {
        constexpr double kLog2e = 1.4426950408889634;
        largest = row_top;
        float below = value_of(key_of(largest) - 1);             // the next value below (0's is not -0)
        if (below == largest) below = value_of(key_of(largest) - 2);
        const double octaves = kLog2e / (double)temperature, far = fabs((double)largest) * octaves * (double)kSteps;
        alone = largest == INFINITY || ((double)largest - (double)below) * octaves > 60.0;
        shift = !alone && far > 1e4;
        factor = !alone && temperature < 1e-30f ? 0x1p90f : 1.0f;
        odd = alone || shift || factor != 1.0f;
        top = value(largest);
        const double each = alone ? 1.0 : octaves / (double)factor;
        parts = 32.0 * each;
        bottom = fmaxf(__double2float_rd((double)top - 80.0 / each), -FLT_MAX);
        slope = (float)(-(double)kSteps * each);
        // a little above, so that the largest is not below 0
        start = (float)((double)kSteps * each * (double)top) + (float)(shift || alone ? 0.0 : far) * 0x1p-22f;
        bits = bits_of(vocab);
    }
    // the logarithm of a token's probability, from the kept weights' sum (1 for the largest)
    __device__ __forceinline__ double log_sum(u64 sum) const { return log((double)sum * __hiloint2double((1023 - bits) << 20, 0)); }
    __device__ __forceinline__ float log_share(float x, double log_sum) const {
        return (float)(((double)x - (double)top) * parts * (0.6931471805599453 / 32.0) - log_sum);
    }
    __device__ __forceinline__ float depth(float x) const { return fmaf(slope, x, start); }
    // the step itself, kBins for all without weight: floor in the low bits of 2^23 + depth
    static __device__ __forceinline__ int step(float depth) {
        return __float_as_int(__fadd_rd(fminf(depth, (float)kBins), 8388608.0f)) & (2 * kBins - 1);
    }
    // 2^bits exp((x - top) / T) to the nearest whole number, and 2^52: the next 32nd of an
    // octave from a table, its exponent moved by the whole octaves, and the rest, at most a
    // 64th, by the interpolating polynomial of degree 4 at Chebyshev's points, off by at most
    // 2^-43.  (Without the table degree 8 is wanted: 14 operations in 64 bits a token, of
    // which the SM does 1.6 a cycle for a warp, and not 9.)  3/2 2^52 added leaves the nearest
    // whole number in the low bits; no branches, so that the chains of several tokens run side by side.
    __device__ __forceinline__ double raised(float x) const {
        constexpr double kRound = 6755399441055744.0;
        const double d = (double)fmaxf(x, bottom) - (double)top;
        const double z = fma(d, parts, kRound), f = fma(d, parts, kRound - z);
        const unsigned whole = (unsigned)__double2loint(z);
        const double root = roots[whole & 31];
        double y = 0x1.3b2b18fa66654p-27;
        y = fma(y, f, 0x1.c6b167e61eadap-20);
        y = fma(y, f, 0x1.ebfbdff817570p-13);
        y = fma(y, f, 0x1.62e42fef6d03fp-6);
        y = fma(y, f, 1.0);
        return fma(y, __hiloint2double((int)((unsigned)__double2hiint(root) + ((whole & ~31u) << 15)), __double2loint(root)), 4503599627370496.0);
    }
    // as 64-bit floating point, sums of which are exact up to 2^53: 2^9 of the largest
    __device__ __forceinline__ double weight_f(float x) const { return raised(x) - 4503599627370496.0; }
    __device__ __forceinline__ u64 weight(float x) const { return (u64)__double_as_longlong(raised(x)) & 0xfffffffffffffull; }
};

// A histogram, weights in three parts of 15 bits (a CTA's sums of each stay below
// 2^32; the row's first histogram, of counts alone, has four copies there, each
// for a quarter of the lanes: tokens of 16 bits have few values, and lanes with the
// same one wait for each other), and the tokens of the steps that are looked into
struct Work {
    uint32_t count[4][kRoom];                // (kBins: tokens without weight; later counts, and the weights' parts)
    u64 chosen[kWarps][kChosen];             // each warp its own
};
struct Shared {
    u64 list[kList];
    u64 said[2][8][4];                       // what the CTAs tell each other, two exchanges in turn
    u64 warps[3][kWarps];
    u64 found[4];
    u64 kept[kWarps];                        // weight of what each warp's part keeps
    u64 last;
    double roots[32], log_sum;
    unsigned listed, chosen[kWarps];
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
__device__ __forceinline__ float warp_scan(float v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const float o = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)(threadIdx.x % 32) >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)(threadIdx.x % 32) >= d) v += o;
    }
    return v;
}
// the same for a count and a weight, and the sum of a third (its bits in `all`)
__device__ __forceinline__ void block_scan(Shared& sh, uint32_t& count, u64& weight, float square, u64 (&all)[3]) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t own = count, c = warp_scan(count);
    const u64 mine = weight, w = warp_scan(weight);
    const float q = warp_scan(square);
    __syncthreads();
    if (lane == 31) {
        sh.warps[0][warp] = c;
        sh.warps[1][warp] = w;
        sh.warps[2][warp] = __float_as_uint(q);
    }
    __syncthreads();
    const bool in = lane < kWarps;
    const uint32_t n = in ? (uint32_t)sh.warps[0][lane] : 0, n_upto = warp_scan(n);
    const u64 o = in ? sh.warps[1][lane] : 0, o_upto = warp_scan(o);
    const float q_upto = warp_scan(in ? __uint_as_float((uint32_t)sh.warps[2][lane]) : 0.0f);
    all[0] = __shfl_sync(0xffffffffu, n_upto, 31);
    all[1] = __shfl_sync(0xffffffffu, o_upto, 31);
    all[2] = __float_as_uint(__shfl_sync(0xffffffffu, q_upto, 31));
    count = c - own + __shfl_sync(0xffffffffu, n_upto - n, warp);
    weight = w - mine + __shfl_sync(0xffffffffu, o_upto - o, warp);
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
    static constexpr int N = 8;
    cg::cluster_group cluster;
    Shared& sh;
    Work& wk;
    const T* slice;          // this CTA's part, on whole vectors: the row's may begin up to N - 1 values before it does
    int first, n, seg;       // its first index (below 0 then), its length, and what a warp takes of it
    int rank, ranks, turn;
    u64 end;                 // the last token's place that counts, as far as it is known
    float end_value;
    int end_index;
    Weigher w;

    __device__ __forceinline__ void together() const {
        if (ranks > 1) cluster.sync();
        else __syncthreads();
    }
    // What each CTA has to say, to all of them
    template <int K>
    __device__ __forceinline__ u64 (&say(const u64 (&mine)[K]))[8][4] {
        u64 (&slots)[8][4] = sh.said[turn];
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

    // N values; what is not the part's counts as -inf
    __device__ __forceinline__ Eight<T> load(int i, bool edge) const {
        Eight<T> v;
        if (!edge) {
            v.load(slice + i);
        } else {
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = i + j < n && first + i + j >= 0 ? to_f32(slice[i + j]) : -INFINITY;
            v.set(x);
        }
        return v;
    }
    // whether some of a warp's vectors from i0 on are not the part's
    __device__ __forceinline__ bool edge_at(int i0) const { return i0 + 32 * N > n || (first < 0 && i0 == 0); }
    __device__ __forceinline__ void values(const Eight<T>& v, float* x) const {
        v.get(x);
        if (w.odd)
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = w.value(x[j]);
    }
    // Every N tokens of this thread: a warp's are consecutive, a lane's N of them too;
    // the next are on their way meanwhile
    template <typename F>
    __device__ __forceinline__ void each_vector(F f) const {
        const int from = threadIdx.x / 32 * seg, to = min(n, from + seg), step = 32 * N;
        if (from >= to) return;
        int i = from + (int)(threadIdx.x % 32) * N;
        Eight<T> next = load(i, edge_at(from));
        for (int i0 = from; i0 < to; i0 += step, i += step) {
            const Eight<T> v = next;
            if (i0 + step < to) next = load(i + step, edge_at(i0 + step));
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
        for (int i0 = from; i0 < to; i0 += 32 * N) f(load(i0 + (int)(threadIdx.x % 32) * N, edge_at(i0)));
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
    __device__ __forceinline__ void end_at(u64 place) {
        end = place;
        end_value = value_at(place);
        end_index = (int)((uint32_t)place - (uint32_t)first);
    }
    __device__ __forceinline__ bool before_end(float x, int i) const { return x > end_value || (x == end_value && i <= end_index); }
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

    // The steps of the row's histogram in which the last kept token lies, for the count
    // k (k >= 0), or else for the share top_p of the weight.  A step's weight is its
    // tokens' number times that of its middle, which each of them is off by at most a
    // factor h = 2^(1/88).  `sure`: steps that the bounds allow; else by the errors' size,
    // 0.46% (the spread over a step) of each step's weight, four times the root of the
    // sum of their squares.
    struct Steps {
        int from, to;               // from == kBins: there is no such token
        u64 before, upto;           // tokens before `from`, and up to `to`
    };
    __device__ __forceinline__ void gather_counts() {
        constexpr int kPer = kBins / kThreads;
        static_assert(kPer == 4, "four steps a thread");
        __syncthreads();
        uint4 sum = reinterpret_cast<const uint4*>(&wk.count[0][0])[threadIdx.x];
#pragma unroll
        for (int k = 1; k < 4; ++k) {
            const uint4 o = reinterpret_cast<const uint4*>(&wk.count[k][0])[threadIdx.x];
            sum = make_uint4(sum.x + o.x, sum.y + o.y, sum.z + o.z, sum.w + o.w);
        }
        reinterpret_cast<uint4*>(&wk.count[0][0])[threadIdx.x] = sum;
        together();                                           // all histograms are there
    }
    __device__ __forceinline__ Steps steps_for(int k, float top_p, bool sure) {
        constexpr int kPer = kBins / kThreads;
        const int mine = kBins / ranks, per = (mine + kThreads - 1) / kThreads;      // this CTA's steps; a thread's, consecutive
        const int from = rank * mine + threadIdx.x * per;
        uint32_t c[kPer] = {}, count = 0;
        u64 w[kPer] = {}, weight = 0;
        float square = 0.0f;
        if (ranks == 1) {
            const uint4 o = reinterpret_cast<const uint4*>(&wk.count[0][0])[threadIdx.x];
            c[0] = o.x;
            c[1] = o.y;
            c[2] = o.z;
            c[3] = o.w;
        } else if ((int)threadIdx.x * per < mine) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= ranks) continue;
                const uint32_t* const o = &cluster.map_shared_rank(&wk, r)->count[0][from];
                c[0] += o[0];
                if (per == 2) c[1] += o[1];
            }
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) count += c[i];
        if (k < 0) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float each = exp2f((float)kBoundBits - (from + i + 0.5f) / kSteps);
                w[i] = c[i] * (u64)each;
                weight += w[i];
                square += (float)w[i] * (float)w[i];
            }
        }
        u64 all[3];
        if (k < 0) {
            block_scan(sh, count, weight, square, all);
        } else {
            u64 v[1] = {count}, sum[1];
            block_scan(sh, v, sum);
            count = (uint32_t)v[0];
            all[0] = sum[0];
            all[1] = all[2] = 0;
        }
        if (threadIdx.x == 0) {
            sh.found[0] = sh.found[1] = kBins;
        }
        const auto& slots = say(all);
        float squares = 0.0f;
        u64 tokens = 0, total = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r < rank) {
                count += (uint32_t)slots[r][0];
                weight += slots[r][1];
            }
            tokens += slots[r][0];
            total += slots[r][1];
            squares += __uint_as_float((uint32_t)slots[r][2]);
        }
        // (from here on the other CTAs may write to `found`)
        // the first step up to which there may be enough, and the first up to which there is
        // (the last, where that is nearly all); 2^(1/44), and room for the 32-bit depths and sums
        u64 least = 0, most = 0;
        if (k < 0) {
            const float whole = (float)total, share = fmaxf(top_p, 0.0f) * whole, wide = 1.0159f * 1.0002f;
            float lower = share / wide, upper = share * wide;
            if (!sure) {
                const float off = 4.0f * 0.0046f * sqrtf(squares) + 1e-5f * whole;
                lower = fmaxf(lower, share - off);
                upper = fminf(upper, share + off);
            }
            least = max((u64)fmaxf(lower, 0.0f), 1ull);
            most = upper > whole * 0.9999f ? ~0ull : max((u64)upper, 1ull);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const bool here = k >= 0 ? count < (uint32_t)k && (uint32_t)k <= count + c[i] : weight < least && least <= weight + w[i];
            const bool there = k >= 0 ? here : weight < most && most <= weight + w[i];
            if (here || there)
                for (int r = 0; r < ranks; ++r) {
                    u64* const f = cluster.map_shared_rank(sh.found, r);
                    if (here) {
                        f[0] = from + i;
                        f[2] = count;
                    }
                    if (there) {
                        f[1] = from + i;
                        f[3] = count + c[i];
                    }
                }
            count += c[i];
            weight += w[i];
        }
        together();
        const bool open = sh.found[1] == kBins;               // no step reaches so far: all of them
        const Steps found{(int)sh.found[0], open ? kBins - 1 : (int)sh.found[1], sh.found[2], open ? tokens : sh.found[3]};
        __syncthreads();
        return found;
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
#pragma unroll 4
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

    // a token into the first CTA's list, from some of a warp's lanes: one of them counts for all
    __device__ __forceinline__ void put(u64 place) {
        const unsigned who = __activemask(), below = __popc(who & ((1u << threadIdx.x % 32) - 1));
        unsigned at = 0;
        if (!below) at = atomicAdd(cluster.map_shared_rank(&sh.listed, 0), (unsigned)__popc(who));
        at = __shfl_sync(who, at, __ffs(who) - 1) + below;
        if (at < kList) cluster.map_shared_rank(sh.list, 0)[at] = place;
    }
    // its length, for the first CTA alone: the others may go on after that one has ended
    __device__ __forceinline__ unsigned in_list() const { return rank == 0 ? min(sh.listed, (unsigned)kList) : 0; }

    // One pass over the row's tokens (PART: up to the place `end`): with WEIGHTS the
    // sums of their weights, of those in steps before `from`, each warp's into `kept`, and of those
    // in steps up to `to`; and the tokens of the steps first..to into `chosen`, as far as each warp
    // has room for its own (`fits`: all have), `before`: how many the CTAs of lower rank have.
    template <bool PART, bool WEIGHTS>
    __device__ __forceinline__ void look(int from, int to, int first_of, u64 (&sums)[3], bool* fits, unsigned* before) {
        unsigned have = 0;
        static_assert(kMostPart / kThreads + N <= 1 << (53 - kMostBits), "a thread's sums are exact in 64-bit floating point");
        double all = 0.0, head = 0.0;
        const float since = (float)from, upto = (float)(to + 1), first_step = (float)first_of;
        const int lane = threadIdx.x % 32;
        each_vector([&](const float* x, int i) {
            unsigned mine = 0, in = 0;
            if constexpr (PART) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (before_end(x[j], i + j)) in |= 1u << j;
                if (!__any_sync(0xffffffffu, in)) return;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = w.depth(x[j]);
                const bool here = !PART || (in >> j & 1);
                if (WEIGHTS) {
                    const double v = w.weight_f(x[j]);
                    if (here && d < (float)kBins) all += v;          // (not -inf)
                    if (here && d < since) head += v;
                }
                mine |= (unsigned)(here && d < upto && d >= first_step) << j;
            }
            // one of each lane's at a time, hardly ever more than two
            for (unsigned who; (who = __ballot_sync(0xffffffffu, mine != 0)) != 0; mine &= mine - 1) {
                const int j = __ffs(mine) - 1;
                float y = x[0];
#pragma unroll
                for (int k = 1; k < N; ++k) y = j == k ? x[k] : y;
                const unsigned at = have + __popc(who & ((1u << lane) - 1));
                if (mine && at < kChosen) wk.chosen[threadIdx.x / 32][at] = place_of(y, first + i + j);
                have += __popc(who);
            }
        });
        sums[0] = (u64)all;
        sums[1] = (u64)head;
        sums[2] = 0;
        if constexpr (WEIGHTS) {
            // up to `to`: the ones before `from` and the chosen, where these do not begin at the largest
            if (first_of) sums[2] = sums[1];
            __syncwarp();
            if (have <= kChosen) {
                for (unsigned k = lane; k < have; k += 32) sums[2] += w.weight(value_at(wk.chosen[threadIdx.x / 32][k]));
            } else {
                each([&](float x, int i) {
                    const float d = w.depth(x);
                    if (d < upto && d >= first_step && (!PART || before_end(x, i))) sums[2] += w.weight(x);
                });
            }
        }
        if (lane == 0) sh.chosen[threadIdx.x / 32] = have;
        u64 said[4] = {0, 0, 0, 0}, many[1] = {lane == 0 ? have + (have > kChosen ? 1ull << 40 : 0) : 0};
        if constexpr (WEIGHTS) {
            const u64 kept = warp_sum(sums[1]);
            if (lane == 0) sh.kept[threadIdx.x / 32] = kept;
            block_sum(sh, sums);
            said[0] = sums[0];
            said[1] = sums[1];
            said[2] = sums[2];
        }
        block_sum(sh, many);
        said[3] = many[0];
        const auto& slots = say(said);
        sums[0] = sums[1] = sums[2] = 0;
        u64 listed = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r == rank) *before = (unsigned)listed;
#pragma unroll
            for (int k = 0; k < 3; ++k) sums[k] += slots[r][k];
            listed += slots[r][3];
        }
        *fits = listed >> 40 == 0;
    }
    // What `look` listed, at most kList tokens, into the first CTA's list
    __device__ __forceinline__ void send(bool fits, int from, int to, unsigned before) {
        if (fits) {
            const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, many = (int)sh.chosen[warp];
            for (int i = 0; i < warp; ++i) before += sh.chosen[i];
            u64* const list = cluster.map_shared_rank(sh.list, 0);
            for (int k = lane; k < many; k += 32)
                if (before + k < kList) list[before + k] = wk.chosen[warp][k];
        } else {
            if (threadIdx.x == 0) sh.listed = 0;
            together();
            each_chosen(false, from, to, [&](float, u64 place) { put(place); });
        }
        together();
    }

    // Each warp's sum of the weights up to `end` of at least `least`, into `kept`
    __device__ __forceinline__ void sum_kept(u64 least) {
        const double least_f = (double)least;
        double sum = 0.0;
        each_vector([&](const float* x, int i) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double o = w.weight_f(x[j]);
                if (before_end(x[j], i + j) && o >= least_f) sum += o;
            }
        });
        const u64 mine = warp_sum((u64)sum);
        __syncthreads();
        if (threadIdx.x % 32 == 0) sh.kept[threadIdx.x / 32] = mine;
        __syncthreads();
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
            const int warp = threadIdx.x / 32, many = (int)sh.chosen[warp];
            for (int k = threadIdx.x % 32; k < many; k += 32) {
                const u64 place = wk.chosen[warp][k];
                f(value_at(place), place);
            }
        } else {
            const float upto = (float)(to + 1), since = (float)from;
            each([&](float x, int i) {
                const float d = w.depth(x);
                if (d >= since && d < upto && before_end(x, i)) f(x, place_of(x, first + i));
            });
        }
    }
};

// Ascending, in place; every thread of the CTA.  A few by counting the smaller ones of
// each (equal ones, which are all of the largest number there is, keep their order); more
// in a bitonic network, two neighbours a thread.  Partners up
// to 63 places apart are in the same warp and meet in registers, the others in shared
// memory (all steps there took four times as long).
constexpr unsigned kCounted = 128;
__device__ __noinline__ void sort_list(u64* a, unsigned n) {
    static_assert(kList == 2 * kThreads, "two a thread");
    const unsigned t = threadIdx.x;
    if (n <= kCounted) {
        u64 mine = 0;
        unsigned at = 0;
        if (t < n) {
            mine = a[t];
#pragma unroll 8
            for (unsigned i = 0; i < n; ++i) {
                const u64 o = a[i];
                at += o < mine || (o == mine && i < t);
            }
        }
        __syncthreads();
        if (t < n) a[at] = mine;
        __syncthreads();
        return;
    }
    u64 x = 2 * t < n ? a[2 * t] : ~0ull, y = 2 * t + 1 < n ? a[2 * t + 1] : ~0ull;
    unsigned size = 64;
    while (size < n) size *= 2;
    for (unsigned run = 2; run <= size; run *= 2) {
        const bool up = (2 * t & run) == 0;
        for (unsigned gap = run / 2; gap >= 2; gap /= 2) {
            u64 ox, oy;
            if (gap < 64) {
                if (2 * t >= size) break;                     // whole warps
                ox = __shfl_xor_sync(0xffffffffu, x, gap / 2);
                oy = __shfl_xor_sync(0xffffffffu, y, gap / 2);
            } else {
                __syncthreads();
                a[2 * t] = x;
                a[2 * t + 1] = y;
                __syncthreads();
                ox = a[2 * t ^ gap];
                oy = a[(2 * t ^ gap) + 1];
            }
            const bool smaller = ((2 * t & gap) == 0) == up;
            x = (x < ox) == smaller ? x : ox;
            y = (y < oy) == smaller ? y : oy;
        }
        if ((x > y) == up) {
            const u64 o = x;
            x = y;
            y = o;
        }
    }
    __syncthreads();
    if (2 * t < size) {
        a[2 * t] = x;
        a[2 * t + 1] = y;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(SampleParams p, int part) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ Shared sh;
    Work& wk = *reinterpret_cast<Work*>(memory);
    constexpr int N = Row<T>::N;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long r = blockIdx.x / ranks;
    const T* const row = static_cast<const T*>(p.logits) + r * p.stride;
    const int first = rank * part - (int)(reinterpret_cast<uintptr_t>(row) % (N * sizeof(T)) / sizeof(T)), n = max(0, min(p.vocab - first, part));
    const int seg = ((part + kWarps - 1) / kWarps + 32 * N - 1) / (32 * N) * (32 * N);
    Row<T> s{cluster, sh, wk, row + first, first, n, seg, rank, ranks, 0, ~0ull, -INFINITY, INT_MIN, {}};
    const float temperature = p.temperatures ? p.temperatures[r] : p.temperature, top_p = p.top_ps ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps ? p.min_ps[r] : p.min_p, u = p.u[r];
    const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const bool greedy = temperature == 0.0f;
    if (ranks > 1) cluster.barrier_arrive();

    if (threadIdx.x < 32) sh.roots[threadIdx.x] = kRoots[threadIdx.x] * (double)(1ull << Weigher::bits_of(p.vocab));
    // the largest value; NaN orders above the others
    Top<T> most;
    s.each_load([&](const Eight<T>& v) { most.add(v); });
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
    w.set(top, temperature, p.vocab);
    w.roots = sh.roots;
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
        if (partly || !counted) s.gather_counts();
        counted = true;
        typename Row<T>::Steps at;
        u64 sums[3], want = (u64)top_k;
        bool fits;
        unsigned before = 0;
        for (int sure = 0; sure < 2; ++sure) {
            at = s.steps_for(weights ? -1 : top_k, top_p, sure != 0);
            if (at.from == kBins) break;
            listed = at.upto <= kList;
            const int first_of = listed ? 0 : at.from;
            if (!weights) s.template look<false, false>(at.from, at.to, first_of, sums, &fits, &before);
            else if (partly) s.template look<true, true>(at.from, at.to, first_of, sums, &fits, &before);
            else s.template look<false, true>(at.from, at.to, first_of, sums, &fits, &before);
            if (!weights) break;
            want = want_of(top_p, sums[0]);
            if (sums[1] < want && want <= sums[2]) break;
        }
        if (at.from == kBins) continue;                   // fewer tokens than k have any weight
        if (listed) {
            // few tokens up to the last step: the first CTA has them all
            s.send(fits, 0, at.to, before);
            (weights ? limit_w : limit_k) = want;
            in_list = (unsigned)at.upto;
            break;
        }
        want -= weights ? sums[1] : at.before;
        // finer parts of the steps, then of the (value, index), until few tokens are left
        u64 in = at.upto - at.before, lo = 0, hi = s.end;
        const float since = (float)at.from, parts = (float)kBins / (float)(at.to + 1 - at.from);
        float low_part = 0.0f, high_part = INFINITY;
        auto part_of = [&](auto f) {
            s.each_chosen(fits, at.from, at.to, [&](float x, u64 place) {
                const float q = (w.depth(x) - since) * parts;
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
        s.end_at(*cluster.map_shared_rank(&sh.last, 0));
        s.together();
        if (!weights && top_k <= kList) {
            s.template look<true, false>(0, kBins - 1, 0, sums, &fits, &before);
            s.send(fits, 0, kBins - 1, before);
            limit_k = (u64)top_k;
            in_list = (unsigned)top_k;
            listed = true;
        }
        if (weights && !least) {
            // what the steps' tokens add to each warp's part, which are its own
            u64 mine = 0;
            s.each_chosen(fits, at.from, at.to, [&](float x, u64 place) {
                if (place <= s.end) mine += w.weight(x);
            });
            mine = warp_sum(mine);
            if (threadIdx.x % 32 == 0) sh.kept[threadIdx.x / 32] += mine;
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
            if (threadIdx.x == kThreads - 1) sh.log_sum = p.logp ? w.log_sum(all[0]) : 0.0;      // while the others sort
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
                    if (p.logp) p.logp[r] = w.log_share(value_of(~(uint32_t)turned[i]), sh.log_sum);
                }
                v[0] += own[i];
            }
        }
        return;
    }

    // everything up to the last: each warp's sum, each CTA's, the whole; then the part of the
    // warp in which the sum passes the target once more
    auto weigh = [&](const float* x, int i, bool in, u64* v) {
        unsigned kept = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) kept |= in && s.before_end(x[j], i + j) ? 1u << j : 0u;
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
    const int lane = threadIdx.x % 32;
    if (!summed) s.sum_kept(least);
    const u64 own = lane < kWarps ? sh.kept[lane] : 0, upto = warp_scan(own);   // each warp has them all
    u64 sum[1] = {__shfl_sync(0xffffffffu, upto, 31)};
    const u64 here = sum[0], below = s.say_sum(sum), target = share_of(share, sum[0], &whole);
    if (target < below || target >= below + here) return;
    // the part in which the target lies, by all warps, some consecutive vectors a thread;
    // then the thread in whose vectors it lies
    const int of = __popc(__ballot_sync(0xffffffffu, below + upto <= target));
    const u64 before = below + __shfl_sync(0xffffffffu, upto - own, of);
    const int from = of * seg, to = min(n, from + seg), many = ((to - from + N - 1) / N + kThreads - 1) / kThreads;
    u64 place[1] = {0}, all[1], v[N];
    for (int k = 0; k < many; ++k) {
        const int i = from + ((int)threadIdx.x * many + k) * N;
        float x[N];
        s.values(s.load(i, i + N > n || first + i < 0), x);
        place[0] += weigh(x, i, i < to, v);
    }
    u64 mine = place[0];
    block_scan(sh, place, all);
    u64 at = before + place[0];
    const bool last = at <= target && target < at + mine;
    if (!__any_sync(0xffffffffu, last)) return;
    for (int k = 0; k < many; ++k) {
        const int i = from + ((int)threadIdx.x * many + k) * N;
        float x[N];
        s.values(s.load(i, i + N > n || first + i < 0), x);
        weigh(x, i, i < to, v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (last && at <= target && target < at + v[j]) {
                p.tokens[r] = first + i + j;
                if (p.logp) p.logp[r] = w.log_share(x[j], w.log_sum(sum[0]));
            }
            at += v[j];
        }
    }
}

// CTAs a row: as many as put two on every SM, with parts of kLeastPart tokens at
// least, and as keep a part's tokens within what the histograms count.  us with
// parts of 4096 and 32768 at least: 1 x 32768 bf16 top-k 15.9 and 17.8, 1 x 131072 bf16
// top-p 41 and 47, 8 x 50001 f32 top-p 34 and 59; 16 x 131072 bf16 top-k 23.7 and 21.4.
template <typename T>
cudaError_t sample_launch(const SampleParams& p, cudaStream_t s) {
    constexpr int N = Row<T>::N, kLeastPart = 4096;
    // rows that are not on whole vectors begin up to N - 1 values into their first ones
    const bool whole = aligned(p.logits, N * sizeof(T)) && (p.rows == 1 || p.stride % N == 0);
    const int places = p.vocab + (whole ? 0 : N - 1);
    auto part_of = [&](int ranks) { return ((places + ranks - 1) / ranks + N - 1) / N * N; };
    int ranks = 1;
    while (std::min(part_of(ranks), p.vocab) > kMostPart || (ranks < 8 && p.rows * ranks * 2 <= 2 * kSmCount && part_of(ranks * 2) >= kLeastPart)) ranks *= 2;
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

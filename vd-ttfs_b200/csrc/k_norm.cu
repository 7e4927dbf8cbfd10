// k_norm.cu -- the residual's addition, the root-mean-square norm of the sum,
// and its result as values or in 8 bits.
//
//   t = x + residual, rounded to its type;  z_i = t_i w_i;  r = 1 / sqrt(mean(t^2) + eps)
//   values z_i r;  or codes round(z_i / u), u = max_i |z_i| / 127, and the scale u r
//
// The norm is one factor for the whole row, so it goes into the scale alone: a
// code does not depend on how r is rounded, and both reductions, of t^2 and of
// |z|, run over the row at once.
//
// Bound by memory: 16381 x 4096 bf16 with a residual, the sum and codes written,
// 470 MB in 75.7 us, 6.2 TB/s of the 6.5 that a plain copy reaches.  One row of
// 1024, and 777 x 1001 f32, 4 us: a launch, the row's latency and one barrier.
#include "step_internal.h"

namespace vdt {
namespace {

constexpr int kMostHeld = 2048;              // vectors of a row that its threads hold at most

// THREADS a row, by its length alone, so that a row's bits do not hang on the
// rows beside it; nor on where it lies: rows that are not on 16 bytes (WIDE
// false) are read value by value, by the same threads in the same order.  A row
// of up to HELD vectors a thread is read once and stays in registers; of longer
// ones the sum is read (or made) a second time.
template <typename T, int HELD, int THREADS, bool CODES, bool WIDE>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS) k_add_rms_norm(NormParams p) {
    constexpr bool kLong = HELD * THREADS == kMostHeld;      // the others' rows are all held
    constexpr int N = Vec16<T>::N, kWarps = THREADS / 32, kRows = THREADS < 128 ? 128 / THREADS : 1;
    __shared__ float squares[kWarps], largest[kWarps];
    const long long r = (long long)blockIdx.x * kRows + threadIdx.x / THREADS;
    if (kRows > 1 && r >= p.rows) return;
    const int thread = threadIdx.x % THREADS, cols = p.cols;
    const T* const x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* const residual = p.residual ? static_cast<const T*>(p.residual) + r * p.residual_stride : nullptr;
    const T* const weight = static_cast<const T*>(p.weight);
    T* const sum = p.sum ? static_cast<T*>(p.sum) + r * p.sum_stride : nullptr;
    const int vecs = cols / N;
    float square = 0.0f, most = 0.0f;

    auto get = [&](const T* from, int at) {
        Vec16<T> v;
        if constexpr (WIDE) {
            v.raw = *reinterpret_cast<const uint4*>(from + (long long)at * N);
        } else {
            float f[N];
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = to_f32(from[(long long)at * N + j]);
            v.set(f);
        }
        return v;
    };
    auto put = [&](T* to, int at, const Vec16<T>& v) {
        if constexpr (WIDE) {
            *reinterpret_cast<uint4*>(to + (long long)at * N) = v.raw;
        } else {
            float f[N];
            v.get(f);
#pragma unroll
            for (int j = 0; j < N; ++j) to[(long long)at * N + j] = from_f32<T>(f[j]);
        }
    };
    auto times = [&](int at, float* f) {
        if (!weight) return;
        float g[N];
        get(weight, at).get(g);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] *= g[j];
    };
    // the sum's values, as it holds them, their squares added to `into`; stored on the way, which may be over x or the residual
    auto take = [&](int at, Vec16<T> v, const Vec16<T>& o, float& into) {
        float f[N];
        v.get(f);
        if (residual) {
            float g[N];
            o.get(g);
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] += g[j];
            v.set(f);
            v.get(f);
            put(sum, at, v);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) into = fmaf(f[j], f[j], into);
        if constexpr (CODES) {
            times(at, f);
#pragma unroll
            for (int j = 0; j < N; ++j) most = max_nan(fabsf(f[j]), most);
        }
        return v;
    };
    Vec16<T> held[HELD], other[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int at = thread + i * THREADS;
        if (at >= vecs) continue;
        held[i] = get(x, at);
        if (residual) other[i] = get(residual, at);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (thread + i * THREADS < vecs) held[i] = take(thread + i * THREADS, held[i], other[i], square);
    // Of the rest a vector at a time, what an addition rounds off brought into the next one: a sum is off
    // by two roundings however long the row (added one by one, a row of 2^24 equal values was off by
    // 10^4 of them).  An infinite sum stays so.
    if constexpr (kLong) {
        float excess = 0.0f;
        for (int at = thread + HELD * THREADS; at < vecs; at += THREADS) {
            const Vec16<T> v = get(x, at);
            float part = 0.0f;
            take(at, v, residual ? get(residual, at) : v, part);
            const float add = part - excess, to = square + add;
            excess = to == INFINITY ? 0.0f : (to - square) - add;
            square = to;
        }
    }
    // values behind the last whole vector, one for each of the first threads
    const int rest = vecs * N + thread;
    float tail = 0.0f;
    if (rest < cols) {
        tail = to_f32(x[rest]);
        if (residual) {
            const T t = from_f32<T>(tail + to_f32(residual[rest]));
            sum[rest] = t;
            tail = to_f32(t);
        }
        square = fmaf(tail, tail, square);
        if (weight) tail *= to_f32(weight[rest]);
        if constexpr (CODES) most = max_nan(fabsf(tail), most);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        square += __shfl_xor_sync(0xffffffffu, square, d);
        if constexpr (CODES) most = max_nan(__shfl_xor_sync(0xffffffffu, most, d), most);
    }
    if constexpr (kWarps > 1) {
        if (thread % 32 == 0) {
            squares[thread / 32] = square;
            largest[thread / 32] = most;
        }
        __syncthreads();
        square = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            square += squares[i];
            if constexpr (CODES) most = max_nan(largest[i], most);
        }
    }
    const float norm = 1.0f / sqrtf(square / (float)cols + p.eps);
    const T* const again = residual ? sum : x;       // each thread its own values
    if constexpr (CODES) {
        const Coder coder(most * kCodeStep);
        int8_t* const out = p.codes + r * p.out_stride;
        if (thread == 0) p.scale[r] = coder.scale * norm;
        auto store = [&](const Vec16<T>& v, int at) {
            float f[N];
            uint32_t w[N / 4];
            v.get(f);
            times(at, f);
            coder.words<N>(f, w);
            if constexpr (!WIDE) {
#pragma unroll
                for (int j = 0; j < N; ++j) out[(long long)at * N + j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
            } else if constexpr (N == 8) {
                *reinterpret_cast<uint2*>(out + (long long)at * N) = make_uint2(w[0], w[1]);
            } else {
                *reinterpret_cast<uint32_t*>(out + (long long)at * N) = w[0];
            }
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (thread + i * THREADS < vecs) store(held[i], thread + i * THREADS);
        if constexpr (kLong)
            for (int at = thread + HELD * THREADS; at < vecs; at += THREADS) store(get(again, at), at);
        if (rest < cols) out[rest] = (int8_t)code_of(tail, coder.scale);
    } else {
        T* const out = static_cast<T*>(p.out) + r * p.out_stride;
        auto store = [&](Vec16<T> v, int at) {
            float f[N];
            v.get(f);
            times(at, f);
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] *= norm;
            v.set(f);
            put(out, at, v);
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (thread + i * THREADS < vecs) store(held[i], thread + i * THREADS);
        if constexpr (kLong)
            for (int at = thread + HELD * THREADS; at < vecs; at += THREADS) store(get(again, at), at);
        if (rest < cols) out[rest] = from_f32<T>(tail * norm);
    }
}

// The fewest threads that hold a row in one to four vectors each (eight, and more read again, in the
// longest).  More of them are faster for a few rows and slower for many, fewer the other way round up
// to a point; the length alone decides.  us for one row and for 16384, bf16 with a residual, codes: 1024
// columns with 32 threads 3.7 and 25.9, with 128 2.4 and 28.0; 2048 columns with 128 threads
// 2.9 and 42.4, with 256 2.6 and 56.9, with 32 5.7 and 50.6; 4096 columns with 128 threads 3.9 and 74.0, with
// 256 3.3 and 83.8; for one row and 8192, 8192 columns with 256 threads 4.8 and 75.6, with 512 4.4 and
// 108.5, with 128 7.3 and 80.9.
template <typename T, bool CODES, bool WIDE>
cudaError_t norm_by_length(const NormParams& p, cudaStream_t s) {
    const int vecs = p.cols / Vec16<T>::N;
    auto go = [&](auto held, auto threads) {
        constexpr int kHeld = held(), kThreads = threads(), kBlock = kThreads < 128 ? 128 : kThreads;
        const long long each = kBlock / kThreads;
        k_add_rms_norm<T, kHeld, kThreads, CODES, WIDE><<<(unsigned)((p.rows + each - 1) / each), kBlock, 0, s>>>(p);
        return cudaGetLastError();
    };
    if (vecs <= 32) return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
    if (vecs <= 64) return go(std::integral_constant<int, 2>{}, std::integral_constant<int, 32>{});
    if (vecs <= 128) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 32>{});
    if (vecs <= 256) return go(std::integral_constant<int, 2>{}, std::integral_constant<int, 128>{});
    if (vecs <= 512) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 128>{});
    if (vecs <= 1024) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 256>{});
    return go(std::integral_constant<int, 8>{}, std::integral_constant<int, 256>{});
}

template <typename T, bool CODES>
cudaError_t norm_launch(const NormParams& p, cudaStream_t s) {
    constexpr int N = Vec16<T>::N;
    auto wide = [&](const void* at, long long stride) { return aligned(at, 16) && (p.rows == 1 || stride * (long long)sizeof(T) % 16 == 0); };
    const bool vec = wide(p.x, p.x_stride) && (!p.residual || (wide(p.residual, p.residual_stride) && wide(p.sum, p.sum_stride))) &&
                     aligned(p.weight, 16) && (CODES ? aligned(p.codes, N) && (p.rows == 1 || p.out_stride % N == 0) : wide(p.out, p.out_stride));
    return vec ? norm_by_length<T, CODES, true>(p, s) : norm_by_length<T, CODES, false>(p, s);
}

}  // namespace

cudaError_t launch_add_rms_norm(const NormParams& p, cudaStream_t s) {
    if (p.codes) {
        if (p.type == VDT_F32) return norm_launch<float, true>(p, s);
        if (p.type == VDT_F16) return norm_launch<__half, true>(p, s);
        return norm_launch<__nv_bfloat16, true>(p, s);
    }
    if (p.type == VDT_F32) return norm_launch<float, false>(p, s);
    if (p.type == VDT_F16) return norm_launch<__half, false>(p, s);
    return norm_launch<__nv_bfloat16, false>(p, s);
}

}  // namespace vdt

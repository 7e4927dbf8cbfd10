// k_int8.cu -- rows rounded to 8 bits, and their product with 8-bit weights.
//
//   scale_i = max_k |x_ik| / 127,  a_ik = round(x_ik / scale_i)
//   y_ij = scale_i * scale'_j * sum_k a_ik w_jk + bias_j
//
// The sum is exact: 8-bit products are added in 32-bit integers, which hold
// 2^31 / 127^2 = 133,144 of them.  What is rounded is the epilogue: three
// 32-bit operations (sum times scale_i, times scale'_j, plus bias_j) and the
// output's own type.
#include "seq_internal.h"

namespace vdt {
namespace {

// ------------------------------------------------------------------ quantise
constexpr int kQuantThreads = 256;

// One CTA a row: the largest magnitude (a first pass), then the codes (a
// second, from L1 / L2).  16-byte loads where the row allows them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) k_quantize_rows(const T* __restrict__ x, int cols,
                                                                 long long x_stride, int8_t* __restrict__ codes,
                                                                 long long codes_stride, float* __restrict__ scale) {
    constexpr int N = Vec16<T>::N;
    __shared__ float part[kQuantThreads / 32];
    chain_release();
    const T* row = x + (long long)blockIdx.x * x_stride;
    int8_t* out = codes + (long long)blockIdx.x * codes_stride;
    const int vecs = VEC ? cols / N : 0;
    float m = 0.0f;
    for (int i = threadIdx.x; i < vecs; i += kQuantThreads) {
        Vec16<T> v;
        v.raw = *reinterpret_cast<const uint4*>(row + (long long)i * N);
        float f[N];
        v.get(f);
#pragma unroll
        for (int j = 0; j < N; ++j) m = max_nan(fabsf(f[j]), m);
    }
    for (int i = vecs * N + threadIdx.x; i < cols; i += kQuantThreads) m = max_nan(fabsf(to_f32(row[i])), m);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max_nan(__shfl_xor_sync(0xffffffffu, m, d), m);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; ++i) m = max_nan(part[i], m);
    const float sc = m * kCodeStep;
    if (threadIdx.x == 0) scale[blockIdx.x] = sc;
    for (int i = threadIdx.x; i < vecs; i += kQuantThreads) {
        Vec16<T> v;
        v.raw = *reinterpret_cast<const uint4*>(row + (long long)i * N);
        float f[N];
        v.get(f);
        uint32_t w[N / 4];
#pragma unroll
        for (int j = 0; j < N / 4; ++j)
            w[j] = (code_of(f[4 * j], sc) & 255) | (code_of(f[4 * j + 1], sc) & 255) << 8 |
                   (code_of(f[4 * j + 2], sc) & 255) << 16 | (uint32_t)code_of(f[4 * j + 3], sc) << 24;
        if constexpr (N == 8) *reinterpret_cast<uint2*>(out + (long long)i * N) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(out + (long long)i * N) = w[0];
    }
    for (int i = vecs * N + threadIdx.x; i < cols; i += kQuantThreads) out[i] = (int8_t)code_of(to_f32(row[i]), sc);
}

// ---------------------------------------------------------------- few rows
// Each warp takes 16 channels and a share of the inner dimension; mma
// m16n8k32 with the channels as its rows and 8 tokens as its columns.  The
// order of the inner dimension is free as long as both sides keep the same,
// so a lane takes 16 consecutive bytes of a row (one wide load) and feeds
// them to two products.
constexpr int kRowsWarps = 8;

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the bytes of 4-byte word `word` (counted from the row's start) that lie below `inner`
__device__ __forceinline__ uint32_t keep_below(uint32_t v, int word, int inner) {
    const int left = inner - 4 * word;
    return left >= 4 ? v : left <= 0 ? 0u : v & ((1u << (8 * left)) - 1u);
}

template <typename T, int NT>
__global__ void __launch_bounds__(kRowsWarps * 32) k_int8_rows(Int8Params p) {
    __shared__ int part[kRowsWarps][16][8 * NT + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int col0 = blockIdx.x * 16;
    const long long row0 = (long long)blockIdx.y * (8 * NT);
    chain_wait();
    int acc[NT][4] = {};
    // rows past the end read the last one; their products are not stored
    const int8_t* w0 = p.w + (long long)min(col0 + g, p.cols - 1) * p.w_stride;
    const int8_t* w1 = p.w + (long long)min(col0 + g + 8, p.cols - 1) * p.w_stride;
    const int8_t* a[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) a[n] = p.a + min(row0 + 8 * n + g, p.rows - 1) * p.a_stride;
    const int steps = (p.inner + 63) / 64;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int s = warp; s < steps; s += kRowsWarps) {
        const int k = s * 64 + t * 16;
        const bool in = k < p.inner;     // a row's storage reaches to the next multiple of 16
        const uint4 u0 = in ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : zero;
        const uint4 u1 = in ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            uint4 b = in ? *reinterpret_cast<const uint4*>(a[n] + k) : zero;
            if (k + 16 > p.inner) {
                b.x = keep_below(b.x, k / 4, p.inner);
                b.y = keep_below(b.y, k / 4 + 1, p.inner);
                b.z = keep_below(b.z, k / 4 + 2, p.inner);
                b.w = keep_below(b.w, k / 4 + 3, p.inner);
            }
            mma_s8(acc[n], u0.x, u1.x, u0.y, u1.y, b.x, b.y);
            mma_s8(acc[n], u0.z, u1.z, u0.w, u1.w, b.z, b.w);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        part[warp][g][8 * n + 2 * t] = acc[n][0];
        part[warp][g][8 * n + 2 * t + 1] = acc[n][1];
        part[warp][g + 8][8 * n + 2 * t] = acc[n][2];
        part[warp][g + 8][8 * n + 2 * t + 1] = acc[n][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += kRowsWarps * 32) {
        const int c = i % 16, r = i / 16;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) sum += part[w][c][r];
        const int col = col0 + c;
        const long long row = row0 + r;
        if (col < p.cols && row < p.rows) {
            float y = (float)sum * p.a_scale[row] * p.w_scale[col];
            if (p.bias) y += p.bias[col];
            static_cast<T*>(p.out)[row * p.out_stride + col] = from_f32<T>(y);
        }
    }
}

template <typename T>
cudaError_t rows_launch(const Int8Params& p, bool after, cudaStream_t s) {
    const int nt = p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
    const dim3 grid((p.cols + 15) / 16, (unsigned)((p.rows + 8 * nt - 1) / (8 * nt)));
    auto kern = nt == 1 ? k_int8_rows<T, 1> : nt == 2 ? k_int8_rows<T, 2> : k_int8_rows<T, 4>;
    if (after) return launch_after(kern, grid, dim3(kRowsWarps * 32), 0, s, p);
    kern<<<grid, kRowsWarps * 32, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t quant_launch(const void* x, long long rows, int cols, long long x_stride, int8_t* codes,
                         long long codes_stride, float* scale, cudaStream_t s) {
    constexpr int N = Vec16<T>::N;
    const bool vec = aligned(x, 16) && (x_stride * (long long)sizeof(T)) % 16 == 0 && aligned(codes, N) &&
                     codes_stride % N == 0;
    const T* in = static_cast<const T*>(x);
    if (vec) k_quantize_rows<T, true><<<(unsigned)rows, kQuantThreads, 0, s>>>(in, cols, x_stride, codes, codes_stride, scale);
    else k_quantize_rows<T, false><<<(unsigned)rows, kQuantThreads, 0, s>>>(in, cols, x_stride, codes, codes_stride, scale);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int type, long long rows, int cols, long long x_stride,
                                 int8_t* codes, long long codes_stride, float* scale, cudaStream_t s) {
    if (type == VDT_F32) return quant_launch<float>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    if (type == VDT_F16) return quant_launch<__half>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    return quant_launch<__nv_bfloat16>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
}

cudaError_t launch_int8_matmul(const Int8Params& p, bool after_codes, cudaStream_t s) {
    if (p.out_type == VDT_F32) return rows_launch<float>(p, after_codes, s);
    if (p.out_type == VDT_F16) return rows_launch<__half>(p, after_codes, s);
    return rows_launch<__nv_bfloat16>(p, after_codes, s);
}

}  // namespace vdt

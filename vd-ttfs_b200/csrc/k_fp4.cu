// k_fp4.cu -- rows in microscaled 4-bit floating point, and their product.
//
// A block of 32 values x_k of a row has one power of two 2^e, the smallest with
// max|x_k| <= 6 * 2^e, and codes c_k: x_k / 2^e rounded to the nearest of 0, 1/2,
// 1, 3/2, 2, 3, 4, 6 and their negatives, ties to the even code.  (Rounding the exponent
// down, as for a block whose largest value may be cut off at 6, would take up to
// a quarter off the outlying values that a scale of their own is there for.)
//
//   y_ij = sum over blocks 2^(e_ib + e'_jb) sum_k c_ik c'_jk + bias_j
//
// The tensor cores multiply such operands as they are, codes from shared memory
// and scales from tensor memory, with 32-bit sums.
#include <cooperative_groups.h>

#include <algorithm>

#include "step_internal.h"

namespace vdt {
namespace {

namespace cg = cooperative_groups;

// The block's scale byte, e + 127, from its largest magnitude's bits: max = m 2^k
// <= 3/2 2^(e + 2), so e = k - 2, or k - 1 for m above 3/2.  255 where there is an
// infinity or NaN.
__device__ __forceinline__ uint32_t scale_byte(float most) {
    const uint32_t b = __float_as_uint(most);
    if (b >= 0x7f800000u) return 255;
    const int e = (int)(b >> 23) - 2 + ((b & 0x7fffffu) > 0x400000u);
    return (uint32_t)max(e, 0);
}
// 2^-e, a normal number for every byte but 255, whose codes are zeros
__device__ __forceinline__ float inverse_of(uint32_t byte) { return byte == 255 ? 0.0f : __uint_as_float((254 - byte) << 23); }
// byte 0 is 2^-127, below the normal numbers
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return byte == 255 ? __uint_as_float(0x7fffffffu) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x400000u);
}

// Eight values' codes, the first in the lowest bits
__device__ __forceinline__ uint32_t codes_of(const float* f) {
    uint32_t w;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return w;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// A block of 32 values as they lie in memory -> its 16 bytes of codes; returns the
// scale's byte.  One thread a block: no exchange, and the scale is made once.
// bf16 values are scaled as they are (a power of two changes no bit but the
// exponent's, and what falls below the smallest number has code 0 anyway).
template <typename T>
__device__ __forceinline__ uint32_t round_block(const uint32_t (&raw)[8 * sizeof(T)], uint4& codes) {
    float most;
    uint32_t w[4];
    if constexpr (sizeof(T) == 4) {
        most = fabsf(__uint_as_float(raw[0]));
#pragma unroll
        for (int i = 1; i < 32; ++i) most = max_or_nan(most, fabsf(__uint_as_float(raw[i])));
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        __nv_bfloat162 m, o;
        memcpy(&m, &raw[0], 4);
        m = __habs2(m);
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            memcpy(&o, &raw[i], 4);
            m = __hmax2_nan(m, __habs2(o));
        }
        most = max_or_nan(__low2float(m), __high2float(m));
    } else {
        __half2 m, o;
        memcpy(&m, &raw[0], 4);
        m = __habs2(m);
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            memcpy(&o, &raw[i], 4);
            m = __hmax2_nan(m, __habs2(o));
        }
        most = max_or_nan(__low2float(m), __high2float(m));
    }
    const uint32_t byte = scale_byte(fabsf(most));
    const float inverse = inverse_of(byte);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float f[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(raw[8 * q + j]) * inverse;
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 by = __float2bfloat162_rn(inverse);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                __nv_bfloat162 o;
                memcpy(&o, &raw[4 * q + j], 4);
                o = __hmul2(o, by);
                uint32_t u;
                memcpy(&u, &o, 4);
                unpack2<T>(u, f[2 * j], f[2 * j + 1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unpack2<T>(raw[4 * q + j], f[2 * j], f[2 * j + 1]);
                f[2 * j] *= inverse;
                f[2 * j + 1] *= inverse;
            }
        }
        w[q] = codes_of(f);
    }
    codes = byte == 255 ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
    return byte;
}
// The block's values, those at or past `left` as zeros.  ALIGN: the bytes that it starts on a multiple of.
template <typename T, int ALIGN>
__device__ __forceinline__ void load_block(const T* from, int left, uint32_t (&raw)[8 * sizeof(T)]) {
    constexpr int kWords = 8 * sizeof(T);
    if (ALIGN == 32 && left >= 32) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(raw[i]), "=r"(raw[i + 1]), "=r"(raw[i + 2]), "=r"(raw[i + 3]), "=r"(raw[i + 4]), "=r"(raw[i + 5]), "=r"(raw[i + 6]),
                           "=r"(raw[i + 7])
                         : "l"(reinterpret_cast<const uint32_t*>(from) + i));
    } else if (ALIGN >= 16 && left >= 32) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(from) + i);
            raw[i] = v.x;
            raw[i + 1] = v.y;
            raw[i + 2] = v.z;
            raw[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                raw[i] = i < left ? __float_as_uint(from[i]) : 0u;
            } else {
                uint16_t lo = 0, hi = 0;
                if (2 * i < left) memcpy(&lo, from + 2 * i, 2);
                if (2 * i + 1 < left) memcpy(&hi, from + 2 * i + 1, 2);
                raw[i] = lo | (uint32_t)hi << 16;
            }
        }
    }
}

// Where the scale of a row's block lies: tiles of 128 rows x 4 blocks, row r's
// four bytes at r % 32 * 16 + r / 32 * 4, which is how the tensor memory takes
// them (lane r % 32, column r / 32)
__device__ __forceinline__ long long scale_at(long long row, int block, long long steps) {
    const int r = (int)(row % kScaleRows);
    return (row / kScaleRows * steps * 2 + block / 4) * kScaleTile + r % 32 * 16 + r / 32 * 4 + block % 4;
}

// ------------------------------------------------------------------ quantise
// A thread a block.  2^across threads (8, 16 or 32) side by side take a row's
// blocks, the scales' padding included, so rows of few columns share a warp.  Bound
// by memory: 8192 x 4096 bf16 14.7 us, 5.8 TB/s (four lanes a block, which exchange
// their maxima, took 26 us and four times the instructions).
constexpr int kPackThreads = 128;
template <typename T, int ALIGN>
__global__ void __launch_bounds__(kPackThreads) k_quantize_fp4(const T* __restrict__ x, long long rows, int cols, long long x_stride,
                                                               uint8_t* __restrict__ codes, long long codes_stride, uint8_t* __restrict__ scale,
                                                               int steps, int across) {
    chain_release();
    const int block = (blockIdx.x << across) + (threadIdx.x & ((1 << across) - 1)), per = kPackThreads >> across;
    const int col = block * kBlock;
    for (long long row = (long long)blockIdx.y * per + (threadIdx.x >> across); row - (threadIdx.x >> across) < rows; row += (long long)gridDim.y * per) {
        const bool in = row < rows && block < steps * (kFp4Step / kBlock);
        uint32_t raw[8 * sizeof(T)];
        if constexpr (ALIGN >= 16) {
            load_block<T, ALIGN>(x + row * x_stride + col, in ? cols - col : 0, raw);
        } else {
            // a block's 32 values by the warp's lanes, then each lane its block; rows of 33 words (f32) or 17
            constexpr int kPitch = sizeof(T) == 4 ? 33 : 34;
            __shared__ T side[kPackThreads / 32][32 * kPitch];
            T* const mine = side[threadIdx.x / 32];
            const int lane = threadIdx.x % 32, mask = (1 << across) - 1;
            __syncwarp();
#pragma unroll 8
            for (int i = 0; i < 32; ++i) {
                const int from = (threadIdx.x & ~31) + i;             // the thread whose block it is
                const long long r = row + (from >> across) - (threadIdx.x >> across);
                const int c = ((blockIdx.x << across) + (from & mask)) * kBlock + lane;
                mine[i * kPitch + lane] = r < rows && c < cols ? x[r * x_stride + c] : from_f32<T>(0.0f);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < (int)(8 * sizeof(T)); ++i) memcpy(&raw[i], mine + lane * kPitch + i * (4 / (int)sizeof(T)), 4);
        }
        uint4 w;
        uint32_t byte = round_block<T>(raw, w);
        // (the last row's storage reaches to the next 16 bytes)
        if (in && col < cols) *reinterpret_cast<uint4*>(codes + row * codes_stride + col / 2) = w;
        // four blocks' bytes together
        byte |= __shfl_down_sync(0xffffffffu, byte, 1) << 8;
        byte |= __shfl_down_sync(0xffffffffu, byte, 2) << 16;
        if (in && block % 4 == 0) *reinterpret_cast<uint32_t*>(scale + scale_at(row, block, steps)) = byte;
    }
}

template <typename T>
cudaError_t pack_launch(const void* x, long long rows, int cols, long long x_stride, uint8_t* codes, long long codes_stride, uint8_t* scale,
                        cudaStream_t s) {
    auto on = [&](int bytes) { return aligned(x, bytes) && (rows == 1 || x_stride * (long long)sizeof(T) % bytes == 0); };
    const int steps = (int)fp4_steps(cols), blocks = steps * (kFp4Step / kBlock), across = steps == 1 ? 3 : steps == 2 ? 4 : 5;
    const long long per = kPackThreads >> across, down = (rows + per - 1) / per;
    const dim3 grid((unsigned)((blocks + (1 << across) - 1) >> across), (unsigned)std::min(down, 65535LL));
    auto kern = on(32) ? k_quantize_fp4<T, 32> : on(16) ? k_quantize_fp4<T, 16> : k_quantize_fp4<T, 1>;
    kern<<<grid, kPackThreads, 0, s>>>(static_cast<const T*>(x), rows, cols, x_stride, codes, codes_stride, scale, steps, across);
    return cudaGetLastError();
}

// --------------------------------------------------------------------- values
__device__ __forceinline__ float value_of(uint32_t code, float scale) {
    const uint32_t m = code & 7;
    const float v = m < 4 ? 0.5f * m : m < 6 ? (float)(m - 2) : 2.0f * (m - 4);
    return (code & 8 ? -v : v) * scale;
}
template <typename T>
__global__ void __launch_bounds__(256) k_fp4_values(const uint8_t* __restrict__ codes, long long codes_stride, const uint8_t* __restrict__ scale,
                                                    long long rows, int cols, T* __restrict__ out, long long out_stride, long long steps) {
    const int per = (cols + 7) / 8;
    const long long units = rows * per;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
        const long long row = u / per;
        const int col = (int)(u - row * per) * 8;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + row * codes_stride + col / 2);
        const float by = scale_of(scale[scale_at(row, col / kBlock, steps)]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < cols) out[row * out_stride + col + j] = from_f32<T>(value_of(w >> (4 * j) & 15, by));
    }
}

// -------------------------------------------------- block-scaled matrix products
// d += a b with scales: 128 rows of both operands' 64 consecutive 4-bit values
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t a_scale, uint32_t b_scale, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape),
        "r"(a_scale), "r"(b_scale), "r"((uint32_t)add)
        : "memory");
}
// a scale tile of 512 bytes into four columns of the tensor memory, the same for each of its four quarters
__device__ __forceinline__ void scales_copy(uint32_t to, uint64_t tile) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(tile) : "memory");
}
// rows of 16 bytes without swizzle, eight to a group of 128 bytes
__device__ __forceinline__ uint64_t scale_desc(uint32_t at) {
    return (uint64_t)((at & 0x3ffff) >> 4) | 1ull << 16 | (uint64_t)(128 >> 4) << 32 | 1ull << 46;
}
// e2m1 operands, both with the inner dimension consecutive, scales of 8 exponent
// bits; `pair`: which two of a scale column's four bytes
__device__ __forceinline__ constexpr uint32_t fp4_shape(int n, int pair) {
    return 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(128 >> 4) << 24 | (uint32_t)(2 * pair) << 29 | (uint32_t)(2 * pair) << 4;
}

constexpr int kStepBytes = kFp4Step / 2;             // 128: a swizzled row of a stage
constexpr int kStepScales = 2 * kScaleTile;          // a stage's scales for 128 rows

// ----------------------------------------------------------------- few rows
// The channels are the products' 128 rows and the tokens, at most NT, their columns, so a
// tile holds 128 channels whatever the number of tokens, and what bounds it is the
// weights' way from memory.  A cluster of CTAs shares a tile's inner dimension, so
// that all SMs load at once and every CTA's stages are on their way from the
// start; the sums meet in shared memory.  X: the type of rows that are still to be
// rounded, which eight warps do for their CTA's part of the inner dimension while
// the weights come; void: they are codes.  24 x 4096 x 8192 f16:
// 9.2 us (17.8 MB of weights, from L2 where they fit; without the rounding 6.7).
constexpr int kFewStages = 4, kRoundWarps = 8;

// Up to kOwnRows the kernel rounds the rows itself.  A call / on the GPU in us, so and
// with two launches, f16: 1 x 4096 x 8192 9.6 / 7.5 and 12.5 / 8.0, 16 x 1024 x 1024
// 7.0 / 4.6 and 9.8 / 6.2, 32 x 4096 x 8192 11.3 / 9.2 and 14.1 / 8.7, 32 x 8192 x 1024
// 8.8 / 6.7 and 12.0 / 7.5; not taken: 64 x 4096 x 8192 15.6 / 13.5 and 14.3 / 11.8.
// Up to kFewRows the tokens may be the columns; above kOwnRows where sharing the
// inner dimension takes more than kFewSteps steps off each CTA (us, so and with the
// tiles below): 64 x 4096 x 4096 6.7 and 8.0, 64 x 8192 x 1024 6.3 and 12.4, 64 x
// 4096 x 8192 8.2 and 7.9, not taken: 64 x 1024 x 1024 5.3 and 4.5.
constexpr int kFewRows = 64, kOwnRows = 32, kFewSteps = 6;

template <int NT>
struct FewShape {
    static constexpr int kCodes = (128 + NT) * kStepBytes;
    static constexpr int kStage = kCodes + 2 * kStepScales;
    static constexpr int kBytes = 1024 + kFewStages * kStage + NT * 512;
    static constexpr int kScalesAt = 64, kScaleCols = 16, kCols = 128;     // tensor memory: sums, then 16 columns of scales a stage
    static_assert(NT <= kScalesAt && kScalesAt + kFewStages * kScaleCols <= kCols, "tile");
};
struct FewBars {
    uint64_t full[kFewStages], empty[kFewStages], done;
    uint32_t tmem;
};

template <typename X, int NT>
__global__ void __launch_bounds__(std::is_void_v<X> ? 192 : 64 + 32 * kRoundWarps) k_fp4_few(const __grid_constant__ CUtensorMap map_w,
                                                                                            const __grid_constant__ CUtensorMap map_a, Fp4Params p) {
    using Shape = FewShape<NT>;
    constexpr bool kOwn = !std::is_void_v<X>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ FewBars bars;
    unsigned char* const smem = smem_raw + ((1024 - (shared_address(smem_raw) & 1023)) & 1023);
    const uint32_t stages = shared_address(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const cg::cluster_group cluster = cg::this_cluster();
    const int split = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tile = blockIdx.x / split, rows = (int)p.rows;
    const int steps = (p.inner + kFp4Step - 1) / kFp4Step;
    const int first = (int)((long long)steps * rank / split), last = (int)((long long)steps * (rank + 1) / split);
    if (threadIdx.x == 0) {
        map_ahead(&map_w);
        for (int i = 0; i < kFewStages; ++i) {
            bar_init(shared_address(&bars.full[i]), kOwn ? 1 + NT / 4 : 1);
            bar_init(shared_address(&bars.empty[i]), 1);
        }
        bar_init(shared_address(&bars.done), 1);
        bar_init_done();
    }
    if (warp == 1) tmem_alloc(shared_address(&bars.tmem), Shape::kCols);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = bars.tmem;
    bool alive = true;

    if (warp == 0) {
        if (lane == 0) {
            auto load_w = [&](int s) {
                const int slot = (s - first) % kFewStages;
                const uint32_t at = stages + slot * Shape::kStage, bar = shared_address(&bars.full[slot]);
                bar_expect(bar, kOwn ? 128 * kStepBytes + kStepScales : Shape::kStage);
                tile_load(at, &map_w, s * kStepBytes, tile * 128, bar);
                bulk_load(at + Shape::kCodes, p.w_scale + ((long long)tile * steps + s) * kStepScales, kStepScales, bar);
            };
            // the weights are the caller's: the first stages' need not wait for the codes
            const int ahead = min(last, first + kFewStages);
            for (int s = first; s < ahead; ++s) load_w(s);
            if constexpr (!kOwn) chain_wait();
            for (int s = first; s < last && alive; ++s) {
                const int slot = (s - first) % kFewStages;
                const uint32_t at = stages + slot * Shape::kStage, bar = shared_address(&bars.full[slot]);
                if (s >= ahead) {
                    if (!(alive = bar_wait(shared_address(&bars.empty[slot]), ((s - first) / kFewStages & 1) ^ 1))) break;
                    load_w(s);
                }
                if constexpr (!kOwn) {
                    tile_load(at + 128 * kStepBytes, &map_a, s * kStepBytes, 0, bar);
                    bulk_load(at + Shape::kCodes + kStepScales, p.a_scale + (long long)s * kStepScales, kStepScales, bar);
                }
            }
            // every load has landed before the CTA ends: the last ones' stages
            for (int s = max(first, last - kFewStages); s < last; ++s)
                bar_wait(shared_address(&bars.full[(s - first) % kFewStages]), (s - first) / kFewStages & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t sums = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t w = tile_desc(stages), a = tile_desc(stages + 128 * kStepBytes), f = scale_desc(stages + Shape::kCodes);
        const bool one = elected();
        for (int s = first; s < last; ++s) {
            const int slot = (s - first) % kFewStages;
            if (!(alive = bar_wait_all(shared_address(&bars.full[slot]), (s - first) / kFewStages & 1))) break;
            tmem_fence_after();
            if (one) {
                const uint32_t sc = sums + Shape::kScalesAt + slot * Shape::kScaleCols;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        scales_copy(sc + h * 8 + j * 4, f + (slot * Shape::kStage + j * kStepScales + h * kScaleTile) / 16);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_fp4(sums, w + (slot * Shape::kStage + k * 32) / 16, a + (slot * Shape::kStage + k * 32) / 16, fp4_shape(NT, k % 2), sc + k / 2 * 8,
                            sc + k / 2 * 8 + 4, s > first || k > 0);
                mma_commit(shared_address(&bars.empty[slot]));
            }
        }
        if (alive && one) mma_commit(shared_address(&bars.done));
    } else if constexpr (kOwn) {
        // A thread a block of a step, eight of them a row; the next step's values on their
        // way meanwhile.  What a step leaves over of the threads takes the next one, so that
        // the steps' loads do not wait for each other.
        constexpr int kGroup = NT * 8, kGroups = 32 * kRoundWarps / kGroup;
        static_assert(kGroups >= 1, "a thread a block");
        const int t = (threadIdx.x - 64) % kGroup, block = t % 8, row = t / 8;
        const X* const x = static_cast<const X*>(p.x) + row * p.x_stride + block * kBlock;
        const uintptr_t off = reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(rows > 1 ? p.x_stride * (long long)sizeof(X) : 0);
        uint32_t raw[8 * sizeof(X)];
        auto load = [&](int s) {
            const int col = s * kFp4Step, left = row < rows && s < last ? p.inner - col - block * kBlock : 0;
            if (off % 32 == 0) load_block<X, 32>(x + col, left, raw);
            else if (off % 16 == 0) load_block<X, 16>(x + col, left, raw);
            else load_block<X, 1>(x + col, left, raw);
        };
        int s = first + (threadIdx.x - 64) / kGroup;
        load(s);
        for (; s < last; s += kGroups) {
            const int slot = (s - first) % kFewStages;
            unsigned char* const at = smem + slot * Shape::kStage;
            uint4 w;
            const uint32_t byte = round_block<X>(raw, w);
            load(s + kGroups);
            if (s - first >= kFewStages) {
                if (!bar_wait_all(shared_address(&bars.empty[slot]), ((s - first) / kFewStages & 1) ^ 1)) break;
            }
            if (row < rows) {
                *reinterpret_cast<uint4*>(at + (128 + row) * kStepBytes + ((block ^ (row & 7)) << 4)) = w;      // swizzled by the row
                at[Shape::kCodes + kStepScales + block / 4 * kScaleTile + row % 32 * 16 + row / 32 * 4 + block % 4] = (unsigned char)byte;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the tensor cores read what these lanes wrote
            __syncwarp();
            if (lane == 0) bar_arrive(shared_address(&bars.full[slot]));
        }
    }

    // the sums: channel 32 (warp % 4) + lane, tokens side by side
    const int quarter = warp % 4;
    float* const part = reinterpret_cast<float*>(smem + kFewStages * Shape::kStage);      // [NT][128]
    if (warp >= 2 && warp < 6) {
        alive = bar_wait_all(shared_address(&bars.done), 0);
        tmem_fence_after();
#pragma unroll
        for (int b = 0; b < (NT + 31) / 32; ++b) {
            uint32_t r[32];
            tmem_load(tmem + (quarter * 32 << 16) + b * 32, r);
            tmem_load_wait();
#pragma unroll
            for (int c = 0; c < (NT < 32 ? NT : 32); ++c)
                part[(b * 32 + c) * 128 + quarter * 32 + lane] = alive ? __uint_as_float(r[c]) : __int_as_float(0x7fffffff);
        }
    }
    tmem_fence_before();
    __syncwarp();
    if (split > 1) cluster.sync();
    else __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tmem_fence_after();
        tmem_free(tmem, Shape::kCols);
    }
    // each CTA adds up its share of the tokens, four channels a thread
    const int from = rows * rank / split, to = rows * (rank + 1) / split;
    const bool wide = p.out_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    for (int i = threadIdx.x; i < (to - from) * 32; i += blockDim.x) {
        const int row = from + i / 32, c = i % 32 * 4, col = tile * 128 + c;
        float4 o[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < split) o[r] = *reinterpret_cast<const float4*>((split > 1 ? cluster.map_shared_rank(part, r) : part) + row * 128 + c);
        float y[4] = {o[0].x, o[0].y, o[0].z, o[0].w};
#pragma unroll
        for (int r = 1; r < 8; ++r)
            if (r < split) {
                y[0] += o[r].x;
                y[1] += o[r].y;
                y[2] += o[r].z;
                y[3] += o[r].w;
            }
        if (p.bias)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < p.cols) y[j] += p.bias[col + j];
        const long long at = row * p.out_stride + col;
        auto put = [&](auto* out) {
            using T = std::remove_pointer_t<decltype(out)>;
            if (wide && col + 4 <= p.cols) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + at) = make_float4(y[0], y[1], y[2], y[3]);
                else *reinterpret_cast<uint2*>(out + at) = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < p.cols) out[at + j] = from_f32<T>(y[j]);
            }
        };
        if (p.out_type == VDT_F32) put(static_cast<float*>(p.out));
        else if (p.out_type == VDT_F16) put(static_cast<__half*>(p.out));
        else put(static_cast<__nv_bfloat16*>(p.out));
    }
    if (split > 1) cluster.sync();                                   // until the others have read this CTA's part
}

// CTAs a tile: as many as the SMs hold at a time (two each, or one with 64 tokens), each with a step at least
int few_split(int cols, int inner, int tokens) {
    const long long tiles = (cols + 127) / 128, steps = fp4_steps(inner);
    int split = 1;
    while (split < 8 && tiles * split * 2 <= (tokens == 64 ? 1 : 2) * kSmCount && steps >= split * 2) split *= 2;
    return split;
}
template <typename X, int NT>
cudaError_t few_launch(const Fp4Params& p, bool after, cudaStream_t s) {
    using Shape = FewShape<NT>;
    CUtensorMap w, a;
    const int bytes = (p.inner + 1) / 2;
    if (p.rows > NT) return cudaErrorInvalidValue;
    if (!byte_rows_map(&w, p.w, p.cols, bytes, p.w_stride, kStepBytes, 128)) return cudaErrorInvalidValue;
    if (std::is_void_v<X>) {
        if (!byte_rows_map(&a, p.a, p.rows, bytes, p.a_stride, kStepBytes, NT)) return cudaErrorInvalidValue;
    } else {
        a = w;
    }
    const cudaError_t e = allow_shared<k_fp4_few<X, NT>>(Shape::kBytes);
    if (e != cudaSuccess) return e;
    const int split = few_split(p.cols, p.inner, NT);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.cols + 127) / 128 * split));
    cfg.blockDim = dim3(std::is_void_v<X> ? 192 : 64 + 32 * kRoundWarps);
    cfg.dynamicSmemBytes = Shape::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = after ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k_fp4_few<X, NT>, w, a, p);
}
template <typename X>
cudaError_t few_by_rows(const Fp4Params& p, bool after, cudaStream_t s) {
    if (p.rows <= 16) return few_launch<X, 16>(p, after, s);
    if constexpr (std::is_void_v<X>) {
        if (p.rows > 32) return few_launch<X, 64>(p, after, s);
    }
    return few_launch<X, 32>(p, after, s);
}

// ---------------------------------------------------------------- many rows
// Persistent CTAs over tiles of 128 rows x BN channels, as for 8-bit integers:
// one thread keeps a ring of stages (256 columns of both sides and their
// scales) full, one copies scales and issues products, eight warps turn sums
// into outputs.  The scales of a stage have columns of the tensor memory of
// their own, so they are written again only after the products that read them.
// Beside them there is no room for two tiles' sums of 256 channels, so the eight
// warps take all of a tile's sums into registers at once (128 a thread) and the
// next tile's products start before the first output is written.  What bounds it
// is the way of the stages from L2, some 19 TB/s; tiles of 192 channels, whose sums fit
// twice, read a sixth more of them.  8192 x 4096 x 8192:
// 103 us, 5.3 PFLOP/s (113 with 192 channels; 79 without the weights' loads, 88 without
// the outputs' stores).
constexpr int kTileRows = 128, kOutWarps = 8, kTileThreads = 64 + 32 * kOutWarps;

template <int BN>
struct TileShape {
    static constexpr int kWTiles = BN <= 128 ? 1 : 2;                      // scale tiles that BN channels may touch
    static constexpr int kCodes = (kTileRows + BN) * kStepBytes;
    static constexpr int kStage = kCodes + (1 + kWTiles) * kStepScales;
    static constexpr int kStages = BN >= 192 ? 4 : BN == 128 ? 5 : 6;
    static constexpr int kSums = BN == 256 ? 1 : 2;                        // tiles whose sums fit beside the scales
    static constexpr int kScaleCols = 8 * (1 + kWTiles);                   // of a stage
    static constexpr int kScalesAt = kSums * BN;
    static constexpr int kUsed = kScalesAt + kStages * kScaleCols;
    static constexpr int kCols = kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kOut = kOutWarps * 2048;                          // 32 rows of 64 bytes for each warp, where outputs are not on 32 bytes
    static constexpr int kBias = 2 * BN * 4;
    static constexpr int kBytes = 1024 + kStages * kStage + kOut + kBias;
    static_assert(kUsed <= 512 && kBytes <= 232448 && kStage % 1024 == 0, "tile");
};

struct TileBars {
    uint64_t full[8], empty[8], done[2], taken[2];
    uint32_t tmem;
};

template <typename T, int BN>
__global__ void __launch_bounds__(kTileThreads, 1) k_fp4_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                                                               Fp4Params p, int tiles_m, int tiles) {
    using Shape = TileShape<BN>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileBars bars;
    unsigned char* smem = smem_raw + ((1024 - (shared_address(smem_raw) & 1023)) & 1023);
    const uint32_t stages = shared_address(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int steps = (p.inner + kFp4Step - 1) / kFp4Step;
    if (threadIdx.x == 0) {
        map_ahead(&map_w);
        map_ahead(&map_a);
        for (int i = 0; i < Shape::kStages; ++i) {
            bar_init(shared_address(&bars.full[i]), 1);
            bar_init(shared_address(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(shared_address(&bars.done[i]), 1);
            bar_init(shared_address(&bars.taken[i]), 32 * kOutWarps);
        }
        bar_init_done();
    }
    if (warp == 1) tmem_alloc(shared_address(&bars.tmem), Shape::kCols);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = bars.tmem;
    const int w_tiles = (p.cols + kScaleRows - 1) / kScaleRows;
    // the channels' part of a stage: codes, and the scale tiles that the channels touch
    auto load_w = [&](uint32_t at, uint32_t bar, int s, int c) {
        tile_load(at + kTileRows * kStepBytes, &map_w, s * kStepBytes, c, bar);
        const int t0 = c / kScaleRows;
#pragma unroll
        for (int i = 0; i < Shape::kWTiles; ++i)            // a tile past the last has the last one's scales; its products are not stored
            bulk_load(at + Shape::kCodes + (1 + i) * kStepScales, p.w_scale + ((long long)min(t0 + i, w_tiles - 1) * steps + s) * kStepScales,
                      kStepScales, bar);
    };
    // the weights are the caller's: the first stages' need not wait for the codes
    const int ahead = min(steps, Shape::kStages);
    if (threadIdx.x == 0)
        for (int s = 0; s < ahead; ++s) {
            const uint32_t bar = shared_address(&bars.full[s]);
            bar_expect(bar, Shape::kStage);
            load_w(stages + s * Shape::kStage, bar, s, blockIdx.x / tiles_m * BN);
        }
    chain_wait();

    if (warp == 0) {
        if (lane == 0) {
            int n = 0;
            bool alive = true;
            for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
                const int t = tile % tiles_m, c = tile / tiles_m * BN;
                for (int s = 0; s < steps; ++s, ++n) {
                    const int slot = n % Shape::kStages;
                    const uint32_t at = stages + slot * Shape::kStage, bar = shared_address(&bars.full[slot]);
                    if (n >= ahead) {
                        if (!(alive = bar_wait(shared_address(&bars.empty[slot]), (n / Shape::kStages & 1) ^ 1))) break;
                        bar_expect(bar, Shape::kStage);
                        load_w(at, bar, s, c);
                    }
                    tile_load(at, &map_a, s * kStepBytes, t * kTileRows, bar);
                    bulk_load(at + Shape::kCodes, p.a_scale + ((long long)t * steps + s) * kStepScales, kStepScales, bar);
                }
            }
            // every load has landed before the CTA ends: the last ones' stages
            for (int i = max(0, n - Shape::kStages); i < n; ++i)
                bar_wait(shared_address(&bars.full[i % Shape::kStages]), i / Shape::kStages & 1);
        }
    } else if (warp == 1) {
        const uint32_t sums = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t a = tile_desc(stages), w = tile_desc(stages + kTileRows * kStepBytes), f = scale_desc(stages + Shape::kCodes);
        const bool one = elected();
        int n = 0, i = 0;
        bool alive = true;
        for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x, ++i) {
            const int half = i % Shape::kSums;
            // the first channel's place in its scale tile, a column for 32
            const uint32_t shift = tile / tiles_m * BN % kScaleRows / 32;
            if (!(alive = bar_wait_all(shared_address(&bars.taken[half]), (i / Shape::kSums & 1) ^ 1))) break;
            tmem_fence_after();
            for (int s = 0; s < steps; ++s, ++n) {
                const int slot = n % Shape::kStages;
                if (!(alive = bar_wait_all(shared_address(&bars.full[slot]), n / Shape::kStages & 1))) break;
                tmem_fence_after();
                if (one) {
                    const uint32_t sc = sums + Shape::kScalesAt + slot * Shape::kScaleCols;
                    // columns: 128 columns of the inner dimension after another, in each the rows' tile, then the channels' tiles
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 1 + Shape::kWTiles; ++j)
                            scales_copy(sc + h * (Shape::kScaleCols / 2) + j * 4, f + (slot * Shape::kStage + j * kStepScales + h * kScaleTile) / 16);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t at = sc + k / 2 * (Shape::kScaleCols / 2);
                        mma_fp4(sums + half * BN, a + (slot * Shape::kStage + k * 32) / 16, w + (slot * Shape::kStage + k * 32) / 16, fp4_shape(BN, k % 2),
                                at, at + 4 + shift, s > 0 || k > 0);
                    }
                    mma_commit(shared_address(&bars.empty[slot]));
                }
            }
            if (alive && one) mma_commit(shared_address(&bars.done[half]));
        }
    } else {
        // a warp reads the rows of its quarter, half of the channels
        constexpr int kCols = BN / 2, kWords = kCols * (int)sizeof(T) / 4;
        const int quarter = warp % 4, thread = threadIdx.x - 64, half_col = (warp - 2) / 4 * kCols;
        unsigned char* stage = smem + Shape::kStages * Shape::kStage + (warp - 2) * 2048;
        float* const bias = reinterpret_cast<float*>(smem + Shape::kStages * Shape::kStage + Shape::kOut);
        T* const out = static_cast<T*>(p.out);
        const bool wide = p.out_stride * sizeof(T) % 32 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
        bool alive = true;
        int i = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++i) {
            const int half = i % Shape::kSums;
            const long long row0 = (long long)(tile % tiles_m) * kTileRows + quarter * 32;
            const int col0 = tile / tiles_m * BN + half_col;
            // the tile before last's are not in use any more: every warp has been past this barrier for the one between
            float* const bs = bias + (i & 1) * BN;
            if (p.bias)
                for (int c = thread; c < BN; c += 32 * kOutWarps) bs[c] = p.bias[min(tile / tiles_m * BN + c, p.cols - 1)];
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kOutWarps) : "memory");
            alive = alive && bar_wait_all(shared_address(&bars.done[half]), i / Shape::kSums & 1);
            tmem_fence_after();
            uint32_t words[kWords];                       // the row's outputs, two to a word for 16 bits
            {
                uint32_t r[kCols / 32][32];
#pragma unroll
                for (int b = 0; b < kCols / 32; ++b) tmem_load(tmem + half * BN + (quarter * 32 << 16) + half_col + b * 32, r[b]);
                tmem_load_wait();
                tmem_fence_before();
                bar_arrive(shared_address(&bars.taken[half]));
#pragma unroll
                for (int b = 0; b < kCols; b += 4) {
                    float f[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = alive ? __uint_as_float(r[b / 32][b % 32 + j]) : __int_as_float(0x7fffffff);
                    if (p.bias) {
                        const float4 d = *reinterpret_cast<const float4*>(bs + half_col + b);
                        f[0] += d.x;
                        f[1] += d.y;
                        f[2] += d.z;
                        f[3] += d.w;
                    }
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) words[b + j] = __float_as_uint(f[j]);
                    } else {
                        words[b / 2] = pack2<T>(f[0], f[1]);
                        words[b / 2 + 1] = pack2<T>(f[2], f[3]);
                    }
                }
            }
            if (wide && col0 + kCols <= p.cols) {
                // each lane its own row, whole sectors
                if (row0 + lane < p.rows) {
                    T* const to = out + (row0 + lane) * p.out_stride + col0;
#pragma unroll
                    for (int c = 0; c < kWords; c += 8)
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + c * 4 / (int)sizeof(T)), "r"(words[c]),
                                     "r"(words[c + 1]), "r"(words[c + 2]), "r"(words[c + 3]), "r"(words[c + 4]), "r"(words[c + 5]), "r"(words[c + 6]),
                                     "r"(words[c + 7])
                                     : "memory");
                }
            } else {
                // rows that do not start on 32 bytes, or end in this block: 64 bytes of them at a
                // time, value by value, a row's side by side, eight rows read before they are written
                constexpr int kSide = 64 / (int)sizeof(T);
#pragma unroll
                for (int c0 = 0; c0 < kCols; c0 += kSide) {
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int w = c0 * (int)sizeof(T) / 4 + 4 * q;
                        *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ (lane / 2 & 3)) << 4)) = make_uint4(words[w], words[w + 1], words[w + 2], words[w + 3]);
                    }
                    __syncwarp();
                    const int c = lane % kSide, at = c * (int)sizeof(T), col = col0 + c0 + c;
#pragma unroll
                    for (int r0 = 0; r0 < kSide; r0 += 8) {
                        T x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const int row = (r0 + k) * (32 / kSide) + lane / kSide;
                            x[k] = *reinterpret_cast<const T*>(stage + row * 64 + (((at >> 4) ^ (row / 2 & 3)) << 4) + (at & 15));
                        }
                        if (col < p.cols)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const long long row = row0 + (r0 + k) * (32 / kSide) + lane / kSide;
                                if (row < p.rows) out[row * p.out_stride + col] = x[k];
                            }
                    }
                }
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tmem_fence_after();
        tmem_free(tmem, Shape::kCols);
    }
}

template <typename T, int BN>
cudaError_t tiles_launch(const Fp4Params& p, bool after, cudaStream_t s) {
    using Shape = TileShape<BN>;
    CUtensorMap a, w;
    const int bytes = (p.inner + 1) / 2;
    if (!byte_rows_map(&a, p.a, p.rows, bytes, p.a_stride, kStepBytes, kTileRows) ||
        !byte_rows_map(&w, p.w, p.cols, bytes, p.w_stride, kStepBytes, BN))
        return cudaErrorInvalidValue;
    const cudaError_t e = allow_shared<k_fp4_tiles<T, BN>>(Shape::kBytes);
    if (e != cudaSuccess) return e;
    const long long tiles_m = (p.rows + kTileRows - 1) / kTileRows, tiles = tiles_m * ((p.cols + BN - 1) / BN);
    if (tiles > 0x7fffffff - 1024) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(tiles < kSmCount ? tiles : kSmCount));
    if (after) return launch_after(k_fp4_tiles<T, BN>, grid, dim3(kTileThreads), Shape::kBytes, s, a, w, p, (int)tiles_m, (int)tiles);
    k_fp4_tiles<T, BN><<<grid, kTileThreads, Shape::kBytes, s>>>(a, w, p, (int)tiles_m, (int)tiles);
    return cudaGetLastError();
}

// The width with the least rounds of CTAs, a tile's time taken as its width and 64 more (the same for each:
// the first stages, the outputs), so that wide tiles win unless the last round is much emptier than a
// narrower one's.  Of 44 shapes of 65 to 8192 rows, 258 to 8192 inner columns and 276 to 11008
// channels the width so chosen took 1.1% more than the best on average and 18% at worst; with 16
// to 192 in place of 64 as much, with 0 3.8% and twice the time.  us with 256, 192, 128 and 64 channels:
// 2048 x 4096 x 4096 18.6, 23.3, 24.9 and 38.0 (256 taken), 738 x 7699 x 3698 26.1, 23.4, 31.5 and 33.3 (192), 777
// x 1001 x 1531 10.2, 9.8, 7.5 and 8.8 (128), 1024 x 1024 x 1024 7.7, 7.9, 5.5 and 4.9 (64); the worst
// 3734 x 1761 x 2371 21.1, 22.0, 18.6 and 25.1 (192).
template <typename T>
cudaError_t tiles_by_width(const Fp4Params& p, bool after, cudaStream_t s) {
    const long long tiles_m = (p.rows + kTileRows - 1) / kTileRows;
    int best = 0;
    long long cost = 0;
    for (const int bn : {256, 192, 128, 64}) {
        const long long tiles = tiles_m * ((p.cols + bn - 1) / bn), c = (tiles + kSmCount - 1) / kSmCount * (bn + 64);
        if (!best || c < cost) {
            best = bn;
            cost = c;
        }
    }
    if (best == 256) return tiles_launch<T, 256>(p, after, s);
    if (best == 192) return tiles_launch<T, 192>(p, after, s);
    if (best == 128) return tiles_launch<T, 128>(p, after, s);
    return tiles_launch<T, 64>(p, after, s);
}

}  // namespace

cudaError_t launch_quantize_fp4(const void* x, int type, long long rows, int cols, long long x_stride, uint8_t* codes, long long codes_stride,
                                uint8_t* scale, cudaStream_t s) {
    if (type == VDT_F32) return pack_launch<float>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    if (type == VDT_F16) return pack_launch<__half>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    return pack_launch<__nv_bfloat16>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
}

cudaError_t launch_fp4_values(const uint8_t* codes, long long codes_stride, const uint8_t* scale, long long rows, int cols, int type, void* out,
                              long long out_stride, cudaStream_t s) {
    const long long blocks = (rows * ((cols + 7) / 8) + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 32 * kSmCount ? blocks : 32 * kSmCount);
    auto go = [&](auto* to) { k_fp4_values<<<grid, 256, 0, s>>>(codes, codes_stride, scale, rows, cols, to, out_stride, fp4_steps(cols)); };
    if (type == VDT_F32) go(static_cast<float*>(out));
    else if (type == VDT_F16) go(static_cast<__half*>(out));
    else go(static_cast<__nv_bfloat16*>(out));
    return cudaGetLastError();
}

bool fp4_rounds_itself(long long rows) { return rows <= kOwnRows; }

cudaError_t launch_fp4_own(const Fp4Params& p, int type, cudaStream_t s) {
    if (type == VDT_F32) return few_by_rows<float>(p, false, s);
    if (type == VDT_F16) return few_by_rows<__half>(p, false, s);
    return few_by_rows<__nv_bfloat16>(p, false, s);
}

cudaError_t launch_fp4_matmul(const Fp4Params& p, bool after_codes, cudaStream_t s) {
    const long long steps = fp4_steps(p.inner), split = few_split(p.cols, p.inner, 64);
    if (p.rows <= kOwnRows || (p.rows <= kFewRows && steps - steps / split > kFewSteps)) return few_by_rows<void>(p, after_codes, s);
    if (p.out_type == VDT_F32) return tiles_by_width<float>(p, after_codes, s);
    if (p.out_type == VDT_F16) return tiles_by_width<__half>(p, after_codes, s);
    return tiles_by_width<__nv_bfloat16>(p, after_codes, s);
}

}  // namespace vdt

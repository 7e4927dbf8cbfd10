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
// Reads every value once, writes a byte for it: bound by memory for many rows
// (8192 x 4096 bf16: 29 us, 3.5 TB/s; the floor is 16), by latency for few.
// One CTA a row: the largest magnitude, then the codes.  Rows of up to HELD
// vectors a thread are read once and stay in registers; longer ones, and rows
// that are not on 16 bytes (HELD 0), are read twice, the second time from L1
// and L2.  (A warp a row, without barriers, took 46 us for 8192 x 4096 bf16.)
template <typename T, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS) k_quantize_rows(const T* __restrict__ x, int cols,
                                                                 long long x_stride, int8_t* __restrict__ codes,
                                                                 long long codes_stride, float* __restrict__ scale) {
    constexpr int N = Vec16<T>::N;
    __shared__ float part[THREADS / 32];
    chain_release();
    const long long r = blockIdx.x;
    const int thread = threadIdx.x;
    const T* row = x + r * x_stride;
    int8_t* out = codes + r * codes_stride;
    const int vecs = HELD ? cols / N : 0;
    float m = 0.0f;
    Largest<T> most;
    Vec16<T> held[HELD ? HELD : 1];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int at = thread + i * THREADS;
        held[i].raw = at < vecs ? *reinterpret_cast<const uint4*>(row + (long long)at * N) : make_uint4(0, 0, 0, 0);
    }
    // single values: what is left of the vectors, or the whole row
    constexpr int kSingle = HELD ? 1 : 8;
    T single[kSingle];
#pragma unroll
    for (int i = 0; i < kSingle; ++i) {
        const int at = vecs * N + thread + i * THREADS;
        single[i] = at < cols ? row[at] : from_f32<T>(0.0f);
    }
    for (int i = vecs * N + thread + kSingle * THREADS; i < cols; i += THREADS) m = max_nan(fabsf(to_f32(row[i])), m);
#pragma unroll
    for (int i = 0; i < kSingle; ++i) m = max_nan(fabsf(to_f32(single[i])), m);
    for (int i = thread + HELD * THREADS; i < vecs; i += THREADS) {
        Vec16<T> v;
        v.raw = *reinterpret_cast<const uint4*>(row + (long long)i * N);
        most.add(v);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) most.add(held[i]);
    m = max_nan(most.value(), m);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max_nan(__shfl_xor_sync(0xffffffffu, m, d), m);
    if (thread % 32 == 0) part[thread / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) m = max_nan(part[i], m);
    const Coder coder(m * kCodeStep);
    if (thread == 0) scale[r] = coder.scale;
    auto store = [&](const Vec16<T>& v, int at) {
        float f[N];
        uint32_t w[N / 4];
        v.get(f);
        coder.words<N>(f, w);
        if constexpr (N == 8) *reinterpret_cast<uint2*>(out + (long long)at * N) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(out + (long long)at * N) = w[0];
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (thread + i * THREADS < vecs) store(held[i], thread + i * THREADS);
    for (int i = thread + HELD * THREADS; i < vecs; i += THREADS) {
        Vec16<T> v;
        v.raw = *reinterpret_cast<const uint4*>(row + (long long)i * N);
        store(v, i);
    }
    auto put = [&](T x, int at) {
        const float q = to_f32(x) * coder.inverse, n = rintf(q);
        out[at] = (int8_t)(coder.exact && fabsf(q - n) <= 0.5f - 1.0f / 32768 ? (int)n : code_of(to_f32(x), coder.scale));
    };
#pragma unroll
    for (int i = 0; i < kSingle; ++i)
        if (vecs * N + thread + i * THREADS < cols) put(single[i], vecs * N + thread + i * THREADS);
    for (int i = vecs * N + thread + kSingle * THREADS; i < cols; i += THREADS) put(row[i], i);
}

// ---------------------------------------------------------------- few rows
// Each warp takes 16 channels and a share of the inner dimension; mma
// m16n8k32 with the channels as its rows and 8 tokens as its columns.  The
// order of the inner dimension is free as long as both sides keep the same,
// so a lane takes 16 consecutive bytes of a row (one wide load) and feeds
// them to two products.  What bounds it is the weights' way from memory: 16
// channels a CTA and eight warps along the inner dimension put every SM to
// work for a few thousand channels, four steps of loads in flight a warp, the
// first before the codes are there.  24 x 4096 x 4096: 9.3 us with the rows'
// rounding (16.7 MB of weights, from L2 where they fit).
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

// Up to here the kernel for few rows, above it the tiles (us on the GPU, few rows
// and tiles): 32 x 4096 x 1024 9.3 and 11.2, 32 x 1024 x 4096 5.7 and 7.4, 64 x 4096 x
// 1024 10.1 and 11.2, 64 x 1024 x 4096 8.3 and 7.2, 40 x 4096 x 4096 18.3 and 11.7.  Wide
// layers turn earlier, 32 x 4096 x 4096 at 13.0 and 11.7, 20 x 4096 x 16384 at 36.9 and
// 21.4, narrow ones later.
constexpr int kFewRows = 32;

// One row of up to 16384 values, or two short ones, are rounded by every CTA for
// itself, into shared memory: one launch instead of two, 2 us of the host's.  The
// values are read from L2 by all CTAs, which wait for their rounding, so more of
// them cost more than the launch.  A call / on the GPU in us, so and with two
// launches: 1 x 1024 x 1024 5.4 / 3.1 and 7.7 / 4.5, 1 x 4096 x 4096 8.2 / 8.3 and
// 8.0 to 10.6 / 8.6, 1 x 16384 x 1024 14.4 / 15.5 and 14.8 / 19.3, 2 x 1024 x 1024
// 6.2 / 4.5 and 8.1 / 4.5; not taken: 2 x 4096 x 4096 10.2 / 10.8 and 8.3 / 9.3,
// 4 x 256 x 256 8.2 / 5.9 and 8.2 / 4.5, 4 x 4096 x 4096 12.9 / 13.6 and 8.3 / 9.4.
constexpr int kOwnRows = 2, kOwnValues = 16384, kOwnShort = 1024;

template <typename X>
__device__ __forceinline__ void round_rows(const Int8Params& p, int8_t* codes, float* scale) {
    constexpr int N = Vec16<X>::N, kThreads = kRowsWarps * 32;
    __shared__ float part[kOwnRows][kRowsWarps];
    const X* const x = static_cast<const X*>(p.x);
    const int stride = (p.inner + 15) / 16 * 16, rows = (int)p.rows;
    const bool wide = p.x_stride % N == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const int vecs = wide ? p.inner / N : 0;
    float m[kOwnRows] = {};
#pragma unroll
    for (int r = 0; r < kOwnRows; ++r) {
        if (r >= rows) break;
        const X* const row = x + r * p.x_stride;
        Largest<X> most;
        for (int i = threadIdx.x; i < vecs; i += kThreads) most.add(Vec16<X>{*reinterpret_cast<const uint4*>(row + i * N)});
        m[r] = most.value();
        for (int i = vecs * N + threadIdx.x; i < p.inner; i += kThreads) m[r] = max_nan(fabsf(to_f32(row[i])), m[r]);
#pragma unroll
        for (int d = 16; d; d >>= 1) m[r] = max_nan(__shfl_xor_sync(0xffffffffu, m[r], d), m[r]);
        if (threadIdx.x % 32 == 0) part[r][threadIdx.x / 32] = m[r];
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
        const X* const row = x + r * p.x_stride;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowsWarps; ++i) top = max_nan(part[r][i], top);
        const Coder coder(top * kCodeStep);
        if (threadIdx.x == 0) scale[r] = coder.scale;
        for (int i = threadIdx.x; i < vecs; i += kThreads) {
            Vec16<X> v;
            v.raw = *reinterpret_cast<const uint4*>(row + i * N);
            float f[N];
            uint32_t w[N / 4];
            v.get(f);
            coder.words<N>(f, w);
#pragma unroll
            for (int j = 0; j < N / 4; ++j) reinterpret_cast<uint32_t*>(codes + r * stride)[i * (N / 4) + j] = w[j];
        }
        for (int i = vecs * N + threadIdx.x; i < p.inner; i += kThreads) codes[r * stride + i] = (int8_t)code_of(to_f32(row[i]), coder.scale);
    }
    __syncthreads();
}

// X: the type of rows that are still to be rounded; void: they are codes
template <typename T, int NT, typename X = void>
__global__ void __launch_bounds__(kRowsWarps * 32) k_int8_rows(Int8Params p) {
    extern __shared__ __align__(16) int8_t own[];            // rows' codes, then their scales
    __shared__ int part[kRowsWarps][16][8 * NT + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int col0 = blockIdx.x * 16;
    const long long row0 = (long long)blockIdx.y * (8 * NT);
    int acc[NT][4] = {};
    // rows past the end read the last one; their products are not stored
    const int8_t* w0 = p.w + (long long)min(col0 + g, p.cols - 1) * p.w_stride;
    const int8_t* w1 = p.w + (long long)min(col0 + g + 8, p.cols - 1) * p.w_stride;
    const int8_t* a[NT];
    const float* a_scale = p.a_scale;
#pragma unroll
    for (int n = 0; n < NT; ++n) a[n] = p.a + min(row0 + 8 * n + g, p.rows - 1) * p.a_stride;
    const int steps = (p.inner + 63) / 64;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    constexpr int kDeep = NT == 4 ? 2 : 4;                   // steps in flight
    // a row's storage reaches to the next multiple of 16
    auto weights = [&](int s, uint4 (&u)[2]) {
        const bool in = s < steps && s * 64 + t * 16 < p.inner;
        u[0] = in ? __ldg(reinterpret_cast<const uint4*>(w0 + s * 64 + t * 16)) : zero;
        u[1] = in ? __ldg(reinterpret_cast<const uint4*>(w1 + s * 64 + t * 16)) : zero;
    };
    auto rows = [&](int s, uint4 (&b)[NT]) {
        const bool in = s < steps && s * 64 + t * 16 < p.inner;
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = in ? *reinterpret_cast<const uint4*>(a[n] + s * 64 + t * 16) : zero;
    };
    uint4 u[kDeep][2], x[kDeep][NT];
    // the weights are the caller's: their first loads need not wait for the codes
#pragma unroll
    for (int d = 0; d < kDeep; ++d) weights(warp + d * kRowsWarps, u[d]);
    chain_wait();
    if constexpr (!std::is_void_v<X>) {
        const int stride = (p.inner + 15) / 16 * 16;
        float* const scale = reinterpret_cast<float*>(own + p.rows * stride);
        round_rows<X>(p, own, scale);
        a_scale = scale;
        a[0] = own + min(g, (int)p.rows - 1) * stride;
    }
    for (int s0 = warp; s0 < steps; s0 += kDeep * kRowsWarps) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) rows(s0 + d * kRowsWarps, x[d]);
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const int s = s0 + d * kRowsWarps, k = s * 64 + t * 16;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint4 b = x[d][n];
                if (k + 16 > p.inner) {
                    b.x = keep_below(b.x, k / 4, p.inner);
                    b.y = keep_below(b.y, k / 4 + 1, p.inner);
                    b.z = keep_below(b.z, k / 4 + 2, p.inner);
                    b.w = keep_below(b.w, k / 4 + 3, p.inner);
                }
                mma_s8(acc[n], u[d][0].x, u[d][1].x, u[d][0].y, u[d][1].y, b.x, b.y);
                mma_s8(acc[n], u[d][0].z, u[d][1].z, u[d][0].w, u[d][1].w, b.z, b.w);
            }
            weights(s + kDeep * kRowsWarps, u[d]);
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
            float y = (float)sum * a_scale[row] * p.w_scale[col];
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

template <typename T, typename X>
cudaError_t own_launch(const Int8Params& p, cudaStream_t s) {
    const size_t bytes = (size_t)p.rows * ((p.inner + 15) / 16 * 16) + p.rows * sizeof(float);
    k_int8_rows<T, 1, X><<<(p.cols + 15) / 16, kRowsWarps * 32, bytes, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t own_by_type(const Int8Params& p, int type, cudaStream_t s) {
    if (type == VDT_F32) return own_launch<T, float>(p, s);
    if (type == VDT_F16) return own_launch<T, __half>(p, s);
    return own_launch<T, __nv_bfloat16>(p, s);
}

// --------------------------------------------------------------- many rows
// Persistent CTAs over tiles of 128 rows x BN channels.  One thread keeps a
// ring of stages (128 bytes of the inner dimension of both sides) full with
// tile loads, one issues the products into the tensor memory, four warps turn
// finished sums into outputs while the next tile's are made in the other half
// of the tensor memory.  Loads past the rows, the channels and the inner size
// give zeros.  A stage is 128 bytes because a swizzled row is; 256 channels a
// tile halve the reads of the rows' codes against 128.  8192 x 4096 x 8192:
// 169 us, 3.25 POP/s, bound by the tensor cores and, back to back, by power.
constexpr int kTileRows = 128, kStageBytes = 128;    // bytes of the inner dimension a stage
constexpr int kGemmThreads = 192;

template <int BN>
struct GemmShape {
    static constexpr int kStage = (kTileRows + BN) * kStageBytes;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kOut = 4 * 4096;                       // a 32-row, 128-byte block for each epilogue warp
    static constexpr int kScales = 2 * 2 * BN * 4;              // channel scales and biases of two tiles
    static constexpr int kBytes = 1024 + kStages * kStage + kOut + kScales;
};

struct GemmBars {
    uint64_t full[8], empty[8], done[2], taken[2];
    uint32_t tmem;
};

template <typename T, int BN>
__global__ void __launch_bounds__(kGemmThreads, 1) k_int8_tiles(const __grid_constant__ CUtensorMap map_a,
                                                                const __grid_constant__ CUtensorMap map_w, Int8Params p,
                                                                int tiles_m, int tiles) {
    using Shape = GemmShape<BN>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ GemmBars bars;
    unsigned char* smem = smem_raw + ((1024 - (shared_address(smem_raw) & 1023)) & 1023);
    const uint32_t stages = shared_address(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int steps = (p.inner + kStageBytes - 1) / kStageBytes;
    if (threadIdx.x == 0) {
        map_ahead(&map_w);
        map_ahead(&map_a);
        for (int i = 0; i < Shape::kStages; ++i) {
            bar_init(shared_address(&bars.full[i]), 1);
            bar_init(shared_address(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(shared_address(&bars.done[i]), 1);
            bar_init(shared_address(&bars.taken[i]), 128);
        }
        bar_init_done();
    }
    if (warp == 1) tmem_alloc(shared_address(&bars.tmem), 2 * BN);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = bars.tmem;
    // the weights are the caller's: the first stages' need not wait for the codes
    const int ahead = min(steps, Shape::kStages);
    if (threadIdx.x == 0)
        for (int s = 0; s < ahead; ++s) {
            const uint32_t bar = shared_address(&bars.full[s]);
            bar_expect(bar, Shape::kStage);
            tile_load(stages + s * Shape::kStage + kTileRows * kStageBytes, &map_w, s * kStageBytes, blockIdx.x / tiles_m * BN, bar);
        }
    chain_wait();

    if (warp == 0) {
        if (lane == 0) {
            int n = 0;
            bool alive = true;
            for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
                const int y = tile % tiles_m * kTileRows, c = tile / tiles_m * BN;
                for (int s = 0; s < steps; ++s, ++n) {
                    const int slot = n % Shape::kStages;
                    const uint32_t at = stages + slot * Shape::kStage, bar = shared_address(&bars.full[slot]);
                    if (n >= ahead) {
                        if (!(alive = bar_wait(shared_address(&bars.empty[slot]), (n / Shape::kStages & 1) ^ 1))) break;
                        bar_expect(bar, Shape::kStage);
                        tile_load(at + kTileRows * kStageBytes, &map_w, s * kStageBytes, c, bar);
                    }
                    tile_load(at, &map_a, s * kStageBytes, y, bar);
                }
            }
            // every load has landed before the CTA ends: the last ones' stages
            for (int i = max(0, n - Shape::kStages); i < n; ++i)
                bar_wait(shared_address(&bars.full[i % Shape::kStages]), i / Shape::kStages & 1);
        }
    } else if (warp == 1) {
        // 32-bit sums, signed 8-bit operands, both with the inner dimension consecutive
        constexpr uint32_t shape = 2u << 4 | 1u << 7 | 1u << 10 | (BN >> 3) << 17 | (kTileRows >> 4) << 24;
        const uint32_t sums = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t a = tile_desc(stages), w = tile_desc(stages + kTileRows * kStageBytes);
        const bool one = elected();
        int n = 0, i = 0;
        bool alive = true;
        for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x, ++i) {
            const int half = i & 1;
            if (!(alive = bar_wait_all(shared_address(&bars.taken[half]), (i / 2 & 1) ^ 1))) break;
            tmem_fence_after();
            for (int s = 0; s < steps; ++s, ++n) {
                const int slot = n % Shape::kStages;
                if (!(alive = bar_wait_all(shared_address(&bars.full[slot]), n / Shape::kStages & 1))) break;
                tmem_fence_after();
                if (one) {
#pragma unroll
                    for (int k = 0; k < kStageBytes / 32; ++k)
                        mma_i8(sums + half * BN, a + (slot * Shape::kStage + k * 32) / 16, w + (slot * Shape::kStage + k * 32) / 16, shape,
                               s > 0 || k > 0);
                    mma_commit(shared_address(&bars.empty[slot]));
                }
            }
            if (alive && one) mma_commit(shared_address(&bars.done[half]));
        }
    } else {
        const int quarter = warp % 4, thread = threadIdx.x - 64;     // a warp reads the rows of its quarter
        unsigned char* stage = smem + Shape::kStages * Shape::kStage + (warp - 2) * 4096;
        float* const scales = reinterpret_cast<float*>(smem + Shape::kStages * Shape::kStage + Shape::kOut);
        T* const out = static_cast<T*>(p.out);
        constexpr int kPer = 16 / sizeof(T), kCols = 8 * kPer < BN ? 8 * kPer : BN;   // columns of 16 bytes; of a block
        constexpr int kPieces = kCols / kPer;                         // 16-byte pieces of a block's row
        const bool wide = p.out_stride * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
        bool alive = true;
        int i = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++i) {
            const int half = i & 1;
            const long long row0 = (long long)(tile % tiles_m) * kTileRows + quarter * 32;
            const int col0 = tile / tiles_m * BN;
            float* const ws = scales + half * 2 * BN;
            // the scales of the tile before last are not in use any more: every
            // warp has been past this barrier for the tile between
            for (int c = thread; c < BN; c += 128) {
                const int col = min(col0 + c, p.cols - 1);
                ws[c] = p.w_scale[col];
                ws[BN + c] = p.bias ? p.bias[col] : 0.0f;
            }
            const float as = p.a_scale[min(row0 + lane, p.rows - 1)];
            asm volatile("bar.sync 1, 128;" ::: "memory");
            alive = alive && bar_wait_all(shared_address(&bars.done[half]), i / 2 & 1);
            tmem_fence_after();
#pragma unroll
            for (int b = 0; b < BN / kCols; ++b) {
#pragma unroll
                for (int part = 0; part < kCols / 32; ++part) {
                    uint32_t r[32];
                    tmem_load(tmem + half * BN + (quarter * 32 << 16) + b * kCols + part * 32, r);
                    tmem_load_wait();
#pragma unroll
                    for (int q = 0; q < 32 / kPer; ++q) {
                        float f[kPer];
                        const int c = b * kCols + part * 32 + q * kPer;
#pragma unroll
                        for (int j = 0; j < kPer; j += 4) {
                            const float4 w = *reinterpret_cast<const float4*>(ws + c + j);
                            const float4 d = *reinterpret_cast<const float4*>(ws + BN + c + j);
                            f[j] = fmaf((float)(int)r[q * kPer + j] * as, w.x, d.x);
                            f[j + 1] = fmaf((float)(int)r[q * kPer + j + 1] * as, w.y, d.y);
                            f[j + 2] = fmaf((float)(int)r[q * kPer + j + 2] * as, w.z, d.z);
                            f[j + 3] = fmaf((float)(int)r[q * kPer + j + 3] * as, w.w, d.w);
                        }
                        if (!alive)
#pragma unroll
                            for (int j = 0; j < kPer; ++j) f[j] = __int_as_float(0x7fffffff);
                        Vec16<T> v;
                        v.set(f);
                        const int chunk = part * (32 / kPer) + q;
                        *reinterpret_cast<uint4*>(stage + lane * 128 + ((chunk ^ (lane & (kPieces - 1))) << 4)) = v.raw;
                    }
                }
                __syncwarp();
                const int col1 = col0 + b * kCols;
                if (wide && col1 + kCols <= p.cols) {
                    // kPieces lanes write a row's bytes
#pragma unroll
                    for (int k = 0; k < kPieces; ++k) {
                        const int r = k * (32 / kPieces) + lane / kPieces, c = lane % kPieces;
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & (kPieces - 1))) << 4));
                        if (row0 + r < p.rows) *reinterpret_cast<uint4*>(out + (row0 + r) * p.out_stride + col1 + c * kPer) = v;
                    }
                } else {
                    // rows that do not start on 16 bytes, or end in this block:
                    // value by value, eight rows read before they are written
                    T* to = out + row0 * p.out_stride + col1;
                    for (int r0 = 0; r0 < 32; r0 += 8, to += 8 * p.out_stride)
#pragma unroll
                        for (int c0 = 0; c0 < kCols; c0 += 32) {
                            const int c = c0 + lane, at = c * (int)sizeof(T);
                            T x[8];
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                x[r] = *reinterpret_cast<const T*>(stage + (r0 + r) * 128 + (((at >> 4) ^ (r & (kPieces - 1))) << 4) + (at & 15));
                            if (col1 + c < p.cols)
#pragma unroll
                                for (int r = 0; r < 8; ++r)
                                    if (row0 + r0 + r < p.rows) to[r * p.out_stride + c] = x[r];
                        }
                }
                __syncwarp();
            }
            tmem_fence_before();
            bar_arrive(shared_address(&bars.taken[half]));
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tmem_fence_after();
        tmem_free(tmem, 2 * BN);
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, reached through the runtime (the library links the
// runtime only); asked for again after a call that did not get it
EncodeTiled encode_tiled() {
    static std::atomic<void*> found{nullptr};
    void* f = found.load(std::memory_order_relaxed);
    if (!f) {
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        found.store(f, std::memory_order_relaxed);
    }
    return reinterpret_cast<EncodeTiled>(f);
}

bool byte_map(CUtensorMap* m, const int8_t* at, long long rows, int inner, long long stride, int box_rows) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {kStageBytes, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(at), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int BN>
cudaError_t tiles_launch(const Int8Params& p, bool after, cudaStream_t s) {
    using Shape = GemmShape<BN>;
    CUtensorMap a, w;
    if (!byte_map(&a, p.a, p.rows, p.inner, p.a_stride, kTileRows) || !byte_map(&w, p.w, p.cols, p.inner, p.w_stride, BN))
        return cudaErrorInvalidValue;
    const cudaError_t e = allow_shared<k_int8_tiles<T, BN>>(Shape::kBytes);
    if (e != cudaSuccess) return e;
    const long long tiles_m = (p.rows + kTileRows - 1) / kTileRows, tiles = tiles_m * ((p.cols + BN - 1) / BN);
    if (tiles > 0x7fffffff - 1024) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(tiles < kSmCount ? tiles : kSmCount));
    if (after)
        return launch_after(k_int8_tiles<T, BN>, grid, dim3(kGemmThreads), Shape::kBytes, s, a, w, p, (int)tiles_m, (int)tiles);
    k_int8_tiles<T, BN><<<grid, kGemmThreads, Shape::kBytes, s>>>(a, w, p, (int)tiles_m, (int)tiles);
    return cudaGetLastError();
}

// The widest tile whose last round of CTAs is not much emptier than a narrower
// one's: rounds times (channels + 64), the 64 for what a tile costs by itself.
// With 0, 64, 128 for it, us: 777 x 4096 x 4096 52.0, 20.9, 20.8; 1500 x 4096 x 4096 80.1,
// 31.4, 33.9; 4000 x 1001 x 1531 35.7, 24.5, 29.3; 4000 x 1024 x 4096 27.7, 29.1, 29.1;
// 777 x 1001 x 1531 14.8, 13.0, 12.4.
template <typename T>
cudaError_t tiles_by_width(const Int8Params& p, bool after, cudaStream_t s) {
    const long long tiles_m = (p.rows + kTileRows - 1) / kTileRows;
    int best = 0;
    long long cost = 0;
    for (const int bn : {256, 128, 64, 32}) {
        const long long tiles = tiles_m * ((p.cols + bn - 1) / bn), c = (tiles + kSmCount - 1) / kSmCount * (bn + 64);
        if (!best || c < cost) {
            best = bn;
            cost = c;
        }
    }
    if (best == 256) return tiles_launch<T, 256>(p, after, s);
    if (best == 128) return tiles_launch<T, 128>(p, after, s);
    if (best == 64) return tiles_launch<T, 64>(p, after, s);
    return tiles_launch<T, 32>(p, after, s);
}

template <typename T>
cudaError_t quant_launch(const void* x, long long rows, int cols, long long x_stride, int8_t* codes,
                         long long codes_stride, float* scale, cudaStream_t s) {
    constexpr int N = Vec16<T>::N;
    const bool vec = aligned(x, 16) && (x_stride * (long long)sizeof(T)) % 16 == 0 && aligned(codes, N) &&
                     codes_stride % N == 0;
    const T* in = static_cast<const T*>(x);
    // many rows: 128 threads each, so that more rows are under way (8192 x 4096
    // bf16: 29 us against 33 with 256); few: 256, for the latency
    auto go = [&](auto threads) {
        constexpr int kThreads = threads();
        const int each = (cols / N + kThreads - 1) / kThreads;             // vectors a thread
        auto kern = !vec        ? k_quantize_rows<T, 0, kThreads>
                    : each <= 1 ? k_quantize_rows<T, 1, kThreads>
                    : each <= 2 ? k_quantize_rows<T, 2, kThreads>
                    : each <= 4 ? k_quantize_rows<T, 4, kThreads>
                                : k_quantize_rows<T, 8, kThreads>;
        kern<<<(unsigned)rows, kThreads, 0, s>>>(in, cols, x_stride, codes, codes_stride, scale);
    };
    if (rows >= 8 * kSmCount) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int type, long long rows, int cols, long long x_stride,
                                 int8_t* codes, long long codes_stride, float* scale, cudaStream_t s) {
    if (type == VDT_F32) return quant_launch<float>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    if (type == VDT_F16) return quant_launch<__half>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
    return quant_launch<__nv_bfloat16>(x, rows, cols, x_stride, codes, codes_stride, scale, s);
}

bool int8_rounds_itself(long long rows, int inner) { return inner <= (rows == 1 ? kOwnValues : kOwnShort) && rows <= kOwnRows; }

cudaError_t launch_int8_own(const Int8Params& p, int type, cudaStream_t s) {
    if (p.out_type == VDT_F32) return own_by_type<float>(p, type, s);
    if (p.out_type == VDT_F16) return own_by_type<__half>(p, type, s);
    return own_by_type<__nv_bfloat16>(p, type, s);
}

cudaError_t launch_int8_matmul(const Int8Params& p, bool after_codes, cudaStream_t s) {
    const bool few = p.rows <= kFewRows;
    if (p.out_type == VDT_F32) return few ? rows_launch<float>(p, after_codes, s) : tiles_by_width<float>(p, after_codes, s);
    if (p.out_type == VDT_F16) return few ? rows_launch<__half>(p, after_codes, s) : tiles_by_width<__half>(p, after_codes, s);
    return few ? rows_launch<__nv_bfloat16>(p, after_codes, s) : tiles_by_width<__nv_bfloat16>(p, after_codes, s);
}

}  // namespace vdt

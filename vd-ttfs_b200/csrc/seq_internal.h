// seq_internal.h -- declarations shared by the sequence operators' kernel
// files (k_int8.cu, k_rope.cu, k_cache.cu, k_attend.cu) and their entry
// points (seq.cu); not part of the public ABI.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "vdt_internal.h"

namespace vdt {

constexpr int kSmCount = 148;
// scale = largest magnitude * kCodeStep; the codes run from -127 to 127
constexpr float kCodeStep = 1.0f / 127.0f;

inline bool type_ok(int t) { return t == VDT_F32 || t == VDT_F16 || t == VDT_BF16; }
inline int type_size(int t) { return t == VDT_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two 16-bit values of a word as 32-bit ones, and back
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    } else {
        __half2 h;
        memcpy(&h, &w, 4);
        const float2 f = __half22float2(h);
        lo = f.x;
        hi = f.y;
    }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t w;
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        memcpy(&w, &h, 4);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        memcpy(&w, &h, 4);
    }
    return w;
}

// 16 bytes of T as 32-bit values, and back
template <typename T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void get(float* f) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(w[i]);
            else unpack2<T>(w[i], f[2 * i], f[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void set(const float* f) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
            else w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Two independent 32-bit multiplications, or multiply-adds
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// The larger of two magnitudes; NaN wins, so that a row with a NaN gets a NaN scale
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }

// The largest magnitude of many values: magnitudes order as their bits do, NaN
// above infinity.  16-bit values two to a word.
template <typename T>
struct Largest {
    uint32_t bits = 0;
    __device__ __forceinline__ void add(const Vec16<T>& v) {
        const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) bits = max(bits, w[i] & 0x7fffffffu);
            else bits = __vmaxu2(bits, w[i] & 0x7fff7fffu);
        }
    }
    __device__ __forceinline__ float value() const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(bits);
        } else {
            float lo, hi;
            unpack2<T>(bits, lo, hi);
            return max_nan(lo, hi);
        }
    }
};

// One value's code: x / scale rounded to the nearest whole number, ties to
// even (the division is the IEEE one: a host that restates it gets the same
// codes).  A scale of 0 (nothing but zeros, or values below the smallest
// scale) leaves the value undivided, which rounds to 0; NaN rounds to 0.
static __device__ __noinline__ int code_of(float x, float scale) {
    const float q = rintf(__fdiv_rn(x, scale > 0.0f ? scale : 1.0f));
    return q != q ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// The codes of values under one scale.  x / scale and x * (1 / scale) differ by
// less than 2^-15 (three roundings of numbers up to 128), so they round to the
// same code unless the product is that near to the middle between two; then,
// and for scales whose reciprocal is not a normal number, the division decides.
struct Coder {
    float scale, inverse;
    bool exact;          // 1 / scale is of use
    __device__ __forceinline__ explicit Coder(float s) : scale(s), inverse(1.0f / s), exact(s > 1e-37f && s < 1e37f) {}
    template <int N>
    __device__ __forceinline__ void words(const float* f, uint32_t* w) const {
        // 1.5 * 2^23 added: the nearest whole number, ties to even, in the low bits
        const float2 round = make_float2(12582912.0f, 12582912.0f), by = make_float2(inverse, inverse);
        float near = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float2 x = make_float2(f[j + i], f[j + i + 1]), r = fma2(x, by, round);
                const float2 n = add2(r, make_float2(-round.x, -round.y)), off = fma2(x, by, make_float2(-n.x, -n.y));
                near = fmaxf(near, fmaxf(fabsf(off.x), fabsf(off.y)));
                c[i] = __float_as_uint(r.x);
                c[i + 1] = __float_as_uint(r.y);
            }
            w[j / 4] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        }
        if (!exact || near > 0.5f - 1.0f / 32768) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                w[j / 4] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[j / 4] |= (uint32_t)(code_of(f[j + i], scale) & 255) << (8 * i);
            }
        }
    }
};

// Four codes of a word, or of one byte of four words, as 32-bit values times a
// scale: code + 128 in the low bits of 2^23, less 2^23 + 128.
__device__ __forceinline__ float2 code_pair(uint32_t lo, uint32_t hi, float scale) {
    const float2 x = add2(make_float2(__uint_as_float(lo), __uint_as_float(hi)), make_float2(-8388736.0f, -8388736.0f));
    return mul2(x, make_float2(scale, scale));
}
__device__ __forceinline__ uint32_t code_byte(uint32_t w, int i) { return __byte_perm(w, 0x4b000000u, 0x7440 | i); }   // w with its signs flipped

// A launch that may start while the kernel before it on the stream ends; the
// kernel calls chain_wait() before it reads what that one wrote.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_after(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Lets a kernel have up to `bytes` of dynamic shared memory, once for each device.
template <auto Kernel>
inline cudaError_t allow_shared(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// ------------------------------------------------- copies into shared memory
// (mbarriers and bulk copies; the waits are bounded)
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void bar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// Every wait ends: after kWaitTries tries (each suspends for about a
// microsecond at most) it gives up and returns false; the kernel then writes
// NaN in the place of what it could not compute.
constexpr int kWaitTries = 1 << 18;
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < kWaitTries; ++i)
        if (bar_test(bar, parity)) return true;
    return false;
}
// the same for a whole warp, which goes on or gives up together
__device__ __forceinline__ bool bar_wait_all(uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, bar_wait(bar, parity));
}
// size and both addresses multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ void map_ahead(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// a two-dimensional box through a tensor map; x counts values, and x times the
// value's size is a multiple of 16 bytes
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// ---------------------------------------------------- fifth-generation tensor cores
// A tile in shared memory, rows of 128 bytes swizzled over 1024 (eight rows)
__device__ __forceinline__ uint64_t tile_desc(uint32_t at) {
    return (uint64_t)((at & 0x3ffff) >> 4) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// True in one lane of the warp.  The products are issued under it, in loops
// that the whole warp runs: their operands then stay in uniform registers
// (issued under `lane == 0`, a product took some 190 cycles to issue).
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// arrives on the barrier once every product issued by this thread is done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
        : "memory");
}
// 32 columns of this warp's 32 rows, a row a lane
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------ 8-bit integer product
cudaError_t launch_quantize_rows(const void* x, int type, long long rows, int cols, long long x_stride,
                                 int8_t* codes, long long codes_stride, float* scale, cudaStream_t s);

struct Int8Params {
    const int8_t* a;        // [rows, inner] codes, rows a_stride bytes apart
    const float* a_scale;   // [rows]
    const int8_t* w;        // [cols, inner] codes, rows w_stride bytes apart
    const float* w_scale;   // [cols]
    const float* bias;      // [cols] or null
    void* out;              // [rows, cols], rows out_stride values apart
    long long rows, a_stride, w_stride, out_stride;
    int cols, inner, out_type;
    const void* x;          // launch_int8_own: the rows, x_stride values apart, instead of a and a_scale
    long long x_stride;
};
// one or two rows that the product's kernel rounds itself
bool int8_rounds_itself(long long rows, int inner);
cudaError_t launch_int8_own(const Int8Params& p, int type, cudaStream_t s);
// after_codes: the kernel before it on the stream is the one that writes `a`
cudaError_t launch_int8_matmul(const Int8Params& p, bool after_codes, cudaStream_t s);

// ---------------------------------------------------- head norms and rotation
struct RopeParams {
    const void *q, *k;                  // [tokens, heads, dim]
    void *q_out, *k_out;
    long long q_token, q_head, k_token, k_head;          // strides in values
    long long qo_token, qo_head, ko_token, ko_head;
    const void *wq, *wk;                // [dim] or null
    const int32_t* at;                  // [tokens] positions
    const float* table;                 // [positions, rot]: cosines, then sines
    long long tokens;
    int positions, rot, layout, norm, heads, kv_heads, dim, type;
    float eps, share;                   // share: 1 / dim for the mean of the squares, 1 for their sum
};
cudaError_t launch_qk_norm_rope(const RopeParams& p, cudaStream_t s);

struct TableParams {
    int positions, rot, scaling;
    double base, factor;                // base: VDT_SCALE_BASE's factor is in it
    double low, high;                   // VDT_SCALE_PARTS: the ramp's ends, in i
    float* table;
};
cudaError_t launch_rope_table(const TableParams& p, cudaStream_t s);

// ------------------------------------------------------------------ the cache
struct CacheRows {
    const int32_t* table;   // [seqs, width] page numbers
    const int32_t* held;    // [seqs] tokens in the cache (before an append)
    const int32_t* starts;  // [seqs + 1] first packed row of each sequence
    int seqs, width;
    long long total;        // packed rows
    int most;               // longest run of packed rows
};
cudaError_t launch_cache_append(const vdt_cache8& c, const CacheRows& r, const void* k, const void* v, int type,
                                long long k_token, long long k_head, long long v_token, long long v_head,
                                cudaStream_t s);
cudaError_t launch_cache_load(const vdt_cache8& c, const CacheRows& r, void* k, void* v, int type, cudaStream_t s);

struct AttendParams {
    vdt_cache8 c;
    CacheRows r;            // r.held: tokens in the cache; r.most: longest run of queries
    const void* q;          // [total, heads, dim]
    void* out;              // [total, heads, dim]
    long long q_token, q_head, out_token, out_head;
    int heads, type, causal, most_kept;
    float scale;            // of the scores, times log2(e)
    float* scratch;
};
size_t attend_scratch_bytes(long long total, int heads, int kv_heads, int dim, int seqs, int most, int most_kept);
bool attend_dim_ok(int dim);
bool attend_fits(int dim, int heads, int kv_heads, int most);
cudaError_t launch_cache_attention(const AttendParams& p, cudaStream_t s);

}  // namespace vdt

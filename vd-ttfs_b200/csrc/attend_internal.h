// attend_internal.h -- what the two attention kernels (k_attend.cu for few
// query rows, k_attend_tiles.cu for many) share.
#pragma once

#include "seq_internal.h"

namespace vdt {

// How the cached tokens are divided among CTAs
struct Chunks {
    int tokens, count;             // of one chunk; chunks
};

// A sequence's queries; none where the caller's offsets do not fit the buffers.
struct Queries {
    long long first;
    int rows;            // queries
    int kept;            // tokens in the cache; -1: more than the table or most_kept allow
};
__device__ __forceinline__ Queries queries_of(const AttendParams& p, int b) {
    Queries s;
    s.first = p.r.starts[b];
    const long long rows = (long long)p.r.starts[b + 1] - s.first;
    s.rows = rows > 0 && rows <= p.r.most && s.first >= 0 && s.first + rows <= p.r.total ? (int)rows : 0;
    const int kept = p.r.held[b];
    s.kept = kept > p.most_kept || (long long)kept > (long long)p.r.width * p.c.page ? -1 : max(kept, 0);
    return s;
}

// Four codes as two pairs of 16-bit floats: code + 128 in the low bits of
// 1024's significand, less 1152.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));   // 1152
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hsub2(x, bias);
    y = __hsub2(y, bias);
    memcpy(&lo, &x, 4);
    memcpy(&hi, &y, 4);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ float inf_f() { return __int_as_float(0x7f800000); }

// values of the queries' and the output's type (f16 or bf16)
__device__ __forceinline__ float load_value(const void* p, long long i, int type) {
    return type == VDT_F16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_value(void* p, long long i, int type, float x) {
    if (type == VDT_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// A run of queries that does not fit the buffers or `most` is not computed: NaN
// to those of its rows that there are, for the heads that share head h of the
// cache.  All threads of one CTA.  Out of line, and given single values: a
// reference to the kernel's parameters would put all of them on the stack (7%
// of the kernels' time).
static __device__ __noinline__ void spoil_rows(void* out, int type, long long token, long long head, long long first, long long end, int head0,
                                               int group, int dim) {
    for (long long i = threadIdx.x; i < (end - first) * group * dim; i += blockDim.x) {
        const int at = (int)(i % (group * dim));
        store_value(out, (first + i / (group * dim)) * token + (head0 + at / dim) * head + at % dim, type, nan_f());
    }
}
__device__ __forceinline__ void spoil_run(const AttendParams& p, int b, int h) {
    const long long first = max((long long)p.r.starts[b], 0LL), end = min((long long)p.r.starts[b + 1], p.r.total);
    const int group = p.heads / p.c.heads;
    spoil_rows(p.out, p.type, p.out_token, p.out_head, first, end, h * group, group, p.c.dim);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Where the tokens are divided, a row and head's chunk leaves its maximum and
// sum and its unscaled output: first all rows' and chunks' pairs, then (on 16
// bytes) all outputs.
struct Partial {
    float2* stats;
    float* sums;
};
__host__ __device__ inline long long partial_pairs(long long rows, int count) { return (rows * count + 1) / 2 * 4; }
__host__ __device__ inline long long partial_floats(long long rows, int count, int dim) {
    return partial_pairs(rows, count) + rows * count * dim;
}
__device__ __forceinline__ Partial partial_of(const AttendParams& p, long long row, int count, int chunk) {
    const long long i = row * count + chunk;
    return {reinterpret_cast<float2*>(p.scratch) + i, p.scratch + partial_pairs(p.r.total * p.heads, count) + i * p.c.dim};
}

// What a row's running sums are relative to, in powers of two: 2^ref the
// weights' sum, 2^(ref + vref) the outputs.  Both references follow what the
// row itself sees: its largest score, and its largest score with the page's
// value scale.  By how much one may be passed before both are taken anew:
constexpr float kSlack = 8.0f, kSlackFactor = 256.0f;
__device__ __forceinline__ bool passes(float x, float ref) { return x > ref + kSlack; }        // also what is above a ref of -inf

// The references for new maxima, and the factors of the sums so far
struct Rescale {
    float sum, out;
};
__device__ __forceinline__ Rescale move_references(float top, float v_top, float& ref, float& vref) {
    const float to = fmaxf(top, ref);
    const float v_to = fmaxf(v_top, vref == -inf_f() ? vref : ref + vref);
    const float v = v_to == -inf_f() ? v_to : v_to - to;
    Rescale by;
    by.sum = ref == -inf_f() ? 0.0f : exp2f(ref - to);
    by.out = vref == -inf_f() ? 0.0f : exp2f((ref - to) + (vref - v));
    ref = to;
    vref = v;
    return by;
}
// A page's value scale over that of the row's references, as the power of two
// that its weights take with them and their sum gives back.  Not under 2^-100:
// a page of zeros still has weights.
__device__ __forceinline__ float page_shift(float v_log, float vref) {
    const float d = v_log - (vref == -inf_f() ? 0.0f : vref);
    return d < -100.0f ? -100.0f : d;
}

// many query rows: one CTA for up to 256 rows (k_attend_tiles.cu)
Chunks plan_tiles(int dim, int heads, int kv_heads, int seqs, int most, int most_kept);
int tile_rows(int dim, long long rows);          // rows of a CTA
cudaError_t launch_attend_tiles(const AttendParams& p, const Chunks& c, cudaStream_t s);

}  // namespace vdt

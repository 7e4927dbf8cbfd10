// k_rope.cu -- the norm of each head of the queries and keys, and the position
// rotation, in one pass.
//
//   y = x * w / sqrt(mean(x^2) + eps)         (VDT_NORM_RMS)
//   y = x * w / sqrt(sum(x^2) + eps)          (VDT_NORM_L2)
//   (a, b) -> (a cos - b sin, b cos + a sin)  for the pairs of the first `rot` values
//
// VDT_ROPE_HALF pairs value i with i + rot / 2, VDT_ROPE_PAIRS 2i with 2i + 1.
// Everything between the load and the store is 32-bit.
#include "seq_internal.h"

namespace vdt {
namespace {

constexpr int kRopeWarps = 4;

struct RopeRow {
    const void* in;
    void* out;
    const void* w;
};

// head h of a token: the queries first, then the keys
template <typename T>
__device__ __forceinline__ RopeRow rope_row(const RopeParams& p, long long token, int h) {
    RopeRow r;
    if (h < p.heads) {
        r.in = static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head;
        r.out = static_cast<T*>(p.q_out) + token * p.qo_token + h * p.qo_head;
        r.w = p.wq;
    } else {
        h -= p.heads;
        r.in = static_cast<const T*>(p.k) + token * p.k_token + h * p.k_head;
        r.out = static_cast<T*>(p.k_out) + token * p.ko_token + h * p.ko_head;
        r.w = p.wk;
    }
    return r;
}

__device__ __forceinline__ float norm_factor(float squares, const RopeParams& p) {
    if (p.norm == VDT_NORM_NONE) return 1.0f;
    return rsqrtf((p.norm == VDT_NORM_RMS ? squares / (float)p.dim : squares) + p.eps);
}

// Any size, stride and alignment: a warp a row, a lane a pair at a time.
template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) k_rope_any(RopeParams p) {
    const int lane = threadIdx.x % 32, all = p.heads + p.kv_heads, half = p.rot / 2;
    const long long rows = p.tokens * all;
    for (long long i = (long long)blockIdx.x * kRopeWarps + threadIdx.x / 32; i < rows;
         i += (long long)gridDim.x * kRopeWarps) {
        const long long token = i / all;
        const RopeRow r = rope_row<T>(p, token, (int)(i - token * all));
        const T* in = static_cast<const T*>(r.in);
        const T* w = static_cast<const T*>(r.w);
        T* out = static_cast<T*>(r.out);
        float sq = 0.0f;
        for (int d = lane; d < p.dim; d += 32) {
            const float x = to_f32(in[d]);
            sq = fmaf(x, x, sq);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
        float f = norm_factor(sq, p);
        const int at = p.rot ? p.at[token] : 0;
        const bool known = !p.rot || (at >= 0 && at < p.positions);
        if (!known) f = __int_as_float(0x7fffffff);      // a position outside the table: NaN
        const float* cs = p.table + (long long)(known ? at : 0) * p.rot;
        for (int j = lane; j < half; j += 32) {
            const int da = p.layout == VDT_ROPE_HALF ? j : 2 * j, db = p.layout == VDT_ROPE_HALF ? j + half : 2 * j + 1;
            const float a = to_f32(in[da]) * f * (w ? to_f32(w[da]) : 1.0f);
            const float b = to_f32(in[db]) * f * (w ? to_f32(w[db]) : 1.0f);
            const float c = cs[j], s = cs[half + j];
            out[da] = from_f32<T>(a * c - b * s);
            out[db] = from_f32<T>(b * c + a * s);
        }
        for (int d = p.rot + lane; d < p.dim; d += 32)
            out[d] = from_f32<T>(to_f32(in[d]) * f * (w ? to_f32(w[d]) : 1.0f));
    }
}

// One thread an angle, in 64 bits (built once for a model).
__global__ void k_rope_table(TableParams p) {
    const int half = p.rot / 2;
    const long long n = (long long)p.positions * half;
    const double magnitude = p.scaling == VDT_SCALE_PARTS ? 0.1 * log(p.factor) + 1.0 : 1.0;
    for (long long j = (long long)blockIdx.x * blockDim.x + threadIdx.x; j < n; j += (long long)gridDim.x * blockDim.x) {
        const long long t = j / half;
        const int i = (int)(j - t * half);
        double f = pow(p.base, -2.0 * i / p.rot);
        if (p.scaling == VDT_SCALE_LINEAR) f /= p.factor;
        if (p.scaling == VDT_SCALE_PARTS) {
            const double ramp = fmin(fmax((i - p.low) / fmax(p.high - p.low, 1e-3), 0.0), 1.0);
            f = f / p.factor * ramp + f * (1.0 - ramp);
        }
        double s, c;
        sincos((double)t * f, &s, &c);
        p.table[t * p.rot + i] = (float)(c * magnitude);
        p.table[t * p.rot + half + i] = (float)(s * magnitude);
    }
}

}  // namespace

cudaError_t launch_rope_table(const TableParams& p, cudaStream_t s) {
    const long long want = ((long long)p.positions * (p.rot / 2) + 127) / 128;
    k_rope_table<<<(unsigned)(want < kSmCount * 16 ? want : kSmCount * 16), 128, 0, s>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_qk_norm_rope(const RopeParams& p, cudaStream_t s) {
    const long long rows = p.tokens * (p.heads + p.kv_heads);
    const long long want = (rows + kRopeWarps - 1) / kRopeWarps;
    const unsigned grid = (unsigned)(want < kSmCount * 16 ? want : kSmCount * 16);
    if (p.type == VDT_F32) k_rope_any<float><<<grid, kRopeWarps * 32, 0, s>>>(p);
    else if (p.type == VDT_F16) k_rope_any<__half><<<grid, kRopeWarps * 32, 0, s>>>(p);
    else k_rope_any<__nv_bfloat16><<<grid, kRopeWarps * 32, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace vdt

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

// Rows of whole 16-byte vectors: LANES lanes a row, a lane two vectors that
// hold each other's partners (half a rotation apart, or neighbours), so the
// rotation stays in the lane.  A warp takes one token and ITER rows for each
// of its lane groups: the angles are read once for all of them, and ITER rows'
// loads are in flight together.
template <typename T, int LANES, int ITER>
__global__ void __launch_bounds__(kRopeWarps * 32) k_rope_rows(RopeParams p, long long items, int parts) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x % LANES, group = threadIdx.x % 32 / LANES;
    constexpr int kGroups = 32 / LANES;
    const long long item = (long long)blockIdx.x * kRopeWarps + threadIdx.x / 32;
    if (item >= items) return;
    const long long token = item / parts;
    const int first = (int)(item - token * parts) * (kGroups * ITER) + group, all = p.heads + p.kv_heads;
    const bool pairs = p.layout == VDT_ROPE_PAIRS, in = lane < p.dim / (2 * N);
    const int turned = p.rot / (2 * N);                    // VDT_ROPE_HALF: lanes that rotate
    int v0 = 2 * lane, v1 = v0 + 1;                        // the lane's vectors
    if (!pairs && lane < turned) {
        v0 = lane;
        v1 = lane + turned;
    }
    const bool t0 = in && v0 * N < p.rot, t1 = in && v1 * N < p.rot;
    Vec16<T> x[ITER][2];
    T* to[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int h = first + i * kGroups;
        const RopeRow r = rope_row<T>(p, token, min(h, all - 1));
        to[i] = h < all ? static_cast<T*>(r.out) : nullptr;
        const T* from = static_cast<const T*>(r.in);
        x[i][0].raw = x[i][1].raw = make_uint4(0, 0, 0, 0);
        if (in && h < all) {
            x[i][0].raw = *reinterpret_cast<const uint4*>(from + v0 * N);
            x[i][1].raw = *reinterpret_cast<const uint4*>(from + v1 * N);
        }
    }
    // the angles: N of them; with neighbours paired half of them are v0's, half v1's
    const int at = p.rot ? p.at[token] : 0;
    const bool known = !p.rot || (at >= 0 && at < p.positions);
    float c[N], s[N];
    {
        const float* row = p.table + (long long)(known ? at : 0) * p.rot + lane * N;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const bool on = pairs && j >= N / 2 && N > 4 ? t1 : t0;
            const float4 a = on ? __ldg(reinterpret_cast<const float4*>(row + j)) : make_float4(1, 1, 1, 1);
            const float4 b = on ? __ldg(reinterpret_cast<const float4*>(row + p.rot / 2 + j)) : make_float4(0, 0, 0, 0);
            c[j] = a.x; c[j + 1] = a.y; c[j + 2] = a.z; c[j + 3] = a.w;
            s[j] = b.x; s[j + 1] = b.y; s[j + 2] = b.z; s[j + 3] = b.w;
        }
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        float a[N], b[N];
        x[i][0].get(a);
        x[i][1].get(b);
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) sq = fmaf(a[j], a[j], fmaf(b[j], b[j], sq));
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
        float f = norm_factor(sq, p);
        if (!known) f = __int_as_float(0x7fffffff);
        const void* weight = first + i * kGroups < p.heads ? p.wq : p.wk;
        if (weight && in) {
            Vec16<T> w;
            float g[N];
            w.raw = __ldg(reinterpret_cast<const uint4*>(weight) + v0);
            w.get(g);
#pragma unroll
            for (int j = 0; j < N; ++j) a[j] *= f * g[j];
            w.raw = __ldg(reinterpret_cast<const uint4*>(weight) + v1);
            w.get(g);
#pragma unroll
            for (int j = 0; j < N; ++j) b[j] *= f * g[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                a[j] *= f;
                b[j] *= f;
            }
        }
        if (pairs) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float ca = c[j / 2], sa = s[j / 2], cb = c[N / 2 + j / 2], sb = s[N / 2 + j / 2];
                const float a0 = a[j], b0 = b[j];
                if (t0) {
                    a[j] = a0 * ca - a[j + 1] * sa;
                    a[j + 1] = a[j + 1] * ca + a0 * sa;
                }
                if (t1) {
                    b[j] = b0 * cb - b[j + 1] * sb;
                    b[j + 1] = b[j + 1] * cb + b0 * sb;
                }
            }
        } else if (t0) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float a0 = a[j];
                a[j] = a0 * c[j] - b[j] * s[j];
                b[j] = b[j] * c[j] + a0 * s[j];
            }
        }
        if (to[i] && in) {
            Vec16<T> y;
            y.set(a);
            *reinterpret_cast<uint4*>(to[i] + v0 * N) = y.raw;
            y.set(b);
            *reinterpret_cast<uint4*>(to[i] + v1 * N) = y.raw;
        }
    }
}

// whether every row and weight starts on 16 bytes, and the rotation keeps to whole vectors
bool whole_vectors(const RopeParams& p) {
    const int n = 16 / type_size(p.type);
    if (p.dim % (2 * n) || p.dim > 64 * n || p.rot % (p.layout == VDT_ROPE_PAIRS && n == 4 ? 8 : 2 * n)) return false;
    for (const long long s : {p.q_token, p.q_head, p.k_token, p.k_head, p.qo_token, p.qo_head, p.ko_token, p.ko_head})
        if (s % n) return false;
    for (const void* a : {p.q, p.k, (const void*)p.q_out, (const void*)p.k_out, p.wq, p.wk, (const void*)p.table})
        if (!aligned(a, 16)) return false;
    return true;
}

template <typename T, int LANES, int ITER>
cudaError_t rows_launch(const RopeParams& p, cudaStream_t s) {
    const int parts = (p.heads + p.kv_heads + 32 / LANES * ITER - 1) / (32 / LANES * ITER);
    const long long items = p.tokens * parts, grid = (items + kRopeWarps - 1) / kRopeWarps;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    k_rope_rows<T, LANES, ITER><<<(unsigned)grid, kRopeWarps * 32, 0, s>>>(p, items, parts);
    return cudaGetLastError();
}

// Several rows a lane group where there are enough of them to fill the GPU: as
// many as leave the fewest places empty at a token's end (40 heads in groups of
// 4: five rows, twice), of those the most.
template <typename T, int LANES>
cudaError_t by_rows(const RopeParams& p, cudaStream_t s) {
    const int all = p.heads + p.kv_heads, each = 32 / LANES, turns = (all + each - 1) / each;
    if (p.tokens * all * LANES < 4LL * 32 * 16 * kSmCount || turns < 2) return rows_launch<T, LANES, 1>(p, s);
    int best = 2;
    for (const int n : {3, 4, 5})
        if ((turns + n - 1) / n * n <= (turns + best - 1) / best * best) best = n;
    if (best == 2) return rows_launch<T, LANES, 2>(p, s);
    if (best == 3) return rows_launch<T, LANES, 3>(p, s);
    if (best == 4) return rows_launch<T, LANES, 4>(p, s);
    return rows_launch<T, LANES, 5>(p, s);
}

template <typename T>
cudaError_t by_lanes(const RopeParams& p, cudaStream_t s) {
    const int need = p.dim / (2 * Vec16<T>::N);
    if (need <= 2) return by_rows<T, 2>(p, s);
    if (need <= 4) return by_rows<T, 4>(p, s);
    if (need <= 8) return by_rows<T, 8>(p, s);
    if (need <= 16) return by_rows<T, 16>(p, s);
    return by_rows<T, 32>(p, s);
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
    if (whole_vectors(p)) {
        if (p.type == VDT_F32) return by_lanes<float>(p, s);
        if (p.type == VDT_F16) return by_lanes<__half>(p, s);
        return by_lanes<__nv_bfloat16>(p, s);
    }
    const long long rows = p.tokens * (p.heads + p.kv_heads);
    const long long want = (rows + kRopeWarps - 1) / kRopeWarps;
    const unsigned grid = (unsigned)(want < kSmCount * 16 ? want : kSmCount * 16);
    if (p.type == VDT_F32) k_rope_any<float><<<grid, kRopeWarps * 32, 0, s>>>(p);
    else if (p.type == VDT_F16) k_rope_any<__half><<<grid, kRopeWarps * 32, 0, s>>>(p);
    else k_rope_any<__nv_bfloat16><<<grid, kRopeWarps * 32, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace vdt

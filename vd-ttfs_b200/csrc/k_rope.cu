// k_rope.cu -- the norm of each head of the queries and keys, and the position
// rotation, in one pass.
//
//   y = x * w / sqrt(mean(x^2) + eps)         (VDT_NORM_RMS)
//   y = x * w / sqrt(sum(x^2) + eps)          (VDT_NORM_L2)
//   (a, b) -> (a cos - b sin, b cos + a sin)  for the pairs of the first `rot` values
//
// VDT_ROPE_HALF pairs value i with i + rot / 2, VDT_ROPE_PAIRS 2i with 2i + 1.
// Everything between the load and the store is 32-bit.  Each value is read and
// written once: 16381 tokens of 40 heads of 128 in bf16 take 80 us, 4.2 TB/s
// (floor 53 us); what is left is the latency of position, angles and rows.
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
    return rsqrtf(fmaf(squares, p.share, p.eps));
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
// rotation stays in the lane.  A warp takes one token and up to ITER heads of
// the queries, or of the keys, for each of its lane groups, all loads in
// flight together.  The weights times the angles are made once for them:
//   a' = f (a w_a cos - b w_b sin),  b' = f (b w_b cos + a w_a sin)
// is then four products and a factor for two values, two values to an
// instruction.  What bounds this is memory: with the products made for each
// row it was the instructions (280 a row and lane against 90).
template <typename T, int LANES, int ITER, bool PAIRS>
__global__ void __launch_bounds__(kRopeWarps * 32) k_rope_rows(RopeParams p, int q_parts) {
    constexpr int N = Vec16<T>::N, kGroups = 32 / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x % 32 / LANES;
    const long long token = (long long)blockIdx.x * kRopeWarps + threadIdx.x / 32;
    if (token >= p.tokens) return;
    const bool keys = (int)blockIdx.y >= q_parts;
    const int first = (blockIdx.y - (keys ? q_parts : 0)) * (kGroups * ITER), all = keys ? p.kv_heads : p.heads;
    const long long in_step = keys ? p.k_head : p.q_head, out_step = keys ? p.ko_head : p.qo_head;
    // the lane's vectors: lanes side by side take vectors side by side
    const int half = p.rot / (2 * N), rest = p.dim / (2 * N) - half;
    const bool on = lane < half + rest, turned = lane < half;
    const int v0 = turned ? lane : half + lane, v1 = v0 + (turned ? half : rest);
    const T* const in = (keys ? static_cast<const T*>(p.k) + token * p.k_token : static_cast<const T*>(p.q) + token * p.q_token) +
                        (first + group) * in_step;
    T* const out = (keys ? static_cast<T*>(p.k_out) + token * p.ko_token : static_cast<T*>(p.q_out) + token * p.qo_token) +
                   (first + group) * out_step;
    Vec16<T> x[ITER][2];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        x[i][0].raw = x[i][1].raw = make_uint4(0, 0, 0, 0);
        if (on && first + group + i * kGroups < all) {
            const T* const from = in + i * kGroups * in_step;
            x[i][0].raw = *reinterpret_cast<const uint4*>(from + v0 * N);
            x[i][1].raw = *reinterpret_cast<const uint4*>(from + v1 * N);
        }
    }
    // factors of a and b in a' (the second negative) and of b and a in b'; of
    // the lanes that do not rotate the first and third are the weights
    float2 fa[2][N / 2], fb[2][N / 2];
    const int at = p.rot ? p.at[token] : 0;
    const bool known = !p.rot || (at >= 0 && at < p.positions);
    {
        float w[2][N];
        const void* const weight = keys ? p.wk : p.wq;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (weight && on) {
                Vec16<T> v;
                v.raw = __ldg(reinterpret_cast<const uint4*>(weight) + (e ? v1 : v0));
                v.get(w[e]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) w[e][j] = 1.0f;
            }
        }
        // the angles: N, of values 0..N - 1 of a; with neighbours paired N / 2 of
        // a's pairs and N / 2 of b's
        float c[N], s[N];
        const float* const row = p.table + (long long)(known ? at : 0) * p.rot;
        constexpr int kRun = PAIRS && N == 4 ? 2 : 4;
#pragma unroll
        for (int j = 0; j < N; j += kRun) {
            const int from = !PAIRS ? lane * N + j : j < N / 2 ? v0 * (N / 2) + j : v1 * (N / 2) + j - N / 2;
#pragma unroll
            for (int q = 0; q < kRun; ++q) {
                c[j + q] = 1.0f;
                s[j + q] = 0.0f;
            }
            if (turned) {
                if constexpr (kRun == 4) {
                    const float4 a = __ldg(reinterpret_cast<const float4*>(row + from)), b = __ldg(reinterpret_cast<const float4*>(row + p.rot / 2 + from));
                    c[j] = a.x; c[j + 1] = a.y; c[j + 2] = a.z; c[j + 3] = a.w;
                    s[j] = b.x; s[j + 1] = b.y; s[j + 2] = b.z; s[j + 3] = b.w;
                } else {
                    const float2 a = __ldg(reinterpret_cast<const float2*>(row + from)), b = __ldg(reinterpret_cast<const float2*>(row + p.rot / 2 + from));
                    c[j] = a.x; c[j + 1] = a.y;
                    s[j] = b.x; s[j + 1] = b.y;
                }
            }
        }
        if (PAIRS) {
            // a vector's pair (x, y): (x, y) (w_x cos, w_y cos) + (y, x) (-w_y sin, w_x sin)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    const float cj = c[e * N / 2 + j], sj = s[e * N / 2 + j];
                    fa[e][j] = make_float2(w[e][2 * j] * cj, w[e][2 * j + 1] * cj);
                    fb[e][j] = make_float2(-w[e][2 * j + 1] * sj, w[e][2 * j] * sj);
                }
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                fa[0][j] = make_float2(w[0][2 * j] * c[2 * j], w[0][2 * j + 1] * c[2 * j + 1]);
                fb[0][j] = make_float2(-w[1][2 * j] * s[2 * j], -w[1][2 * j + 1] * s[2 * j + 1]);
                fa[1][j] = make_float2(w[1][2 * j] * c[2 * j], w[1][2 * j + 1] * c[2 * j + 1]);
                fb[1][j] = make_float2(w[0][2 * j] * s[2 * j], w[0][2 * j + 1] * s[2 * j + 1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (first + i * kGroups >= all) break;               // of the whole warp
        float2 a[N / 2], b[N / 2];
        x[i][0].get(reinterpret_cast<float*>(a));
        x[i][1].get(reinterpret_cast<float*>(b));
        float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) sq = fma2(a[j], a[j], fma2(b[j], b[j], sq));
        float squares = sq.x + sq.y;
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, d);
        const float f1 = known ? norm_factor(squares, p) : __int_as_float(0x7fffffff);
        const float2 f = make_float2(f1, f1);
        float2 ya[N / 2], yb[N / 2];
        if (turned) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const float2 pa = PAIRS ? make_float2(a[j].y, a[j].x) : b[j], pb = PAIRS ? make_float2(b[j].y, b[j].x) : a[j];
                ya[j] = mul2(f, fma2(pa, fb[0][j], mul2(a[j], fa[0][j])));
                yb[j] = mul2(f, fma2(pb, fb[1][j], mul2(b[j], fa[1][j])));
            }
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                ya[j] = mul2(f, mul2(a[j], fa[0][j]));
                yb[j] = mul2(f, mul2(b[j], fa[1][j]));
            }
        }
        if (on && first + group + i * kGroups < all) {
            T* const to = out + i * kGroups * out_step;
            Vec16<T> y;
            y.set(reinterpret_cast<const float*>(ya));
            *reinterpret_cast<uint4*>(to + v0 * N) = y.raw;
            y.set(reinterpret_cast<const float*>(yb));
            *reinterpret_cast<uint4*>(to + v1 * N) = y.raw;
        }
    }
}

// whether every row and weight starts on 16 bytes, and a lane's two vectors
// rotate both or neither
bool whole_vectors(const RopeParams& p) {
    const int n = 16 / type_size(p.type);
    if (p.dim % (2 * n) || p.dim > 64 * n || p.rot % (2 * n)) return false;
    for (const long long s : {p.q_token, p.q_head, p.k_token, p.k_head, p.qo_token, p.qo_head, p.ko_token, p.ko_head})
        if (s % n) return false;
    for (const void* a : {p.q, p.k, (const void*)p.q_out, (const void*)p.k_out, p.wq, p.wk, (const void*)p.table})
        if (!aligned(a, 16)) return false;
    return true;
}

template <typename T, int LANES, int ITER>
cudaError_t rows_launch(const RopeParams& p, cudaStream_t s) {
    constexpr int kEach = 32 / LANES * ITER;
    const int q_parts = (p.heads + kEach - 1) / kEach, k_parts = (p.kv_heads + kEach - 1) / kEach;
    const dim3 grid((unsigned)((p.tokens + kRopeWarps - 1) / kRopeWarps), q_parts + k_parts);
    if (p.layout == VDT_ROPE_PAIRS) k_rope_rows<T, LANES, ITER, true><<<grid, kRopeWarps * 32, 0, s>>>(p, q_parts);
    else k_rope_rows<T, LANES, ITER, false><<<grid, kRopeWarps * 32, 0, s>>>(p, q_parts);
    return cudaGetLastError();
}

// Four rows a lane group where there are enough of them to fill the GPU
template <typename T, int LANES>
cudaError_t by_rows(const RopeParams& p, cudaStream_t s) {
    const long long rows = p.tokens * (p.heads + p.kv_heads);
    return rows * LANES >= 4LL * 32 * 16 * kSmCount ? rows_launch<T, LANES, 4>(p, s) : rows_launch<T, LANES, 1>(p, s);
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

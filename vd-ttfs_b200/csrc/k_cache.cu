// k_cache.cu -- a paged cache of keys and values held in 8 bits.
//
// A page holds `page` tokens of one sequence.  Its codes are k[page_no][head]
// [token][dim] and v[page_no][head][dim][token] (the attention's second product
// sums over tokens, so a value row keeps its tokens side by side), each
// [page_no][head] under one scale.
//
// Appending: with m the largest magnitude of the new tokens in a page,
//   scale' = max(scale, m / 127) if tokens are in the page already, else m / 127
//   old codes: round(code * (scale / scale')),  new codes: round(x / scale')
// An old code moves only where a new token is larger than all before it.
//
// Bound by memory for prompts (6 of up to 4093 tokens, 8 heads of 128 in bf16,
// appended and read back: 58 us, 3.6 TB/s; floor 33 us) and by latency for a
// token a sequence (48 of them, both calls: 9.4 us).
#include <type_traits>

#include "seq_internal.h"

namespace vdt {
namespace {

constexpr int kCacheThreads = 128;

// A sequence's part of a call: packed rows [first, first + rows), or none
// where the caller's offsets do not fit the buffers.
struct Part {
    long long first;
    int rows, held;
};
__device__ __forceinline__ Part part_of(const CacheRows& r, int b) {
    Part p;
    p.first = r.starts[b];
    const long long rows = (long long)r.starts[b + 1] - p.first;
    p.held = r.held[b];
    const bool ok = rows > 0 && rows <= r.most && p.first >= 0 && p.first + rows <= r.total && p.held >= 0 && p.held <= 1 << 30;
    p.rows = ok ? (int)rows : 0;
    return p;
}
// The page's number, or -1 where the table has none
__device__ __forceinline__ int page_of(const CacheRows& r, int b, int j, int pages) {
    if (j >= r.width) return -1;
    const int n = r.table[(long long)b * r.width + j];
    return n >= 0 && n < pages ? n : -1;
}

__device__ __forceinline__ float block_max(float m) {
    __shared__ float part[kCacheThreads / 32];
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max_nan(__shfl_xor_sync(0xffffffffu, m, d), m);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCacheThreads / 32; ++i) m = max_nan(part[i], m);
    __syncthreads();
    return m;
}

// The tokens of a call that fall into one page of one head
struct Place {
    int n, old;             // new tokens; tokens before them in the page
    long long first, slot;  // the first one's packed row; page number * heads + head
};
__device__ __forceinline__ bool place_of(const vdt_cache8& c, const CacheRows& r, int h, Place& o) {
    const int b = blockIdx.z;
    const Part p = part_of(r, b);
    if (!p.rows) return false;
    const int j = p.held / c.page + blockIdx.x;
    const int lo = max(p.held, j * c.page), hi = min(p.held + p.rows, (j + 1) * c.page);
    if (lo >= hi) return false;
    const int no = page_of(r, b, j, c.pages);
    if (no < 0) return false;
    o.n = hi - lo;
    o.old = lo - j * c.page;
    o.first = p.first + (lo - p.held);
    o.slot = (long long)no * c.heads + h;
    return true;
}

// The scale after the new tokens' largest magnitude m; old codes rounded anew
// where it grew.  All threads of the CTA.
__device__ __forceinline__ float grow(const vdt_cache8& c, const Place& o, bool values, float m) {
    float* scale = (values ? c.v_scale : c.k_scale) + o.slot;
    int8_t* codes = (values ? c.v : c.k) + o.slot * c.page * c.dim;
    float to = m * kCodeStep;
    const float was = o.old ? *scale : 0.0f;
    if (o.old) to = max_nan(to, was);
    __syncthreads();
    if (threadIdx.x == 0) *scale = to;
    const float ratio = o.old && to > 0.0f ? __fdiv_rn(was, to) : 1.0f;
    if (ratio != 1.0f)
        for (int i = threadIdx.x; i < o.old * c.dim; i += kCacheThreads) {
            int8_t* q = codes + (values ? (long long)(i / o.old) * c.page + i % o.old : (long long)i);
            *q = (int8_t)rintf((float)*q * ratio);
        }
    return to;
}

// Any stride and alignment: one CTA for each (page touched, head, sequence).
template <typename T>
__global__ void __launch_bounds__(kCacheThreads) k_cache_append_any(vdt_cache8 c, CacheRows r, const T* __restrict__ k,
                                                                    const T* __restrict__ v, long long k_token, long long k_head,
                                                                    long long v_token, long long v_head) {
    Place o;
    const int h = blockIdx.y, dim = c.dim;
    if (!place_of(c, r, h, o)) return;
    for (int side = 0; side < 2; ++side) {
        const T* x = side ? v + o.first * v_token + h * v_head : k + o.first * k_token + h * k_head;
        const long long step = side ? v_token : k_token;
        int8_t* codes = (side ? c.v : c.k) + o.slot * c.page * dim;
        float m = 0.0f;
        for (int i = threadIdx.x; i < o.n * dim; i += kCacheThreads) m = max_nan(fabsf(to_f32(x[i / dim * step + i % dim])), m);
        const float to = grow(c, o, side, block_max(m));
        for (int i = threadIdx.x; i < o.n * dim; i += kCacheThreads) {
            const int t = i / dim, d = i % dim;
            codes[side ? (long long)d * c.page + o.old + t : (long long)(o.old + t) * dim + d] = (int8_t)code_of(to_f32(x[t * step + d]), to);
        }
    }
}

// A value tile in shared memory: byte (d, t) of [dim][page].  The words of a
// row are permuted by the row's group of eight, so that lanes that hold eight
// dimensions each of one token meet on as few banks as there are words.
template <int P>
__device__ __forceinline__ int tile_byte(int d, int t) {
    return d * P + ((t / 4 ^ (d / 8 & (P / 4 - 1))) * 4) + t % 4;
}

// Rows of whole 16-byte vectors: one CTA for each (page touched, head, sequence)
// and for keys and values apart.  The page's new vectors are read once and stay
// in registers (at most 64 tokens x 256 values over 128 threads); keys go out as
// they are, values through shared memory, where their tokens come to lie side
// by side.
template <typename T, int D, int P>
__global__ void __launch_bounds__(kCacheThreads) k_cache_append_rows(vdt_cache8 c, CacheRows r, const T* __restrict__ k,
                                                                     const T* __restrict__ v, long long k_token, long long k_head,
                                                                     long long v_token, long long v_head) {
    constexpr int N = Vec16<T>::N, kRow = D / N, kHeld = (P * kRow + kCacheThreads - 1) / kCacheThreads;
    __shared__ __align__(16) unsigned char tile[D * P];
    Place o;
    const bool side = (int)blockIdx.y >= c.heads;
    const int h = blockIdx.y - (side ? c.heads : 0);
    if (!place_of(c, r, h, o)) return;
    const T* x = side ? v + o.first * v_token + h * v_head : k + o.first * k_token + h * k_head;
    const long long step = side ? v_token : k_token;
    int8_t* codes = (side ? c.v : c.k) + o.slot * (P * D);
    // a thread has vector e of tokens t; of values that start a page, four
    // tokens side by side, whose codes make whole words
    constexpr bool kFours = kHeld % 4 == 0 && kCacheThreads % kRow == 0;
    const bool fours = kFours && side && o.old == 0;
    auto place = [&](int i, int& t, int& e) {
        const int at = threadIdx.x + i * kCacheThreads;
        t = at / kRow;
        e = at % kRow;
        if (fours) {
            t = 4 * (threadIdx.x / kRow + i / 4 * (kCacheThreads / kRow)) + i % 4;
            e = threadIdx.x % kRow;
        }
    };
    Vec16<T> held[kHeld];
    Largest<T> most;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        int t, e;
        place(i, t, e);
        held[i].raw = t < o.n ? *reinterpret_cast<const uint4*>(x + t * step + e * N) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most.add(held[i]);
    const Coder coder(grow(c, o, side, block_max(most.value())));
    if (fours) {
        if constexpr (kFours) {
#pragma unroll
            for (int i = 0; i < kHeld; i += 4) {
                int t, e;
                place(i, t, e);
                uint32_t w[4][N / 4];
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    float f[N];
                    held[i + a].get(f);
                    coder.words<N>(f, w[a]);
                }
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const uint32_t x0 = w[0][j / 4], x1 = w[1][j / 4], x2 = w[2][j / 4], x3 = w[3][j / 4];
                    const uint32_t a = __byte_perm(x0, x1, 0x5140), b = __byte_perm(x2, x3, 0x5140);     // dimensions j, j + 1
                    const uint32_t d = __byte_perm(x0, x1, 0x7362), g = __byte_perm(x2, x3, 0x7362);     // j + 2, j + 3
                    const uint32_t y[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(d, g, 0x5410),
                                           __byte_perm(d, g, 0x7632)};
#pragma unroll
                    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint32_t*>(tile + tile_byte<P>(e * N + j + q, t)) = y[q];
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            int t, e;
            place(i, t, e);
            if (t >= o.n) continue;
            float f[N];
            uint32_t w[N / 4];
            held[i].get(f);
            coder.words<N>(f, w);
            if (!side) {
                int8_t* to = codes + (o.old + t) * D + e * N;
                if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(to) = w[0];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) tile[tile_byte<P>(e * N + j, o.old + t)] = (unsigned char)(w[j / 4] >> (8 * (j % 4)));
            }
        }
    }
    if (!side) return;
    __syncthreads();
    if (o.n == P) {
        for (int i = threadIdx.x; i < D * P / 16; i += kCacheThreads) {
            const int d = i / (P / 16), t = i % (P / 16) * 16;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(tile + tile_byte<P>(d, t + 4 * j));
            *reinterpret_cast<uint4*>(codes + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        for (int i = threadIdx.x; i < D * o.n; i += kCacheThreads) {
            const int d = i / o.n, t = o.old + i % o.n;
            codes[d * P + t] = (int8_t)tile[tile_byte<P>(d, t)];
        }
    }
}

// One CTA for each (page, head, sequence), for keys and values apart: its
// tokens as values, packed.  Value codes go through shared memory.
template <typename T, int D, int P>
__global__ void __launch_bounds__(kCacheThreads) k_cache_load(vdt_cache8 c, CacheRows r, T* __restrict__ k, T* __restrict__ v) {
    constexpr int N = Vec16<T>::N, kRow = D / N;
    __shared__ __align__(16) unsigned char tile[D * P];
    const bool side = (int)blockIdx.y >= c.heads;
    const int b = blockIdx.z, h = blockIdx.y - (side ? c.heads : 0), j = blockIdx.x;
    const long long start = r.starts[b], rows = (long long)r.starts[b + 1] - start;
    const int kept = r.held[b];
    if (kept > rows || kept > r.most || start < 0 || start + rows > r.total) {
        // lengths that do not fit the buffers or `most`: NaN to those of the run's rows that there are
        if (j == 0 && kept > 0)
            for (long long i = max(start, 0LL) * D + threadIdx.x; i < min(start + rows, r.total) * D; i += kCacheThreads)
                (side ? v : k)[(i / D * c.heads + h) * D + i % D] = from_f32<T>(__int_as_float(0x7fffffff));
        return;
    }
    const int n = min(kept - j * P, P);
    if (n <= 0) return;
    const int no = page_of(r, b, j, c.pages);
    const long long slot = (long long)max(no, 0) * c.heads + h, at = slot * (P * D);
    const float scale = no < 0 ? __int_as_float(0x7fffffff) : (side ? c.v_scale : c.k_scale)[slot];   // a page that is not in the cache: NaN
    const long long out = ((start + (long long)j * P) * c.heads + h) * D, step = (long long)c.heads * D;
    if (side) {
        const uint4* from = reinterpret_cast<const uint4*>(c.v + at);
        for (int i = threadIdx.x; i < D * P / 16; i += kCacheThreads) {
            const uint4 x = from[i];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            const int d = i / (P / 16), t = i % (P / 16) * 16;
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<uint32_t*>(tile + tile_byte<P>(d, t + 4 * q)) = w[q];
        }
        __syncthreads();
    }
    if (side) {
        // a word is four tokens of a dimension: N of them make four rows' vectors
        for (int i = threadIdx.x; i < (n + 3) / 4 * kRow; i += kCacheThreads) {
            const int t = i / kRow * 4, e = i % kRow;
            uint32_t w[N];
#pragma unroll
            for (int q = 0; q < N; ++q) w[q] = *reinterpret_cast<const uint32_t*>(tile + tile_byte<P>(e * N + q, t)) ^ 0x80808080u;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                if (t + a >= n) break;
                float2 f[N / 2];
#pragma unroll
                for (int q = 0; q < N; q += 2) f[q / 2] = code_pair(code_byte(w[q], a), code_byte(w[q + 1], a), scale);
                Vec16<T> y;
                y.set(reinterpret_cast<const float*>(f));
                *reinterpret_cast<uint4*>(v + out + (t + a) * step + e * N) = y.raw;
            }
        }
        return;
    }
    for (int i = threadIdx.x; i < n * kRow; i += kCacheThreads) {
        const int t = i / kRow, e = i % kRow;
        float2 f[N / 2];
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(c.k + at + t * D + e * N + q) ^ 0x80808080u;
            f[q / 2] = code_pair(code_byte(w, 0), code_byte(w, 1), scale);
            f[q / 2 + 1] = code_pair(code_byte(w, 2), code_byte(w, 3), scale);
        }
        Vec16<T> y;
        y.set(reinterpret_cast<const float*>(f));
        *reinterpret_cast<uint4*>(k + out + t * step + e * N) = y.raw;
    }
}

// calls go(dim, page) with both as compile-time constants
template <typename Go>
cudaError_t by_shape(const vdt_cache8& c, Go go) {
    auto by_page = [&](auto dim) {
        if (c.page == 16) return go(dim, std::integral_constant<int, 16>{});
        if (c.page == 32) return go(dim, std::integral_constant<int, 32>{});
        return go(dim, std::integral_constant<int, 64>{});
    };
    switch (c.dim) {
        case 32: return by_page(std::integral_constant<int, 32>{});
        case 64: return by_page(std::integral_constant<int, 64>{});
        case 96: return by_page(std::integral_constant<int, 96>{});
        case 128: return by_page(std::integral_constant<int, 128>{});
        case 192: return by_page(std::integral_constant<int, 192>{});
        default: return by_page(std::integral_constant<int, 256>{});
    }
}

template <typename T>
cudaError_t append(const vdt_cache8& c, const CacheRows& r, const void* k, const void* v, long long kt, long long kh,
                   long long vt, long long vh, cudaStream_t s) {
    const dim3 grid((r.most + c.page - 2) / c.page + 1, c.heads, r.seqs);
    const T *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v);
    constexpr int N = Vec16<T>::N;
    if (!aligned(k, 16) || !aligned(v, 16) || kt % N || kh % N || vt % N || vh % N) {
        k_cache_append_any<T><<<grid, kCacheThreads, 0, s>>>(c, r, kp, vp, kt, kh, vt, vh);
        return cudaGetLastError();
    }
    return by_shape(c, [&](auto dim, auto page) {
        k_cache_append_rows<T, dim(), page()><<<dim3(grid.x, 2 * grid.y, grid.z), kCacheThreads, 0, s>>>(c, r, kp, vp, kt, kh, vt, vh);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t load(const vdt_cache8& c, const CacheRows& r, void* k, void* v, cudaStream_t s) {
    const dim3 grid((r.most + c.page - 1) / c.page, 2 * c.heads, r.seqs);
    return by_shape(c, [&](auto dim, auto page) {
        k_cache_load<T, dim(), page()><<<grid, kCacheThreads, 0, s>>>(c, r, static_cast<T*>(k), static_cast<T*>(v));
        return cudaGetLastError();
    });
}

}  // namespace

cudaError_t launch_cache_append(const vdt_cache8& c, const CacheRows& r, const void* k, const void* v, int type,
                                long long kt, long long kh, long long vt, long long vh, cudaStream_t s) {
    if (type == VDT_F32) return append<float>(c, r, k, v, kt, kh, vt, vh, s);
    if (type == VDT_F16) return append<__half>(c, r, k, v, kt, kh, vt, vh, s);
    return append<__nv_bfloat16>(c, r, k, v, kt, kh, vt, vh, s);
}

cudaError_t launch_cache_load(const vdt_cache8& c, const CacheRows& r, void* k, void* v, int type, cudaStream_t s) {
    if (type == VDT_F32) return load<float>(c, r, k, v, s);
    if (type == VDT_F16) return load<__half>(c, r, k, v, s);
    return load<__nv_bfloat16>(c, r, k, v, s);
}

}  // namespace vdt

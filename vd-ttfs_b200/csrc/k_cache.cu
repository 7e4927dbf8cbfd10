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
    const bool ok = rows > 0 && rows <= r.most && p.first >= 0 && p.first + rows <= r.total && p.held >= 0;
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

// One CTA for each (page touched, head, sequence).
template <typename T>
__global__ void __launch_bounds__(kCacheThreads) k_cache_append(vdt_cache8 c, CacheRows r, const T* __restrict__ k,
                                                                const T* __restrict__ v, long long k_token,
                                                                long long k_head, long long v_token, long long v_head) {
    const int b = blockIdx.z, h = blockIdx.y;
    const Part p = part_of(r, b);
    if (!p.rows) return;
    const int j = p.held / c.page + blockIdx.x;
    const int lo = max(p.held, j * c.page), hi = min(p.held + p.rows, (j + 1) * c.page);
    if (lo >= hi) return;
    const int no = page_of(r, b, j, c.pages);
    if (no < 0) return;
    const int n = hi - lo, old = lo - j * c.page, dim = c.dim;      // new tokens, tokens before them in the page
    const long long first = p.first + (lo - p.held), at = ((long long)no * c.heads + h) * c.page * dim;
    for (int side = 0; side < 2; ++side) {
        const T* x = side ? v + first * v_token + h * v_head : k + first * k_token + h * k_head;
        const long long step = side ? v_token : k_token;
        int8_t* codes = (side ? c.v : c.k) + at;
        float* scale = (side ? c.v_scale : c.k_scale) + (long long)no * c.heads + h;
        float m = 0.0f;
        for (int i = threadIdx.x; i < n * dim; i += kCacheThreads) m = max_nan(fabsf(to_f32(x[i / dim * step + i % dim])), m);
        m = block_max(m);
        float to = m * kCodeStep;
        const float was = old ? *scale : 0.0f;
        if (old) to = max_nan(to, was);
        __syncthreads();
        if (threadIdx.x == 0) *scale = to;
        const float ratio = old && to > 0.0f ? __fdiv_rn(was, to) : 1.0f;
        if (old && ratio != 1.0f)
            for (int i = threadIdx.x; i < old * dim; i += kCacheThreads) {
                int8_t* q = codes + (side ? (long long)(i % dim) * c.page + i / dim : (long long)i);
                *q = (int8_t)rintf((float)*q * ratio);
            }
        for (int i = threadIdx.x; i < n * dim; i += kCacheThreads) {
            const int t = i / dim, d = i % dim;
            codes[side ? (long long)d * c.page + old + t : (long long)(old + t) * dim + d] =
                (int8_t)code_of(to_f32(x[t * step + d]), to);
        }
    }
}

// One CTA for each (page, head, sequence): its tokens as values, packed.
template <typename T>
__global__ void __launch_bounds__(kCacheThreads) k_cache_load(vdt_cache8 c, CacheRows r, T* __restrict__ k, T* __restrict__ v) {
    const int b = blockIdx.z, h = blockIdx.y, j = blockIdx.x;
    const long long start = r.starts[b], rows = (long long)r.starts[b + 1] - start;
    const int kept = r.held[b];
    const int n = min(kept - j * c.page, c.page);
    if (n <= 0 || kept > rows || start < 0 || start + rows > r.total) return;
    const int no = page_of(r, b, j, c.pages);
    const float nan = __int_as_float(0x7fffffff);        // a page that is not in the cache
    const long long slot = (long long)max(no, 0) * c.heads + h, at = slot * c.page * c.dim;
    const float ks = no < 0 ? nan : c.k_scale[slot], vs = no < 0 ? nan : c.v_scale[slot];
    for (int i = threadIdx.x; i < n * c.dim; i += kCacheThreads) {
        const int t = i / c.dim, d = i % c.dim;
        const long long to = ((start + j * c.page + t) * c.heads + h) * c.dim + d;
        k[to] = from_f32<T>((float)c.k[at + i] * ks);
        v[to] = from_f32<T>((float)c.v[at + (long long)d * c.page + t] * vs);
    }
}

template <typename T>
cudaError_t append(const vdt_cache8& c, const CacheRows& r, const void* k, const void* v, long long kt, long long kh,
                   long long vt, long long vh, cudaStream_t s) {
    const dim3 grid((r.most + c.page - 1) / c.page + 1, c.heads, r.seqs);
    k_cache_append<T><<<grid, kCacheThreads, 0, s>>>(c, r, static_cast<const T*>(k), static_cast<const T*>(v), kt, kh, vt, vh);
    return cudaGetLastError();
}
template <typename T>
cudaError_t load(const vdt_cache8& c, const CacheRows& r, void* k, void* v, cudaStream_t s) {
    const dim3 grid((r.most + c.page - 1) / c.page, c.heads, r.seqs);
    k_cache_load<T><<<grid, kCacheThreads, 0, s>>>(c, r, static_cast<T*>(k), static_cast<T*>(v));
    return cudaGetLastError();
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

// k_attend.cu -- attention over the paged 8-bit cache (layout: k_cache.cu).
//
//   out_i = sum_j softmax_j(scale * q_i . (ks_j K_j)) vs_j V_j
//
// over the tokens j that query i sees; K, V are codes, ks and vs their pages'
// scales.  A row that sees nothing gives 0.  The codes go to the tensor cores
// as 16-bit floats, which hold -127..127 exactly; the products are summed in
// 32 bits, and the running maximum and sum of the softmax are 32-bit.
//
// The queries' rounding: q is scaled by a power of two for each row so that
// its largest magnitude is in [1, 2); a 16-bit float then holds every bf16 or
// f16 value whole down to 2^-14 of that (below, to 2^-24 of it).  The weights
// exp(s - max) are in [0, 1]; vs is a page's, so it goes into them relative to
// the largest vs so far, and into the sums' rescaling when that grows.  Their
// rounding to 16 bits is at most 2^-11: that of an f16 output, an eighth of a
// bf16 one's, and it averages over the tokens.
#include "attend_internal.h"

namespace vdt {
namespace {

constexpr int kUnit = 64;          // tokens that a warp takes at a time

// ------------------------------------------------------------ few query rows
// One CTA: a sequence, a head of the cache, 16 of the rows (query, head of
// the group) that share it, and a chunk of the tokens.  Its warps take units
// of 64 tokens in turn; each warp has its own ring of shared memory, into
// which the units' codes are copied in bulk (a page's codes of one head are
// consecutive).  The warps' sums are joined in shared memory, the chunks' by
// k_attend_join.
constexpr int kRowsWarps = 4;
constexpr int kRing = 3;           // entries of a warp's ring; a unit's keys are one, its values one
constexpr int kMostChunk = 4096;   // tokens of a chunk: bounds the page lists in shared memory

// Chunks so that the grid has a few CTAs for each SM, none under 64 tokens a
// warp.  With one chunk the CTAs write the output themselves.
Chunks plan_chunks(int heads, int kv_heads, int seqs, int most, int most_kept) {
    const long long tiles = (long long)kv_heads * seqs * (((long long)most * (heads / kv_heads) + 15) / 16);
    const long long target = 8 * kSmCount;
    const long long want = (target + tiles - 1) / tiles;
    long long tokens = ((long long)most_kept + want - 1) / want;
    constexpr int step = kUnit * kRowsWarps;
    tokens = (tokens + step - 1) / step * step;
    if (tokens < step) tokens = step;
    if (tokens > kMostChunk) tokens = kMostChunk;
    long long count = ((long long)most_kept + tokens - 1) / tokens;
    return {(int)tokens, (int)(count < 1 ? 1 : count)};
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct RowsLayout {
    uint32_t ring, q, bars, pages, bytes;
};
__host__ __device__ inline RowsLayout rows_layout(int dim, int chunk, int page) {
    RowsLayout l;
    const uint32_t ring = (uint32_t)(kRowsWarps * kRing * kUnit * dim);
    const uint32_t sums = (uint32_t)(kRowsWarps * 16 * (dim + 2) * 4);     // reuses the ring
    l.ring = 0;
    l.q = ring > sums ? ring : sums;
    l.bars = l.q + dim * 32 + 64;
    l.pages = l.bars + kRowsWarps * kRing * 8;
    l.bytes = l.pages + chunk / page * 12;
    return l;
}

template <int D, int P>
__global__ void __launch_bounds__(kRowsWarps * 32) k_attend_rows(AttendParams p, int chunk) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kGroups = P / 16;              // 16-token groups of a page
    constexpr int kPages = kUnit / P;            // pages of a unit
    const RowsLayout lay = rows_layout(D, chunk, P);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int b = blockIdx.z, group = p.heads / p.c.heads;
    const int tile = blockIdx.y / p.c.heads, h = blockIdx.y % p.c.heads;
    const Queries s = queries_of(p, b);
    const int rows = s.rows * group - tile * 16;              // rows of this tile
    if (rows <= 0) return;
    const bool split = gridDim.x > 1;
    // tokens that a row sees: all, or up to its own place at the sequence's end
    auto sees = [&](int r) {
        if (r >= rows || s.kept < 0) return 0;
        return p.causal ? max(0, s.kept - s.rows + (tile * 16 + r) / group + 1) : s.kept;
    };
    const int lim0 = sees(g), lim1 = sees(g + 8);
    const int begin = blockIdx.x * chunk, end = min(begin + chunk, sees(min(rows, 16) - 1));
    if (begin >= end && split) return;                        // the join knows as well
    const int units = max(0, (end - begin + kUnit - 1) / kUnit);

    float* q_scale = reinterpret_cast<float*>(smem + lay.q + D * 32);
    uint4* q_frag = reinterpret_cast<uint4*>(smem + lay.q);
    int* pages = reinterpret_cast<int*>(smem + lay.pages);
    float* k_scale = reinterpret_cast<float*>(pages + chunk / P);
    float* v_scale = k_scale + chunk / P;
    const uint32_t bars = shared_address(smem + lay.bars) + warp * kRing * 8;
    const uint32_t ring = shared_address(smem + lay.ring) + warp * kRing * kUnit * D;

    if (lane < kRing) bar_init(bars + lane * 8, 1);
    // the chunk's pages: number and scales; one that is not in the cache is
    // read as page 0 under NaN scales, one past the end is not read at all
    for (int i = threadIdx.x; i < units * kPages; i += kRowsWarps * 32) {
        const int j = begin / P + i;
        int no = -1;
        float ks = 0.0f, vs = 0.0f;
        if (j * P < end) {
            no = p.r.table[(long long)b * p.r.width + j];
            const bool known = no >= 0 && no < p.c.pages;
            if (!known) no = 0;
            ks = known ? p.c.k_scale[(long long)no * p.c.heads + h] : nan_f();
            vs = known ? p.c.v_scale[(long long)no * p.c.heads + h] : nan_f();
            if (vs == inf_f()) vs = nan_f();      // it would be what all other weights are relative to
        }
        pages[i] = no;
        k_scale[i] = ks;
        v_scale[i] = vs;
    }
    // the queries, each row scaled by a power of two
    for (int r = warp; r < 16; r += kRowsWarps) {
        float x[D / 32], m = 0.0f;
        const bool in = r < rows;
        const int row = tile * 16 + r;
        const long long q = (s.first + row / group) * p.q_token + (long long)(h * group + row % group) * p.q_head;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = in ? load_value(p.q, q + lane + 32 * i, p.type) : 0.0f;
            m = fmaxf(m, fabsf(x[i]));
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const int e = m > 0.0f && m < inf_f() ? max(-126, min(126, ilogbf(m))) : 0;
        if (lane == 0) q_scale[r] = scalbnf(1.0f, e);
        const float f = scalbnf(1.0f, -e);
        // value d of row r sits where the lane that multiplies it looks
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            const bool wide = d < D / 64 * 64;               // 64-wide blocks, then one of 32
            const int in64 = wide ? d % 64 : d % 32, tt = wide ? in64 / 16 : in64 / 8, byte = wide ? in64 % 16 : in64 % 8;
            const int step = (wide ? d / 64 * 4 : D / 64 * 4) + byte / 4;
            const int reg = (byte % 4) / 2 * 2 + r / 8;
            __half* at = reinterpret_cast<__half*>(q_frag + step * 32 + (r % 8) * 4 + tt) + reg * 2 + byte % 2;
            *at = __float2half_rn(x[i] * f);
        }
    }
    bar_init_done();
    __syncthreads();

    const long long block = (long long)P * D;                // bytes of a page's codes of one head
    auto fetch = [&](int entry) {                            // entry 2i: unit warp + i * warps' keys, 2i + 1: its values
        const int u = warp + (entry / 2) * kRowsWarps;
        if (u >= units) return;
        const uint32_t bar = bars + (entry % kRing) * 8, to = ring + (entry % kRing) * (kUnit * D);
        int n = 0;
#pragma unroll
        for (int i = 0; i < kPages; ++i) n += pages[u * kPages + i] >= 0;
        bar_expect(bar, (uint32_t)(n * block));
        const int8_t* from = entry % 2 ? p.c.v : p.c.k;
        for (int i = 0; i < n; ++i)                          // those past the end are the last ones
            bulk_load(to + (uint32_t)(i * block), from + ((long long)pages[u * kPages + i] * p.c.heads + h) * block,
                      (uint32_t)block, bar);
    };
    if (lane == 0)
        for (int e = 0; e < kRing; ++e) fetch(e);

    const float f0 = q_scale[g] * p.scale, f1 = q_scale[g + 8] * p.scale;
    float o[D / 8][4] = {}, m0 = -inf_f(), m1 = -inf_f(), l0 = 0.0f, l1 = 0.0f, vref = 0.0f;
    bool alive = true;
    for (int i = 0, u = warp; u < units; ++i, u += kRowsWarps) {
        // scores of 64 tokens: tile n's column c is token (c / 2) * (P / 4) +
        // 4 * group + 2 * half + c % 2 of its page, so that a lane ends up
        // with tokens that lie side by side in a value row
        float sc[kUnit / 8][4] = {};
        const int ek = 2 * i, ev = 2 * i + 1;
        alive = bar_wait_all(bars + (ek % kRing) * 8, (ek / kRing) & 1);
        if (!alive) break;
        const unsigned char* kt = smem + lay.ring + (warp * kRing + ek % kRing) * (kUnit * D);
#pragma unroll
        for (int c = 0; c < (D + 63) / 64; ++c) {
            constexpr int kWide = D / 64;
            const bool wide = c < kWide;
            uint32_t a[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (wide || j < 2) {
                    const uint4 v = q_frag[(c * 4 + j) * 32 + lane];
                    a[j][0] = v.x; a[j][1] = v.y; a[j][2] = v.z; a[j][3] = v.w;
                }
#pragma unroll
            for (int n = 0; n < kUnit / 8; ++n) {
                const int pg = n / (2 * kGroups), j16 = n / 2 % kGroups, hf = n % 2;
                const int token = pg * P + (g / 2) * (P / 4) + 4 * j16 + 2 * hf + g % 2;
                const unsigned char* at = kt + token * D + c * 64 + t * (wide ? 16 : 8);
                uint32_t w[4], lo, hi;
                if (wide) {
                    const uint4 v = *reinterpret_cast<const uint4*>(at);
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    w[0] = v.x; w[1] = v.y; w[2] = w[3] = 0;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (wide || j < 2) {
                        codes_to_f16(w[j], lo, hi);
                        mma_f16(sc[n], a[j], lo, hi);
                    }
            }
        }
        __syncwarp();
        if (lane == 0) fetch(ek + kRing);
        // softmax: a lane has columns 2t and 2t + 1 of rows g and g + 8
        const int base = begin + u * kUnit;
        float vnew = vref;
#pragma unroll
        for (int pg = 0; pg < kPages; ++pg) vnew = fmaxf(vnew, v_scale[u * kPages + pg]);
        float t0 = m0, t1 = m1;
        const bool partial = base + kUnit > min(lim0, lim1);
#pragma unroll
        for (int n = 0; n < kUnit / 8; ++n) {
            const int pg = n / (2 * kGroups), j16 = n / 2 % kGroups, hf = n % 2;
            const float ks = k_scale[u * kPages + pg];
            const int token = base + pg * P + t * (P / 4) + 4 * j16 + 2 * hf;
            sc[n][0] *= f0 * ks;
            sc[n][1] *= f0 * ks;
            sc[n][2] *= f1 * ks;
            sc[n][3] *= f1 * ks;
            if (partial) {
                if (token >= lim0) sc[n][0] = -inf_f();
                if (token + 1 >= lim0) sc[n][1] = -inf_f();
                if (token >= lim1) sc[n][2] = -inf_f();
                if (token + 1 >= lim1) sc[n][3] = -inf_f();
            }
            t0 = fmaxf(t0, fmaxf(sc[n][0], sc[n][1]));
            t1 = fmaxf(t1, fmaxf(sc[n][2], sc[n][3]));
        }
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        const float r0 = t0 == -inf_f() ? 0.0f : t0, r1 = t1 == -inf_f() ? 0.0f : t1;   // nothing seen yet
        const float e0 = exp2f(m0 - r0), e1 = exp2f(m1 - r1);
        const float grow = vnew > 0.0f ? vref / vnew : 1.0f;
        m0 = t0;
        m1 = t1;
        l0 *= e0;
        l1 *= e1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= e0 * grow;
            o[n][1] *= e0 * grow;
            o[n][2] *= e1 * grow;
            o[n][3] *= e1 * grow;
        }
        vref = vnew;
        uint32_t w[kUnit / 8][2];
#pragma unroll
        for (int n = 0; n < kUnit / 8; ++n) {
            const int pg = n / (2 * kGroups);
            const float vs = v_scale[u * kPages + pg], f = vnew > 0.0f ? vs / vnew : vs;
            float x[4] = {exp2f(sc[n][0] - r0), exp2f(sc[n][1] - r0), exp2f(sc[n][2] - r1), exp2f(sc[n][3] - r1)};
            l0 += x[0] + x[1];
            l1 += x[2] + x[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = partial && x[j] == 0.0f ? 0.0f : x[j] * f;   // a scale that is not a number stays with those who see it
            w[n][0] = pack_f16(x[0], x[1]);
            w[n][1] = pack_f16(x[2], x[3]);
        }
        alive = bar_wait_all(bars + (ev % kRing) * 8, (ev / kRing) & 1);
        if (!alive) break;
        const unsigned char* vt = smem + lay.ring + (warp * kRing + ev % kRing) * (kUnit * D);
#pragma unroll
        for (int pg = 0; pg < kPages; ++pg)
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                const unsigned char* at = vt + pg * P * D + (n * 8 + g) * P + t * (P / 4);
                uint32_t c[4];
                if constexpr (P == 64) {
                    const uint4 v = *reinterpret_cast<const uint4*>(at);
                    c[0] = v.x; c[1] = v.y; c[2] = v.z; c[3] = v.w;
                } else if constexpr (P == 32) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    c[0] = v.x; c[1] = v.y;
                } else {
                    c[0] = *reinterpret_cast<const uint32_t*>(at);
                }
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    const int s0 = pg * 2 * kGroups + 2 * j;
                    const uint32_t a[4] = {w[s0][0], w[s0][1], w[s0 + 1][0], w[s0 + 1][1]};
                    uint32_t lo, hi;
                    codes_to_f16(c[j], lo, hi);
                    mma_f16(o[n], a, lo, hi);
                }
            }
        __syncwarp();
        if (lane == 0) fetch(ev + kRing);
    }
    // a wait that ran out: the copies in flight get as long again to end
    if (!alive)
        for (int e = 0; e < kRing; ++e)
            for (int ph = 0; ph < 2; ++ph) bar_wait(bars + e * 8, ph);
    // join the warps (every copy that was begun has been waited for)
    const bool dead = __syncthreads_or(!alive);
    float* sums = reinterpret_cast<float*>(smem);            // [warp][row][D], then [warp][row][2]
    float* tops = sums + kRowsWarps * 16 * D;
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (!dead) {
        float* to = sums + (warp * 16 + g) * D + 2 * t;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            to[n * 8] = o[n][0] * vref;
            to[n * 8 + 1] = o[n][1] * vref;
            to[n * 8 + 8 * D] = o[n][2] * vref;
            to[n * 8 + 8 * D + 1] = o[n][3] * vref;
        }
        if (t == 0) {
            tops[(warp * 16 + g) * 2] = m0;
            tops[(warp * 16 + g) * 2 + 1] = l0;
            tops[(warp * 16 + g + 8) * 2] = m1;
            tops[(warp * 16 + g + 8) * 2 + 1] = l1;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(rows, 16) * D; i += kRowsWarps * 32) {
        const int r = i / D, d = i % D, row = tile * 16 + r;
        float top = -inf_f(), sum = 0.0f, l = 0.0f;
        if (dead || s.kept < 0) {
            sum = l = nan_f();
        } else {
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, tops[(w * 16 + r) * 2]);
            const float ref = top == -inf_f() ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float e = exp2f(tops[(w * 16 + r) * 2] - ref);
                sum += e * sums[(w * 16 + r) * D + d];
                l += e * tops[(w * 16 + r) * 2 + 1];
            }
        }
        const long long token = s.first + row / group;
        const int head = h * group + row % group;
        if (split) {
            float* to = p.scratch + ((token * p.heads + head) * gridDim.x + blockIdx.x) * (D + 2);
            to[2 + d] = sum;
            if (d == 0) {
                to[0] = top;
                to[1] = l;
            }
        } else {
            store_value(p.out, token * p.out_token + head * p.out_head + d, p.type, l == 0.0f ? 0.0f : sum / l);
        }
    }
}

// One warp for each row and head: its chunks' sums, joined.
__global__ void __launch_bounds__(128) k_attend_join(AttendParams p, int chunk, int count, int tile) {
    const int lane = threadIdx.x % 32, group = p.heads / p.c.heads, dim = p.c.dim;
    const long long i = (long long)blockIdx.x * 4 + threadIdx.x / 32;
    chain_wait();
    if (i >= p.r.total * p.heads) return;
    const long long token = i / p.heads;
    const int head = (int)(i % p.heads);
    // the row's sequence: the last whose first row is not past it
    int lo = 0, hi = p.r.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (p.r.starts[mid] <= token) lo = mid; else hi = mid - 1;
    }
    const Queries s = queries_of(p, lo);
    if (token < s.first || token >= s.first + s.rows) return;
    const int at = (int)(token - s.first);
    const long long out = token * p.out_token + head * p.out_head;
    if (s.kept < 0) {
        for (int d = lane; d < dim; d += 32) store_value(p.out, out + d, p.type, nan_f());
        return;
    }
    // the chunks that the row's tile has: up to the tokens its last row sees
    const int row = at * group + head % group, last = min(row / tile * tile + tile - 1, s.rows * group - 1) / group;
    const int sees = p.causal ? max(0, s.kept - s.rows + last + 1) : s.kept;
    const int n = min((sees + chunk - 1) / chunk, count);
    const float* from = p.scratch + i * count * (dim + 2);
    float top = -inf_f(), l = 0.0f;
    for (int c = 0; c < n; ++c) top = fmaxf(top, from[(long long)c * (dim + 2)]);
    const float ref = top == -inf_f() ? 0.0f : top;
    for (int c = 0; c < n; ++c) l += exp2f(from[(long long)c * (dim + 2)] - ref) * from[(long long)c * (dim + 2) + 1];
    for (int d = lane; d < dim; d += 32) {
        float sum = 0.0f;
        for (int c = 0; c < n; ++c)
            sum += exp2f(from[(long long)c * (dim + 2)] - ref) * from[(long long)c * (dim + 2) + 2 + d];
        store_value(p.out, out + d, p.type, l == 0.0f ? 0.0f : sum / l);
    }
}

template <int D, int P>
cudaError_t rows_launch(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    const RowsLayout lay = rows_layout(D, c.tokens, P);
    const long long tiles = ((long long)p.r.most * (p.heads / p.c.heads) + 15) / 16;
    const dim3 grid(c.count, (unsigned)(tiles * p.c.heads), p.r.seqs);
    cudaError_t e = allow_shared<k_attend_rows<D, P>>((int)rows_layout(D, kMostChunk, P).bytes);
    if (e != cudaSuccess) return e;
    k_attend_rows<D, P><<<grid, kRowsWarps * 32, lay.bytes, s>>>(p, c.tokens);
    return cudaGetLastError();
}

template <int D>
cudaError_t by_page(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    switch (p.c.page) {
        case 16: return rows_launch<D, 16>(p, c, s);
        case 32: return rows_launch<D, 32>(p, c, s);
        default: return rows_launch<D, 64>(p, c, s);
    }
}

cudaError_t by_dim(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    switch (p.c.dim) {
        case 32: return by_page<32>(p, c, s);
        case 64: return by_page<64>(p, c, s);
        case 96: return by_page<96>(p, c, s);
        case 128: return by_page<128>(p, c, s);
        case 192: return by_page<192>(p, c, s);
        default: return by_page<256>(p, c, s);
    }
}

}  // namespace

bool attend_dim_ok(int dim) { return dim == 32 || dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256; }

// Many rows go to the tile kernel where it has the head's size; up to 16 rows
// fill one tile of this file's kernel, which reads the cache as fast.
bool use_tiles(int dim, int heads, int kv_heads, int most) {
    return attend_tiles_dim(dim) && (long long)most * (heads / kv_heads) > 16;
}

Chunks plan(int dim, int heads, int kv_heads, int seqs, int most, int most_kept) {
    return use_tiles(dim, heads, kv_heads, most) ? plan_tiles(heads, kv_heads, seqs, most, most_kept)
                                                 : plan_chunks(heads, kv_heads, seqs, most, most_kept);
}

// the grid's y counts tiles of 16 rows
bool attend_fits(int dim, int heads, int kv_heads, int most) {
    return use_tiles(dim, heads, kv_heads, most) || ((long long)most * (heads / kv_heads) + 15) / 16 * kv_heads <= 65535;
}

size_t attend_scratch_bytes(long long total, int heads, int kv_heads, int dim, int seqs, int most, int most_kept) {
    const Chunks c = plan(dim, heads, kv_heads, seqs, most, most_kept);
    return c.count == 1 ? 0 : (size_t)total * heads * c.count * (dim + 2) * sizeof(float);
}

cudaError_t launch_cache_attention(const AttendParams& p, cudaStream_t s) {
    const bool tiles = use_tiles(p.c.dim, p.heads, p.c.heads, p.r.most);
    const Chunks c = plan(p.c.dim, p.heads, p.c.heads, p.r.seqs, p.r.most, p.most_kept);
    const cudaError_t e = tiles ? launch_attend_tiles(p, c, s) : by_dim(p, c, s);
    if (e != cudaSuccess || c.count == 1) return e;
    const long long n = p.r.total * p.heads;
    const int rows = tiles ? tile_rows((long long)p.r.most * (p.heads / p.c.heads)) : 16;
    return launch_after(k_attend_join, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, s, p, c.tokens, c.count, rows);
}

}  // namespace vdt

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
// f16 value whole down to 2^-14 of that (below, to 2^-24 of it).
//
// A token's weight is its score's power and its page's vs together, in powers
// of two: 2^(s + log2(vs)), and it is made relative to the largest such weight
// that its own row sees (2^o).  A page that the row does not see, or that has
// next to no probability, then takes no bits from the others however large its
// values are.  The 16-bit weight is off by at most 2^-11 of itself, or, below
// 2^-14 of the largest, by 2^-25 of that: the former is the rounding of an f16
// output, an eighth of a bf16 one's, and it averages over the tokens.  The
// weights' own sum is 32-bit and relative to the largest score (2^m): a page's
// weights before the rounding, times 2^(o - m) / vs.
//
// m and o are not the running maxima themselves: they move only when a row
// passes one of them by more than 2^8 (as a factor); 16-bit floats have room
// for that, and the sums are rescaled a few times instead of at every step.
#include "attend_internal.h"

namespace vdt {
namespace {

constexpr int kUnit = 64;          // tokens that a warp takes at a time

// ------------------------------------------------------------ few query rows
// One CTA: a sequence, a head of the cache, up to 8 x NR of the rows (query,
// head of the group) that share it, and a chunk of the tokens.  Its warps take
// units of 64 tokens in turn; each warp has its own ring of shared memory, into
// which the units' codes are copied in bulk (a page's codes of one head are
// consecutive).  The warps' sums are joined in shared memory, the chunks' by
// k_attend_join.
//
// Bound by memory where the caches are long: 64 sequences of 1,023 to 8,191
// tokens, 32 heads of 128 over 8, take 110 us, 5.6 TB/s of codes (floor 95);
// the warps' instructions (some 1,100 for 64 tokens of 128 values, half of them
// the codes' way to 16 bits) come close behind, and the start and end of a CTA.
//
// Tokens are the rows of the first product (S^T = K Q^T) and values' dimensions
// those of the second (O^T = V^T P^T), the queries the columns, eight at a time:
// the codes, turned into 16-bit floats once, serve all the queries, and one
// query costs half of what 16 would.  A lane ends up with tokens that lie side
// by side in a value row: row m of 16 is token (m % 8 / 2) (P / 4) + 4 j + (m /
// 8) 2 + m % 2 of its page, j counting the page's groups of 16.
constexpr int kRowsWarps = 4;
constexpr int kRing = 2;           // entries of a warp's ring; a unit's keys are one, its values one
constexpr int kMostChunk = 4096;   // tokens of a chunk: bounds the page lists in shared memory

// groups of eight rows of a CTA
int row_groups(long long rows) { return rows <= 8 ? 1 : 2; }

// Fewer tiles than the SMs have room for (three CTAs each, as heads of up to 128
// have it): as many chunks as fill it once (a second round of a few CTAs costs as
// much as the first: 100,000 tokens in 66 chunks of 8 heads of 128 took 63 us, in 49
// 50 us).  More tiles: chunks of about 2048 tokens, which even out sequences of
// different lengths (64 of 1,000 to 8,191 tokens: 121 us with 1536 or 2048, 127 with
// 2816).  None under 64 tokens a warp.  With one chunk the CTAs write the output
// themselves.
//
// Of heads of 192 two CTAs fit, of 256 one, and three are counted for them as well:
// sequences of different lengths gain by the more chunks what a long one alone
// loses (us, with three and with what fits: 16 of 1,400 to 8,000 tokens, 8 cached
// heads of 192 49 and 59, of 256 70 and 77; one of 100,000, 8 of 192 75 and 60, of 256
// 94 and 100; one of 30,000, 4 of 256 32 and 24).
constexpr int kEvenChunk = 2048;

Chunks plan_chunks(int heads, int kv_heads, int seqs, int most, int most_kept) {
    const long long rows = (long long)most * (heads / kv_heads), each = 8 * row_groups(rows);
    const long long tiles = kv_heads * seqs * ((rows + each - 1) / each), slots = 3 * kSmCount;
    const long long want = tiles < slots ? slots / tiles : ((long long)most_kept + kEvenChunk - 1) / kEvenChunk;
    long long tokens = ((long long)most_kept + want - 1) / (want ? want : 1);
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
// an 8 x 8 block of 16-bit values, a row's pair a lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int N>
__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(at);
    }
}

struct RowsLayout {
    uint32_t q, bars, pages, bytes;          // the ring is first
};
__host__ __device__ inline RowsLayout rows_layout(int dim, int groups, int chunk, int page) {
    RowsLayout l;
    const uint32_t ring = (uint32_t)(kRowsWarps * kRing * kUnit * dim);
    const uint32_t sums = (uint32_t)(kRowsWarps * 8 * groups * (dim + 2) * 4);     // reuses the ring
    l.q = ring > sums ? ring : sums;
    l.bars = l.q + dim * 16 * groups + 32 * groups;
    l.pages = l.bars + kRowsWarps * kRing * 8;
    l.bytes = l.pages + chunk / page * 12;
    return l;
}

template <int D, int P, int NR>
__global__ void __launch_bounds__(kRowsWarps * 32) k_attend_rows(AttendParams p, int chunk) {
    extern __shared__ __align__(128) unsigned char smem[];
    chain_release();
    constexpr int kGroups = P / 16;              // 16-token groups of a page
    constexpr int kPages = kUnit / P;            // pages of a unit
    constexpr int kRows = 8 * NR;
    constexpr int kPart = kUnit / 16;            // 16-token groups of a unit
    const RowsLayout lay = rows_layout(D, NR, chunk, P);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int b = blockIdx.z, group = p.heads / p.c.heads;
    const int tile = blockIdx.y / p.c.heads, h = blockIdx.y % p.c.heads;
    const Queries s = queries_of(p, b);
    const int rows = s.rows * group - tile * kRows;           // rows of this tile
    if (rows <= 0) {
        if (s.rows == 0 && blockIdx.x == 0 && tile == 0) spoil_run(p, b, h);       // nothing to do for an empty run
        return;
    }
    const bool split = gridDim.x > 1;
    // tokens that a row sees: all, or up to its own place at the sequence's end
    auto sees = [&](int r) {
        if (r >= rows || s.kept < 0) return 0;
        return p.causal ? max(0, s.kept - s.rows + (tile * kRows + r) / group + 1) : s.kept;
    };
    const int begin = blockIdx.x * chunk, end = min(begin + chunk, sees(min(rows, kRows) - 1));
    if (begin >= end && split) return;                        // the join knows as well
    const int units = max(0, (end - begin + kUnit - 1) / kUnit);
    int limit[NR][2], least = 0x7fffffff;                     // of the lane's columns; of all rows there are
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) limit[n][i] = sees(8 * n + 2 * t + i);
    least = sees(0);

    float* q_scale = reinterpret_cast<float*>(smem + lay.q + D * 16 * NR);
    uint2* q_frag = reinterpret_cast<uint2*>(smem + lay.q);
    int* pages = reinterpret_cast<int*>(smem + lay.pages);
    float* k_scale = reinterpret_cast<float*>(pages + chunk / P);
    float* v_log = k_scale + chunk / P;
    const uint32_t bars = shared_address(smem + lay.bars) + warp * kRing * 8;
    const uint32_t ring = shared_address(smem) + warp * kRing * kUnit * D;

    if (lane < kRing) bar_init(bars + lane * 8, 1);
    // the chunk's pages: number, scale, logarithm of the values' scale; one
    // that is not in the cache is read as page 0 under scales that are not
    // numbers, one past the end is not read at all
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
        v_log[i] = vs > 0.0f ? log2f(vs) : vs == 0.0f ? -inf_f() : nan_f();
    }
    // the queries, each row scaled by a power of two
    for (int r = warp; r < kRows; r += kRowsWarps) {
        float x[D / 32], m = 0.0f;
        const bool in = r < rows;
        const int row = tile * kRows + r;
        const long long q = (s.first + row / group) * p.q_token + (long long)(h * group + row % group) * p.q_head;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = in ? load_value(p.q, q + lane + 32 * i, p.type) : 0.0f;
            m = fmaxf(m, fabsf(x[i]));
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const int e = m > 0.0f && m < inf_f() ? max(-126, min(126, ilogbf(m))) : 0;
        if (lane == 0) q_scale[r] = scalbnf(fabsf(p.scale), e);
        const float f = copysignf(scalbnf(1.0f, -e), p.scale);        // a negative scale goes into the queries
        // value d of row r sits where the lane that multiplies it looks
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            const bool wide = d < D / 64 * 64;               // 64-wide blocks, then one of 32
            const int in64 = wide ? d % 64 : d % 32, tt = wide ? in64 / 16 : in64 / 8, byte = wide ? in64 % 16 : in64 % 8;
            const int step = (wide ? d / 64 * 4 : D / 64 * 4) + byte / 4;
            __half* at = reinterpret_cast<__half*>(q_frag + (step * NR + r / 8) * 32 + (r % 8) * 4 + tt) + byte % 4;
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

    // the lane's columns: factor, what their sum (2^ref) and the outputs
    // (2^(ref + vref)) are relative to, the weights' sum
    float f[NR][2], ref[NR][2], vref[NR][2], sum[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[n][i] = q_scale[8 * n + 2 * t + i];
            ref[n][i] = vref[n][i] = -inf_f();
            sum[n][i] = 0.0f;
        }
    float o[D / 16][NR][4] = {};
    bool alive = true;
    for (int i = 0, u = warp; u < units; ++i, u += kRowsWarps) {
        const int ek = 2 * i, ev = 2 * i + 1, base = begin + u * kUnit;
        const bool partial = base + kUnit > least;
        const unsigned char* kt = smem + (warp * kRing + ek % kRing) * (kUnit * D);
        const unsigned char* vt = smem + (warp * kRing + ev % kRing) * (kUnit * D);
        alive = bar_wait_all(bars + (ek % kRing) * 8, (ek / kRing) & 1);
        if (!alive) break;
        {
            float sc[kPart][NR][4] = {};
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c) {
                constexpr int kWide = D / 64;
                const bool wide = c < kWide;
                uint32_t x[kPart][4], y[kPart][4];           // of tokens m and m + 8 of 16
#pragma unroll
                for (int m = 0; m < kPart; ++m) {
                    const int pg = m / kGroups, j16 = m % kGroups;
                    const unsigned char* at = kt + (pg * P + (g / 2) * (P / 4) + 4 * j16 + g % 2) * D + c * 64 + t * (wide ? 16 : 8);
                    if (wide) {
                        const uint4 a = *reinterpret_cast<const uint4*>(at), d = *reinterpret_cast<const uint4*>(at + 2 * D);
                        x[m][0] = a.x; x[m][1] = a.y; x[m][2] = a.z; x[m][3] = a.w;
                        y[m][0] = d.x; y[m][1] = d.y; y[m][2] = d.z; y[m][3] = d.w;
                    } else {
                        const uint2 a = *reinterpret_cast<const uint2*>(at), d = *reinterpret_cast<const uint2*>(at + 2 * D);
                        x[m][0] = a.x; x[m][1] = a.y;
                        y[m][0] = d.x; y[m][1] = d.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if (!wide && w >= 2) continue;
                    uint2 q[NR];
#pragma unroll
                    for (int n = 0; n < NR; ++n) q[n] = q_frag[((c * 4 + w) * NR + n) * 32 + lane];
#pragma unroll
                    for (int m = 0; m < kPart; ++m) {
                        uint32_t a[4];
                        codes_to_f16(x[m][w], a[0], a[2]);
                        codes_to_f16(y[m][w], a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NR; ++n) mma_f16(sc[m][n], a, q[n].x, q[n].y);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) fetch(ek + kRing);
            // scores, in powers of two; the lane's tokens are base + page + t' (P / 4) + ... of rows g and g + 8
            bool over = false;
            float top[NR][2], v_top[NR][2];                  // largest score; largest with its page's value scale
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) top[n][e] = v_top[n][e] = -inf_f();
#pragma unroll
            for (int pg = 0; pg < kPages; ++pg) {
                const float ks = k_scale[u * kPages + pg], vl = v_log[u * kPages + pg];
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float most[2] = {-inf_f(), -inf_f()};
#pragma unroll
                    for (int m = pg * kGroups; m < (pg + 1) * kGroups; ++m) {
                        const int token = base + pg * P + (g / 2) * (P / 4) + 4 * (m % kGroups) + g % 2;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = sc[m][n][e] * (f[n][e % 2] * ks);
                            if (partial) v = token + e / 2 * 2 < limit[n][e % 2] ? v : -inf_f();
                            sc[m][n][e] = v;
                            most[e % 2] = fmaxf(most[e % 2], v);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        top[n][e] = fmaxf(top[n][e], most[e]);
                        v_top[n][e] = fmaxf(v_top[n][e], most[e] + vl);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) over = over || passes(top[n][e], ref[n][e]) || passes(v_top[n][e], ref[n][e] + vref[n][e]);
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = top[n][e], y = v_top[n][e];
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) {
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                        }
                        const Rescale by = move_references(x, y, ref[n][e], vref[n][e]);
                        sum[n][e] *= by.sum;
#pragma unroll
                        for (int m = 0; m < D / 16; ++m) {
                            o[m][n][e] *= by.out;
                            o[m][n][e + 2] *= by.out;
                        }
                    }
            }
            alive = bar_wait_all(bars + (ev % kRing) * 8, (ev / kRing) & 1);
            if (!alive) break;
            uint32_t w[kPart][NR][2];
            float of_page[NR][2];                            // a page's weights, summed
#pragma unroll
            for (int m = 0; m < kPart; ++m) {
                const int pg = m / kGroups, j16 = m % kGroups;
                const int token = base + pg * P + (g / 2) * (P / 4) + 4 * j16 + g % 2;
                const float vl = v_log[u * kPages + pg];
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float x[4], d[2], r[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        d[e] = page_shift(vl, vref[n][e]);
                        r[e] = ref[n][e] == -inf_f() ? 0.0f : ref[n][e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = exp2_fast(sc[m][n][e] - r[e % 2] + d[e % 2]);
                        if (partial) x[e] = token + e / 2 * 2 < limit[n][e % 2] ? x[e] : 0.0f;     // also for scales that are not numbers
                    }
                    const float a = x[0] + x[2], c = x[1] + x[3];
                    of_page[n][0] = j16 == 0 ? a : of_page[n][0] + a;
                    of_page[n][1] = j16 == 0 ? c : of_page[n][1] + c;
                    if (j16 == kGroups - 1)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            sum[n][e] = partial && of_page[n][e] == 0.0f ? sum[n][e] : fmaf(of_page[n][e], exp2_fast(-d[e]), sum[n][e]);
                    w[m][n][0] = transposed(pack_f16(x[0], x[1]));
                    w[m][n][1] = transposed(pack_f16(x[2], x[3]));
                }
            }
            // a value row's tokens of kRun groups lie side by side
            constexpr int kRun = kGroups < kPart ? kGroups : kPart;
#pragma unroll
            for (int m0 = 0; m0 < kPart; m0 += kRun) {
                const int pg = m0 / kGroups, j16 = m0 % kGroups;
                const unsigned char* at = vt + pg * P * D + g * P + t * (P / 4) + 4 * j16;
#pragma unroll
                for (int q = 0; q < D / 16; ++q) {
                    uint32_t x[kRun], y[kRun];               // of dimensions m and m + 8 of 16
                    load_words<kRun>(at + q * 16 * P, x);
                    load_words<kRun>(at + (q * 16 + 8) * P, y);
#pragma unroll
                    for (int m = 0; m < kRun; ++m) {
                        uint32_t a[4];
                        codes_to_f16(x[m], a[0], a[2]);
                        codes_to_f16(y[m], a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NR; ++n) mma_f16(o[q][n], a, w[m0 + m][n][0], w[m0 + m][n][1]);
                    }
                }
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
    float* tops = sums + kRowsWarps * kRows * D;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float v_scale = exp2f(vref[n][e] - kSlack);          // 2^vref may be too large for 32 bits where its product is not
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], d);
            const int row = warp * kRows + 8 * n + 2 * t + e;
            if (!dead) {
#pragma unroll
                for (int m = 0; m < D / 16; ++m) {
                    sums[row * D + m * 16 + g] = o[m][n][e] * v_scale * kSlackFactor;
                    sums[row * D + m * 16 + g + 8] = o[m][n][e + 2] * v_scale * kSlackFactor;
                }
                if (g == 0) {
                    tops[row * 2] = ref[n][e];
                    tops[row * 2 + 1] = sum[n][e];
                }
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < min(rows, kRows) * D; i += kRowsWarps * 32) {
        const int r = i / D, d = i % D, row = tile * kRows + r;
        float top = -inf_f(), sum = 0.0f, l = 0.0f;
        if (dead || s.kept < 0) {
            sum = l = nan_f();
        } else {
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, tops[(w * kRows + r) * 2]);
            const float to = top == -inf_f() ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float e = exp2f(tops[(w * kRows + r) * 2] - to);
                sum += e * sums[(w * kRows + r) * D + d];
                l += e * tops[(w * kRows + r) * 2 + 1];
            }
        }
        const long long token = s.first + row / group;
        const int head = h * group + row % group;
        if (split) {
            const Partial to = partial_of(p, token * p.heads + head, gridDim.x, blockIdx.x);
            to.sums[d] = sum;
            if (d == 0) *to.stats = make_float2(top, l);
        } else {
            store_value(p.out, token * p.out_token + head * p.out_head + d, p.type, l == 0.0f ? 0.0f : sum / l);
        }
    }
}

// A packed row and head whose chunks are to be joined
struct JoinRow {
    long long out;          // where its output starts
    int chunks;             // -1: no such row; -2: more tokens than the table or most_kept allow
};
__device__ __forceinline__ JoinRow join_row(const AttendParams& p, long long token, int head, int chunk, int count, int tile) {
    const int lane = threadIdx.x % 32, group = p.heads / p.c.heads;
    // its sequence: the last whose first row is not past it (the lanes look at 32 at a time)
    int seq = -1;
    for (int j = 0; j < p.r.seqs; j += 32) {
        const unsigned not_past = __ballot_sync(0xffffffffu, j + lane < p.r.seqs && p.r.starts[j + lane] <= token);
        if (not_past) seq = j + 31 - __clz(not_past);
        if (not_past != 0xffffffffu) break;
    }
    if (seq < 0) return {0, -1};
    const Queries s = queries_of(p, seq);
    if (token < s.first || token >= s.first + s.rows) return {0, -1};
    // the chunks that the row's tile has: up to the tokens its last row sees
    const int row = (int)(token - s.first) * group + head % group, last = min(row / tile * tile + tile - 1, s.rows * group - 1) / group;
    const int sees = p.causal ? max(0, s.kept - s.rows + last + 1) : s.kept;
    return {token * p.out_token + head * p.out_head, s.kept < 0 ? -2 : min((sees + chunk - 1) / chunk, count)};
}

// Four of a lane's values; lane + 32 i counts groups of four
__device__ __forceinline__ void add_four(float (&sum)[4], const float4& v, float f) {
    sum[0] = fmaf(f, v.x, sum[0]);
    sum[1] = fmaf(f, v.y, sum[1]);
    sum[2] = fmaf(f, v.z, sum[2]);
    sum[3] = fmaf(f, v.w, sum[3]);
}

// Up to 32 chunks: a warp a row, a lane a chunk's maximum and sum.
__global__ void __launch_bounds__(128) k_attend_join_few(AttendParams p, int chunk, int count, int tile) {
    const int lane = threadIdx.x % 32, four = p.c.dim / 4;
    const long long i = (long long)blockIdx.x * 4 + threadIdx.x / 32;
    const bool in = i < p.r.total * p.heads;
    const JoinRow r = in ? join_row(p, i / p.heads, (int)(i % p.heads), chunk, count, tile) : JoinRow{0, -1};
    chain_wait();                            // before any return: what follows on the stream may count on it
    if (r.chunks == -1) return;
    const Partial from = partial_of(p, i, count, 0);
    const float2 own = lane < r.chunks ? from.stats[lane] : make_float2(-inf_f(), 0.0f);
    float top = own.x;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float factor = exp2f(own.x - (top == -inf_f() ? 0.0f : top));
    float l = factor * own.y, sum[2][4] = {};
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    for (int c0 = 0; c0 < r.chunks; c0 += 4) {
        float4 v[4][2];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                v[c][j] = c0 + c < r.chunks && lane + 32 * j < four
                              ? reinterpret_cast<const float4*>(from.sums + (long long)(c0 + c) * p.c.dim)[lane + 32 * j]
                              : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float f = __shfl_sync(0xffffffffu, factor, c0 + c);
#pragma unroll
            for (int j = 0; j < 2; ++j) add_four(sum[j], v[c][j], f);
        }
    }
    if (r.chunks == -2) l = nan_f();
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (lane + 32 * j < four)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                store_value(p.out, r.out + (lane + 32 * j) * 4 + e, p.type, l == 0.0f ? 0.0f : sum[j][e] / l);
}

// More chunks: a CTA a row.  The chunks' factors are made by all threads and
// kept in shared memory; then each warp adds up every fourth chunk, eight of
// them in flight.
constexpr int kJoinThreads = 128, kJoinChunks = 512;

__global__ void __launch_bounds__(kJoinThreads) k_attend_join(AttendParams p, int chunk, int count, int tile) {
    __shared__ float factor[kJoinChunks], part[4][256], side[2][4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, four = p.c.dim / 4;
    const JoinRow r = join_row(p, blockIdx.x / p.heads, blockIdx.x % p.heads, chunk, count, tile);
    chain_wait();
    if (r.chunks == -1) return;
    float top = -inf_f(), l = 0.0f, sum[2][4] = {};
    for (int first = 0; first < r.chunks; first += kJoinChunks) {
        const int here = min(r.chunks - first, kJoinChunks);
        const Partial from = partial_of(p, blockIdx.x, count, first);
        constexpr int kEach = kJoinChunks / kJoinThreads;
        float2 v[kEach];
        float most = top;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int c = threadIdx.x + i * kJoinThreads;
            v[i] = c < here ? from.stats[c] : make_float2(-inf_f(), 0.0f);
            most = fmaxf(most, v[i].x);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        __syncthreads();
        if (lane == 0) side[0][warp] = most;
        __syncthreads();
        most = fmaxf(fmaxf(side[0][0], side[0][1]), fmaxf(side[0][2], side[0][3]));
        const float ref = most == -inf_f() ? 0.0f : most, by = exp2f(top - ref);
        top = most;
        l *= by;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[j][e] *= by;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float f = exp2f(v[i].x - ref);
            factor[threadIdx.x + i * kJoinThreads] = f;       // 0 past the last
            l += f * v[i].y;
        }
        __syncthreads();
        for (int c0 = warp; c0 < here; c0 += 32) {
            float4 x[8][2];
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    x[c][j] = c0 + 4 * c < here && lane + 32 * j < four
                                  ? reinterpret_cast<const float4*>(from.sums + (long long)(c0 + 4 * c) * p.c.dim)[lane + 32 * j]
                                  : make_float4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float f = c0 + 4 * c < here ? factor[c0 + 4 * c] : 0.0f;
#pragma unroll
                for (int j = 0; j < 2; ++j) add_four(sum[j], x[c][j], f);
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (lane == 0) side[1][warp] = l;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[warp][(lane + 32 * j) * 4 + e] = sum[j][e];
    __syncthreads();
    l = (side[1][0] + side[1][1]) + (side[1][2] + side[1][3]);
    if (r.chunks == -2) l = nan_f();
    for (int d = threadIdx.x; d < p.c.dim; d += kJoinThreads) {
        const float x = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
        store_value(p.out, r.out + d, p.type, l == 0.0f ? 0.0f : x / l);
    }
}

template <int D, int P, int NR>
cudaError_t rows_launch(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    const RowsLayout lay = rows_layout(D, NR, c.tokens, P);
    const long long rows = (long long)p.r.most * (p.heads / p.c.heads), tiles = (rows + 8 * NR - 1) / (8 * NR);
    const dim3 grid(c.count, (unsigned)(tiles * p.c.heads), p.r.seqs);
    const cudaError_t e = allow_shared<k_attend_rows<D, P, NR>>((int)rows_layout(D, NR, kMostChunk, P).bytes);
    if (e != cudaSuccess) return e;
    k_attend_rows<D, P, NR><<<grid, kRowsWarps * 32, lay.bytes, s>>>(p, c.tokens);
    return cudaGetLastError();
}

template <int D, int P>
cudaError_t by_rows(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    return row_groups((long long)p.r.most * (p.heads / p.c.heads)) == 1 ? rows_launch<D, P, 1>(p, c, s) : rows_launch<D, P, 2>(p, c, s);
}

template <int D>
cudaError_t by_page(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    switch (p.c.page) {
        case 16: return by_rows<D, 16>(p, c, s);
        case 32: return by_rows<D, 32>(p, c, s);
        default: return by_rows<D, 64>(p, c, s);
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

// Up to 16 rows go to this file's kernel, more to the tile kernel: with 32 rows
// of 16 heads of 64 over 16 caches of up to 1500 tokens this one (made for four
// groups of eight rows) took 45 us, with 32 of 128 over 2000 tokens 28 us; the
// tile kernel 38 and 24.
bool use_tiles(int heads, int kv_heads, int most) { return (long long)most * (heads / kv_heads) > 16; }

Chunks plan(int dim, int heads, int kv_heads, int seqs, int most, int most_kept) {
    return use_tiles(heads, kv_heads, most) ? plan_tiles(dim, heads, kv_heads, seqs, most, most_kept)
                                                 : plan_chunks(heads, kv_heads, seqs, most, most_kept);
}

// the grid's y counts tiles of rows
bool attend_fits(int dim, int heads, int kv_heads, int most) {
    const long long rows = (long long)most * (heads / kv_heads), each = 8 * row_groups(rows);
    return use_tiles(heads, kv_heads, most) || (rows + each - 1) / each * kv_heads <= 65535;
}

size_t attend_scratch_bytes(long long total, int heads, int kv_heads, int dim, int seqs, int most, int most_kept) {
    const Chunks c = plan(dim, heads, kv_heads, seqs, most, most_kept);
    return c.count == 1 ? 0 : (size_t)partial_floats((long long)total * heads, c.count, dim) * sizeof(float);
}

cudaError_t launch_cache_attention(const AttendParams& p, cudaStream_t s) {
    const bool tiles = use_tiles(p.heads, p.c.heads, p.r.most);
    const Chunks c = plan(p.c.dim, p.heads, p.c.heads, p.r.seqs, p.r.most, p.most_kept);
    const cudaError_t e = tiles ? launch_attend_tiles(p, c, s) : by_dim(p, c, s);
    if (e != cudaSuccess || c.count == 1) return e;
    const long long n = p.r.total * p.heads, rows = (long long)p.r.most * (p.heads / p.c.heads);
    const int tile = tiles ? tile_rows(p.c.dim, rows) : 8 * row_groups(rows);
    if (c.count <= 32) return launch_after(k_attend_join_few, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, s, p, c.tokens, c.count, tile);
    return launch_after(k_attend_join, dim3((unsigned)n), dim3(kJoinThreads), 0, s, p, c.tokens, c.count, tile);
}

}  // namespace vdt

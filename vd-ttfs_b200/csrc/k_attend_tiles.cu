// k_attend_tiles.cu -- attention over the paged 8-bit cache for many query
// rows, on the fifth-generation tensor cores (mathematics: k_attend.cu).
//
// One CTA: a sequence, a head of the cache, one or two tiles of 128 of the
// rows (query, head of the group) that share it.  For 128 tokens at a time,
//   S = Q K^T    128 x 128 x dim   from shared memory into tensor memory
//   P = exp2(S c - m)              tensor memory -> registers -> tensor memory
//   O += P V     128 x dim x 128   P from tensor memory, V from shared memory
// and every part has its own warps, joined by barriers:
//   - four warps for each tile: a thread has a row, so the softmax needs no
//     exchange; P takes the place of S;
//   - one warp reads the page table and the pages' scales ahead and copies the
//     pages' codes into shared memory;
//   - four warps turn those into 16-bit floats, again in shared memory (rows of
//     128 bytes, swizzled, with what the product sums over side by side: a
//     value row's tokens are so in the cache already);
//   - one thread issues the products: with two tiles, one tile's run while the
//     other's softmax does.
// O is not divided or rescaled on the way unless a row's largest score, or its
// largest weight with the page's value scale, grows by more than 2^8 over what
// they are relative to (the weights are 16-bit floats, which have room for that).
//
// Three prompts of up to 2049 tokens behind up to 4096 cached ones, 32 heads of
// 128 over 8: 390 us, 773 TFLOP/s (46% of the measured bf16 peak).  A step of
// two tiles is 2,048 cycles of products and as many of exponentials (16 a
// cycle); both tiles' softmaxes run side by side, then wait for the products,
// since the tensor memory has no room for the next step's scores beside two
// tiles' scores and sums.  Taking turns instead: 451 us, as one tile's softmax
// alone does not fill the SM.  One tile a CTA reads and turns the codes twice as
// often and is taken where there are no rows for two.
#include "attend_internal.h"

namespace vdt {
namespace {

constexpr int kTile = 128;        // query rows of a tile
constexpr int kAhead = 4;         // steps that the page lists are ahead
template <int D, int NT, int P>
struct Shape {
    static constexpr int kStep = D <= 128 ? 128 : 64;              // tokens of a step
    static constexpr int kSub = (D + 63) / 64;                     // 64-wide blocks of a head
    static constexpr int kQ = kSub * kTile * 128, kK = kSub * kStep * 128, kV = kStep / 64 * D * 128;
    static constexpr int kPages = kStep / P;
    static constexpr int kRaw = kStep * D;                         // the codes of a step's keys, or values
    static constexpr int kSoft = 4 * NT, kCode = kSoft, kIssue = kSoft + 4, kList = kSoft + 5;   // first warps of each part
    // two tiles share out registers by groups of four warps: two have nothing to do
    static constexpr int kThreads = (NT == 2 ? kSoft + 8 : kSoft + 6) * 32;
    static constexpr int kTmem = NT * (kStep + D) <= 256 ? 256 : 512;
    static constexpr int kBytes = 1024 + NT * kQ + 2 * kK + 2 * kV + 2 * kRaw;
    // one tile of a small head leaves room for a second CTA on the SM; its
    // softmax then holds half of the scores at a time
    static constexpr int kPerSm = NT == 1 && D <= 64 ? 2 : 1, kHold = kPerSm == 2 ? 64 : kStep;
};
// registers a thread with two tiles: at launch, and how the four groups of
// warps share them out
constexpr int kRegs = 128, kSoftRegs = 200, kCodeRegs = 64, kIssueRegs = 48;
static_assert(2 * kSoftRegs + kCodeRegs + kIssueRegs == 4 * kRegs, "registers");

template <int N>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int NT, int PAGES>
struct State {
    uint64_t k_full[2], k_free[2], v_full[2], v_free[2], raw_full[2], raw_free[2], s_full[NT], p_full[NT], o_done[NT];
    uint64_t list_full[kAhead], list_free[kAhead];
    uint32_t tmem;
    float k_scale[kAhead][PAGES], v_log[kAhead][PAGES];    // of the values' scales, the logarithm
};

// d (128 x N, 32-bit) (+)= a b^T for 16 columns of 16-bit floats
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&r)[32]) {
    uint32_t a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        a[i] = r[i];
        b[i] = r[16 + i];
    }
    tmem_store16(at, a);
    tmem_store16(at + 16, b);
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// what this thread wrote to shared memory is there for the tensor cores
__device__ __forceinline__ void fence_shared_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 codes to two 16-byte pieces `chunk` and `chunk + 1` of a swizzled row;
// `flip` writes the second first (lanes that would meet on one bank)
__device__ __forceinline__ void store_codes(unsigned char* rows, int row, int chunk, const uint4& w, bool flip) {
    uint4 a, b;
    codes_to_f16(w.x, a.x, a.y);
    codes_to_f16(w.y, a.z, a.w);
    codes_to_f16(w.z, b.x, b.y);
    codes_to_f16(w.w, b.z, b.w);
    unsigned char* at = rows + row * 128;
    *reinterpret_cast<uint4*>(at + (((chunk + flip) ^ (row & 7)) << 4)) = flip ? b : a;
    *reinterpret_cast<uint4*>(at + (((chunk + !flip) ^ (row & 7)) << 4)) = flip ? a : b;
}

template <int D, int NT, int P>
__global__ void __launch_bounds__(Shape<D, NT, P>::kThreads, Shape<D, NT, P>::kPerSm) k_attend_tiles(AttendParams p, int chunk, int count) {
    using Sh = Shape<D, NT, P>;
    constexpr int kPages = Sh::kPages, kStep = Sh::kStep;
    extern __shared__ unsigned char smem_raw[];
    __shared__ State<NT, kPages> st;
    chain_release();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int b = blockIdx.z, h = blockIdx.y, group = p.heads / p.c.heads;
    // the longest rows first: they see the most tokens
    const int part = blockIdx.x % count, row0 = (gridDim.x / count - 1 - blockIdx.x / count) * (NT * kTile);
    const Queries s = queries_of(p, b);
    const int rows = s.rows * group;
    if (row0 >= rows) {
        if (rows == 0 && blockIdx.x == 0) spoil_run(p, b, h);          // nothing to do for an empty run
        return;
    }
    auto sees = [&](int r) {                       // tokens that row r of the sequence sees
        if (r >= rows || s.kept < 0) return 0;
        return p.causal ? max(0, s.kept - s.rows + r / group + 1) : s.kept;
    };
    const int begin = part * chunk;
    // steps that each tile takes, and the longer of them
    int steps[NT], most = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int last = min(row0 + (t + 1) * kTile, rows) - 1;
        const int end = row0 + t * kTile < rows ? min(begin + chunk, sees(last)) : 0;
        steps[t] = max(0, (end - begin + kStep - 1) / kStep);
        most = max(most, steps[t]);
    }
    if (count > 1 && begin >= max(1, sees(min(row0 + NT * kTile, rows) - 1))) return;     // the join knows as well

    unsigned char* smem = smem_raw + ((1024 - (shared_address(smem_raw) & 1023)) & 1023);
    unsigned char* const kt = smem + NT * Sh::kQ;
    unsigned char* const vt = kt + 2 * Sh::kK;
    unsigned char* const raw = vt + 2 * Sh::kV;    // keys' codes, then values'
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(shared_address(&st.k_full[i]), 4);
            bar_init(shared_address(&st.k_free[i]), 1);
            bar_init(shared_address(&st.v_full[i]), 4);
            bar_init(shared_address(&st.v_free[i]), 1);
            bar_init(shared_address(&st.raw_full[i]), 1);
            bar_init(shared_address(&st.raw_free[i]), 4);
        }
        for (int i = 0; i < NT; ++i) {
            bar_init(shared_address(&st.s_full[i]), 1);
            bar_init(shared_address(&st.p_full[i]), kTile);
            bar_init(shared_address(&st.o_done[i]), 1);
        }
        for (int i = 0; i < kAhead; ++i) {
            bar_init(shared_address(&st.list_full[i]), 1);
            bar_init(shared_address(&st.list_free[i]), 4 * NT);
        }
        bar_init_done();
    }
    if (warp == Sh::kIssue) tmem_alloc(shared_address(&st.tmem), Sh::kTmem);

    // a softmax thread's row: its queries into shared memory, scaled by a power of two
    float q_scale = 0.0f;
    long long token = 0;
    int head = 0, limit = 0;
    const int mine = row0 + threadIdx.x;           // softmax threads are the first NT * 128
    if (warp < Sh::kSoft) {
        limit = sees(mine);
        token = s.first + mine / group;
        head = h * group + mine % group;
        unsigned char* const to = smem + warp / 4 * Sh::kQ;
        const int r = threadIdx.x % kTile;
        const long long from = token * p.q_token + (long long)head * p.q_head;
        const bool in = mine < rows, wide = p.q_token % 8 == 0 && p.q_head % 8 == 0 && reinterpret_cast<uintptr_t>(p.q) % 16 == 0;
        // the row as it is: all its loads are in flight together
        uint4 raw_q[D / 8];
        const __half* const q = static_cast<const __half*>(p.q) + from;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) raw_q[i] = in && wide ? *reinterpret_cast<const uint4*>(q + i * 8) : make_uint4(0, 0, 0, 0);
        if (in && !wide) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                __half v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = q[i * 8 + j];
                memcpy(&raw_q[i], v, 16);
            }
        }
        auto eight = [&](int i, float (&f)[8]) {
            if (p.type == VDT_F16) {
                Vec16<__half> v{raw_q[i]};
                v.get(f);
            } else {
                Vec16<__nv_bfloat16> v{raw_q[i]};
                v.get(f);
            }
        };
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            float f[8];
            eight(i, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[j]));
        }
        const int e = m > 0.0f && m < inf_f() ? max(-126, min(126, ilogbf(m))) : 0;
        q_scale = scalbnf(fabsf(p.scale), e);
        const float f1 = copysignf(scalbnf(1.0f, -e), p.scale);        // a negative scale goes into the queries
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            float f[8];
            eight(i, f);
            uint4 w;
            w.x = pack_f16(f[0] * f1, f[1] * f1);
            w.y = pack_f16(f[2] * f1, f[3] * f1);
            w.z = pack_f16(f[4] * f1, f[5] * f1);
            w.w = pack_f16(f[6] * f1, f[7] * f1);
            *reinterpret_cast<uint4*>(to + i / 8 * (kTile * 128) + r * 128 + ((i % 8 ^ (r & 7)) << 4)) = w;
        }
        fence_shared_async();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = st.tmem, tmem_o = tmem + NT * kStep;
    bool alive = true;

    if (warp < Sh::kSoft) {
        // ------------------------------------------------------------ softmax
        if constexpr (NT == 2) take_registers<kSoftRegs>();
        const int t = warp / 4;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;             // this warp's rows of the tensor memory
        const uint32_t at_s = tmem + t * kStep + lanes, at_o = tmem_o + t * D + lanes;
        int my_steps = 0;
#pragma unroll
        for (int i = 0; i < NT; ++i) my_steps = i == t ? steps[i] : my_steps;
        float ref = -inf_f(), vref = -inf_f(), sum = 0.0f;
        const bool busy = __any_sync(0xffffffffu, mine < rows);
        for (int j = 0; j < most; ++j) {
            const int slot = j % kAhead;
            alive = bar_wait_all(shared_address(&st.list_full[slot]), j / kAhead & 1);
            if (!alive) break;
            if (j < my_steps) {
                const int left = limit - (begin + j * kStep);          // tokens of the step that the row sees
                const bool partial = __any_sync(0xffffffffu, left < kStep);
                alive = bar_wait_all(shared_address(&st.s_full[t]), j & 1);
                if (!alive) break;
                tmem_fence_after();
                if (!busy) {                                           // rows past the last: whatever stands there
                    tmem_fence_before();
                    bar_arrive(shared_address(&st.p_full[t]));
                    if (lane == 0) bar_arrive(shared_address(&st.list_free[slot]));
                    continue;
                }
                constexpr int kHold = Sh::kHold;
                uint32_t r[kHold / 32][32];
                auto load = [&](int from) {
#pragma unroll
                    for (int i = 0; i < kHold / 32; ++i) tmem_load(at_s + from + i * 32, r[i]);
                };
                float c[kPages], top = -inf_f(), v_top = -inf_f();
#pragma unroll
                for (int from = kStep - kHold; from >= 0; from -= kHold) {
                    load(from);
                    if (from == kStep - kHold)
#pragma unroll
                        for (int i = 0; i < kPages; ++i) c[i] = st.k_scale[slot][i] * q_scale;
                    tmem_load_wait();
                    if (partial)
#pragma unroll
                        for (int i = 0; i < kHold; ++i) r[i / 32][i % 32] = from + i < left ? r[i / 32][i % 32] : 0xff800000u;
#pragma unroll
                    for (int i = 0; i < kHold; i += P < 32 ? P : 32) {
                        constexpr int kRun = P < 32 ? P : 32;          // in four chains
                        float m[4];
#pragma unroll
                        for (int q = 0; q < kRun; ++q) {
                            const float x = __uint_as_float(r[i / 32][i % 32 + q]);
                            m[q % 4] = q < 4 ? x : fmaxf(m[q % 4], x);
                        }
                        const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * c[(from + i) / P];
                        top = fmaxf(top, most);
                        v_top = fmaxf(v_top, most + st.v_log[slot][(from + i) / P]);
                    }
                }
                const bool up = passes(top, ref) || passes(v_top, ref + vref);
                if (__any_sync(0xffffffffu, up)) {
                    Rescale by = {1.0f, 1.0f};
                    if (up) by = move_references(top, v_top, ref, vref);
                    sum *= by.sum;
                    if (j > 0) {
                        alive = bar_wait_all(shared_address(&st.o_done[t]), (j - 1) & 1);
                        if (!alive) break;
                        tmem_fence_after();
                        for (int i = 0; i < D; i += 16) {
                            uint32_t o[16];
                            tmem_load16(at_o + i, o);
                            tmem_load_wait();
#pragma unroll
                            for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * by.out);
                            tmem_store16(at_o + i, o);
                        }
                    }
                }
                // a weight times its page's scale over 2^vref is one power of
                // two; the sum of the weights takes the scale out again
                const float shift = ref == -inf_f() ? 0.0f : -ref;
#pragma unroll
                for (int from = 0; from < kStep; from += kHold) {
                    if (from) {
                        load(from);
                        tmem_load_wait();
                    }
#pragma unroll
                    for (int i = from / P; i < (from + kHold) / P; ++i) {
                        const float f = page_shift(st.v_log[slot][i], vref), d = shift + f;
                        const float2 by = make_float2(c[i], c[i]), add = make_float2(d, d);
                        float2 l[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                        for (int a = i * P; a < (i + 1) * P; a += 2) {
                            const int q = a - from;
                            float2 x = fma2(make_float2(__uint_as_float(r[q / 32][q % 32]), __uint_as_float(r[q / 32][q % 32 + 1])), by, add);
                            x = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                            if (partial) {                             // also for scales that are not numbers
                                x.x = a < left ? x.x : 0.0f;
                                x.y = a + 1 < left ? x.y : 0.0f;
                            }
                            l[a / 2 % 2] = add2(l[a / 2 % 2], x);
                            r[q / 64][q / 2 % 32] = pack_f16(x.x, x.y);
                        }
                        const float l0 = (l[0].x + l[1].x) + (l[0].y + l[1].y);
                        sum = partial && i * P >= left ? sum : fmaf(l0, exp2_fast(-f), sum);
                    }
#pragma unroll
                    for (int i = 0; i < kHold / 64; ++i) tmem_store32(at_s + from / 2 + i * 32, r[i]);
                }
                tmem_store_wait();
                tmem_fence_before();
                bar_arrive(shared_address(&st.p_full[t]));
            }
            __syncwarp();
            if (lane == 0) bar_arrive(shared_address(&st.list_free[slot]));
        }
        // ------------------------------------------------------------- output
        if (alive && my_steps) alive = bar_wait_all(shared_address(&st.o_done[t]), (my_steps - 1) & 1);
        tmem_fence_after();
        const bool bad = !alive || s.kept < 0;
        const float v_scale = exp2f(vref - kSlack);                     // 2^vref may be too large for 32 bits where its product is not
        const float scale = bad ? nan_f() : count > 1 ? v_scale : sum == 0.0f ? 0.0f : v_scale / sum;
        const bool nothing = !bad && sum == 0.0f;                       // no token seen (O may not have been written)
        const long long out = token * p.out_token + (long long)head * p.out_head;
        const Partial rest = partial_of(p, token * p.heads + head, count, part);
        const bool wide = p.out_token % 8 == 0 && p.out_head % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
        if (count > 1 && mine < rows) *rest.stats = make_float2(ref, bad ? nan_f() : sum);
#pragma unroll
        for (int i = 0; i < D; i += 32) {
            uint32_t r[32];
            __syncwarp();
            tmem_load(at_o + i, r);
            tmem_load_wait();
            if (mine >= rows) continue;
            if (count > 1) {
#pragma unroll
                for (int q = 0; q < 32; q += 4) {
                    float f[4];
#pragma unroll
                    for (int a = 0; a < 4; ++a) f[a] = nothing ? 0.0f : __uint_as_float(r[q + a]) * scale * kSlackFactor;
                    *reinterpret_cast<float4*>(rest.sums + i + q) = make_float4(f[0], f[1], f[2], f[3]);
                }
            } else if (wide) {
#pragma unroll
                for (int q = 0; q < 32; q += 8) {
                    float f[8];
#pragma unroll
                    for (int a = 0; a < 8; ++a) f[a] = nothing ? 0.0f : __uint_as_float(r[q + a]) * scale * kSlackFactor;
                    uint4* to = reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + out + i + q);
                    if (p.type == VDT_F16) {
                        Vec16<__half> v;
                        v.set(f);
                        *to = v.raw;
                    } else {
                        Vec16<__nv_bfloat16> v;
                        v.set(f);
                        *to = v.raw;
                    }
                }
            } else {
#pragma unroll
                for (int q = 0; q < 32; ++q) store_value(p.out, out + i + q, p.type, nothing ? 0.0f : __uint_as_float(r[q]) * scale * kSlackFactor);
            }
        }
    } else if (warp < Sh::kIssue) {
        // ------------------------------------------------- codes to 16 bits
        if constexpr (NT == 2) give_registers<kCodeRegs>();
        const int thread = threadIdx.x - Sh::kCode * 32;
        constexpr int kPer = kStep * D / 16 / 128;                     // 16-byte pieces of a thread, keys or values
        constexpr int kRow = D / 16, kBlock = P * D / 16;              // of a token's keys, of a page
        for (int j = 0; j < most; ++j) {
            const int slot = j & 1, phase = (j / 2 & 1) ^ 1;
            alive = bar_wait_all(shared_address(&st.raw_full[0]), j & 1) && bar_wait_all(shared_address(&st.k_free[slot]), phase);
            if (!alive) break;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int at = thread + i * 128, row = at / kRow, e = at % kRow;
                store_codes(kt + slot * Sh::kK + e / 4 * (kStep * 128), row, e % 4 * 2, *reinterpret_cast<const uint4*>(raw + at * 16), e & 4);
            }
            fence_shared_async();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(shared_address(&st.raw_free[0]));
                bar_arrive(shared_address(&st.k_full[slot]));
            }
            alive = bar_wait_all(shared_address(&st.raw_full[1]), j & 1) && bar_wait_all(shared_address(&st.v_free[slot]), phase);
            if (!alive) break;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int at = thread + i * 128, pg = at / kBlock, rest = at % kBlock, row = rest / (P / 16);
                const int block = pg * (P / 16) + rest % (P / 16);     // 16 tokens of the step
                store_codes(vt + slot * Sh::kV + block / 4 * (D * 128), row, block % 4 * 2,
                            *reinterpret_cast<const uint4*>(raw + Sh::kRaw + at * 16), false);
            }
            fence_shared_async();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(shared_address(&st.raw_free[1]));
                bar_arrive(shared_address(&st.v_full[slot]));
            }
        }
    } else if (warp == Sh::kIssue) {
        // ---------------------------------------------------------- products
        if constexpr (NT == 2) give_registers<kIssueRegs>();
        constexpr uint32_t shape = 1u << 4 | (kTile >> 4) << 24;       // 32-bit sums of 16-bit floats
        constexpr uint32_t shape_s = shape | (kStep >> 3) << 17, shape_o = shape | (D >> 3) << 17;
        const uint32_t at = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_at = tile_desc(shared_address(smem)), k_at = tile_desc(shared_address(kt)), v_at = tile_desc(shared_address(vt));
        const bool one = elected();
        auto scores = [&](int t, int slot) {
            if (one) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_shared(at + t * kStep, q_at + (t * Sh::kQ + k / 4 * (kTile * 128) + k % 4 * 32) / 16,
                               k_at + (slot * Sh::kK + k / 4 * (kStep * 128) + k % 4 * 32) / 16, shape_s, k > 0);
                mma_commit(shared_address(&st.s_full[t]));
            }
        };
        auto outputs = [&](int t, int slot, bool add) {
            if (one) {
#pragma unroll
                for (int k = 0; k < kStep / 16; ++k)
                    mma_tensor(at + NT * kStep + t * D, at + t * kStep + k * 8, v_at + (slot * Sh::kV + k / 4 * (D * 128) + k % 4 * 32) / 16,
                               shape_o, add || k > 0);
                mma_commit(shared_address(&st.o_done[t]));
            }
        };
        if (most && (alive = bar_wait_all(shared_address(&st.k_full[0]), 0))) {
            tmem_fence_after();
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (steps[t]) scores(t, 0);
            if (one) mma_commit(shared_address(&st.k_free[0]));
        }
        for (int j = 0; j < most && alive; ++j) {
            const int slot = j & 1, next = slot ^ 1;
            if (!(alive = bar_wait_all(shared_address(&st.v_full[slot]), j / 2 & 1))) break;
            if (j + 1 < most && !(alive = bar_wait_all(shared_address(&st.k_full[next]), (j + 1) / 2 & 1))) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (j >= steps[t] || !alive) continue;
                if (!(alive = bar_wait_all(shared_address(&st.p_full[t]), j & 1))) continue;
                tmem_fence_after();
                outputs(t, slot, j > 0);
                if (j + 1 < steps[t]) scores(t, next);                 // behind the product that reads P in S's place
            }
            if (one) {
                mma_commit(shared_address(&st.v_free[slot]));
                if (j + 1 < most) mma_commit(shared_address(&st.k_free[next]));
            }
        }
        // the last commit has arrived before the CTA ends
        if (most && alive) bar_wait_all(shared_address(&st.v_free[(most - 1) & 1]), (most - 1) / 2 & 1);
    } else if (warp == Sh::kList) {
        // ----------------------------------------------- page lists and codes
        if constexpr (NT == 2) give_registers<kIssueRegs>();
        const int end = min(begin + chunk, s.kept);
        const bool on = lane < kPages;
        // step j's page: -1 past the end, -2 if it is not in the cache
        auto page = [&](int j) {
            const int first = begin + j * kStep + lane * P;
            if (!on || first >= end) return -1;
            const int no = p.r.table[(long long)b * p.r.width + first / P];
            return no >= 0 && no < p.c.pages ? no : -2;
        };
        auto scale = [&](const float* of, int no) {                    // one that is not in the cache, or is infinite: not a number
            const float x = no >= 0 ? of[(long long)no * p.c.heads + h] : 0.0f;
            return no == -2 || x == inf_f() ? nan_f() : x;
        };
        constexpr uint32_t kBlock = P * D;
        auto copy = [&](int side, int j, int no) {
            const uint32_t bar = shared_address(&st.raw_full[side]);
            if (!bar_wait_all(shared_address(&st.raw_free[side]), (j & 1) ^ 1)) return false;
            const int n = __popc(__ballot_sync(0xffffffffu, no != -1));
            if (lane == 0) bar_expect(bar, n * kBlock);
            __syncwarp();
            if (no != -1)
                bulk_load(shared_address(raw + side * Sh::kRaw) + lane * kBlock,
                          (side ? p.c.v : p.c.k) + ((long long)max(no, 0) * p.c.heads + h) * kBlock, kBlock, bar);
            return true;
        };
        int no = most ? page(0) : -1, next = most > 1 ? page(1) : -1;
        float ks = scale(p.c.k_scale, no), vs = scale(p.c.v_scale, no);
        int j = 0;
        for (; j < most; ++j) {
            const int slot = j % kAhead;
            alive = bar_wait_all(shared_address(&st.list_free[slot]), (j / kAhead & 1) ^ 1);
            if (!alive) break;
            const float m = vs > 0.0f ? log2f(vs) : vs == 0.0f || no == -1 ? -inf_f() : nan_f();
            if (on) {
                st.k_scale[slot][lane] = ks;
                st.v_log[slot][lane] = m;
            }
            __syncwarp();
            if (lane == 0) bar_arrive(shared_address(&st.list_full[slot]));
            const int now = no;
            no = next;
            ks = scale(p.c.k_scale, no);
            vs = scale(p.c.v_scale, no);
            next = j + 2 < most ? page(j + 2) : -1;
            if (!(alive = copy(0, j, now) && copy(1, j, now))) break;
        }
        if (!alive)                                                    // what is in flight gets as long again to land
            for (int side = 0; side < 2; ++side)
                for (int ph = 0; ph < 2; ++ph) bar_wait(shared_address(&st.raw_full[side]), ph);
    } else if constexpr (NT == 2) {
        give_registers<kIssueRegs>();
    }
    // the products are done: every tile's last commit has been waited for
    tmem_fence_before();
    __syncthreads();
    if (warp == Sh::kIssue) {
        __syncwarp();
        tmem_fence_after();
        tmem_free(tmem, Sh::kTmem);
    }
}

template <int D, int NT, int P>
cudaError_t tiles_launch(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    using Sh = Shape<D, NT, P>;
    cudaError_t e = allow_shared<k_attend_tiles<D, NT, P>>(Sh::kBytes);
    if (e != cudaSuccess) return e;
    if constexpr (NT == 2) {
        // the groups share out exactly what the block is launched with; with
        // less they would wait for ever
        static std::atomic<int> regs{0};
        if (!regs.load(std::memory_order_relaxed)) {
            cudaFuncAttributes a{};
            e = cudaFuncGetAttributes(&a, k_attend_tiles<D, NT, P>);
            if (e != cudaSuccess) return e;
            regs.store(a.numRegs, std::memory_order_relaxed);
        }
        if (regs.load(std::memory_order_relaxed) < kRegs) return cudaErrorInvalidKernelImage;
    }
    const long long rows = (long long)p.r.most * (p.heads / p.c.heads), x = (rows + NT * kTile - 1) / (NT * kTile) * c.count;
    if (x > 0x7fffffff) return cudaErrorInvalidValue;
    k_attend_tiles<D, NT, P><<<dim3((unsigned)x, p.c.heads, p.r.seqs), Sh::kThreads, Sh::kBytes, s>>>(p, c.tokens, c.count);
    return cudaGetLastError();
}

template <int D, int NT>
cudaError_t by_page(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    switch (p.c.page) {
        case 16: return tiles_launch<D, NT, 16>(p, c, s);
        case 32: return tiles_launch<D, NT, 32>(p, c, s);
        default: return tiles_launch<D, NT, 64>(p, c, s);
    }
}

template <int NT>
cudaError_t by_dim(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    switch (p.c.dim) {
        case 32: return by_page<32, NT>(p, c, s);
        case 64: return by_page<64, NT>(p, c, s);
        case 96: return by_page<96, NT>(p, c, s);
        case 128: return by_page<128, NT>(p, c, s);
        case 192: return by_page<192, 1>(p, c, s);
        default: return by_page<256, 1>(p, c, s);
    }
}

}  // namespace

// Two tiles share the turned codes where there are the rows, and where the
// tensor memory holds both tiles' scores and sums: up to 128 values a head.
int tile_rows(int dim, long long rows) { return rows <= kTile || dim > 128 ? kTile : 2 * kTile; }

// The tokens divided where the tiles alone leave SMs idle, 512 of them at least
// to a CTA.  With 1024 and with 512, us: 33 queries over 2000 tokens, 8 heads of 64
// 25.4 and 16.8; 200 over 2000, 2 sequences, 8 heads of 128 35.2 and 25.9; 300 over
// 16000, 4 heads of 64 over one 31.1 and 27.4.  With 256 these take 12.9, 22.4 and
// 27.4; where the joining of more chunks outweighs it has not been looked for.
Chunks plan_tiles(int dim, int heads, int kv_heads, int seqs, int most, int most_kept) {
    const long long rows = (long long)most * (heads / kv_heads), each = tile_rows(dim, rows);
    const long long ctas = (long long)kv_heads * seqs * ((rows + each - 1) / each);
    const long long want = kSmCount / ctas;
    if (want <= 1) return {(most_kept + kTile - 1) / kTile * kTile, 1};
    long long tokens = ((long long)most_kept + want - 1) / want;
    tokens = (tokens + kTile - 1) / kTile * kTile;
    if (tokens < 4 * kTile) tokens = 4 * kTile;
    const long long count = ((long long)most_kept + tokens - 1) / tokens;
    return {(int)tokens, (int)(count < 1 ? 1 : count)};
}

cudaError_t launch_attend_tiles(const AttendParams& p, const Chunks& c, cudaStream_t s) {
    return tile_rows(p.c.dim, (long long)p.r.most * (p.heads / p.c.heads)) == kTile ? by_dim<1>(p, c, s) : by_dim<2>(p, c, s);
}

}  // namespace vdt

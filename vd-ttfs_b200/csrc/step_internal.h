// step_internal.h -- declarations shared by the kernels of a decoder's step
// around its products and attention (k_fp4.cu, k_norm.cu, k_plan.cu,
// k_sample.cu) and their entry points (step.cu); not part of the public ABI.
#pragma once

#include "seq_internal.h"

namespace vdt {

// ------------------------------------------- microscaled 4-bit floating point
constexpr int kBlock = 32;                 // values under one scale
constexpr int kScaleRows = 128;            // rows of a scale tile
constexpr int kScaleTile = 512;            // its bytes: 128 rows, 4 blocks
constexpr int kFp4Step = 256;              // columns that codes and scales are loaded by: 128 bytes of codes

inline long long fp4_steps(long long cols) { return (cols + kFp4Step - 1) / kFp4Step; }

cudaError_t launch_quantize_fp4(const void* x, int type, long long rows, int cols, long long x_stride, uint8_t* codes, long long codes_stride,
                                uint8_t* scale, cudaStream_t s);
cudaError_t launch_fp4_values(const uint8_t* codes, long long codes_stride, const uint8_t* scale, long long rows, int cols, int type, void* out,
                              long long out_stride, cudaStream_t s);

struct Fp4Params {
    const uint8_t* a;       // [rows, inner / 2] codes, rows a_stride bytes apart
    const uint8_t* a_scale;
    const uint8_t* w;       // [cols, inner / 2]
    const uint8_t* w_scale;
    const float* bias;      // [cols] or null
    void* out;
    long long rows, a_stride, w_stride, out_stride;
    int cols, inner, out_type;
    const void* x;          // rows that the product rounds itself, instead of a and a_scale
    long long x_stride;
};
// few rows, which the product's kernel rounds itself
bool fp4_rounds_itself(long long rows);
cudaError_t launch_fp4_own(const Fp4Params& p, int type, cudaStream_t s);
// after_codes: the kernel before it on the stream is the one that writes `a`
cudaError_t launch_fp4_matmul(const Fp4Params& p, bool after_codes, cudaStream_t s);

// ------------------------------------------------- residual's addition and norm
struct NormParams {
    const void *x, *residual, *weight;      // [rows, cols]; [rows, cols] or null; [cols] or null
    void *sum, *out;                        // the sum (null without a residual); values, or
    int8_t* codes;                          // codes and
    float* scale;                           // their scales
    long long rows, x_stride, residual_stride, sum_stride, out_stride;
    int cols, type;
    float eps;
};
cudaError_t launch_add_rms_norm(const NormParams& p, cudaStream_t s);

// ------------------------------------------------------------------ page tables
struct PlanParams {
    const int32_t *ring, *span;             // free pages; the first one's place and their number
    int32_t* pages;                         // [seqs, width]
    const int32_t *held, *fresh;
    int32_t *kept, *starts, *positions, *span_out;
    int64_t* slots;
    int32_t* scratch;
    long long total;
    int size, width, seqs, page, shift;     // shift: set by the launch, log2(page) or -1
    bool wide;                              // so is this: positions and slots on 16 bytes
};
size_t plan_scratch_bytes(int seqs);
cudaError_t launch_plan_pages(const PlanParams& p, cudaStream_t s);

struct FreeParams {
    int32_t* ring;
    const int32_t *span, *pages, *held;
    const uint8_t* done;
    int32_t *held_out, *span_out;
    int size, width, seqs, page, shift;
};
cudaError_t launch_free_pages(const FreeParams& p, cudaStream_t s);

// --------------------------------------------------------------------- sampling
constexpr int kMostVocab = 1 << 19;
struct SampleParams {
    const void* logits;
    const float *u, *temperatures, *top_ps, *min_ps;     // [rows]; the last three may be null
    const int32_t* top_ks;
    int32_t* tokens;
    float* logp;                                         // or null
    long long rows, stride;
    int vocab, type, top_k;
    float temperature, top_p, min_p;
};
cudaError_t launch_sample(const SampleParams& p, cudaStream_t s);

}  // namespace vdt

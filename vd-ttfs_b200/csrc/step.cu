// step.cu -- entry points of a decoder's step around its products and attention
// (include/vdttfs.h): checks of the arguments, then one or two launches on
// the caller's stream.
#include <cmath>

#include "step_internal.h"

using namespace vdt;

namespace {

constexpr int kMostSeqs = 65535;
constexpr long long kMostRows = 1 << 30;
constexpr int kMostCols = 1 << 30;         // kernels step past the last by up to a few thousand, in 32 bits
constexpr int kMostPages = 1 << 30;        // likewise, by a warp's

#define STEP_REQUIRE(cond, text) \
    do {                         \
        if (!(cond)) return api_fail(VDT_ERR_INVALID, text); \
    } while (0)

int launched(cudaError_t e, const char* what) { return e == cudaSuccess ? VDT_OK : api_cuda_fail(e, what); }

bool overlap(const void* a, long long a_bytes, const void* b, long long b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
long long code_bytes(long long cols) { return (cols + 1) / 2; }
long long code_stride(long long cols) { return (code_bytes(cols) + 15) / 16 * 16; }
size_t scale_bytes(long long rows, long long cols) { return (size_t)((rows + kScaleRows - 1) / kScaleRows) * fp4_steps(cols) * 2 * kScaleTile; }

int check_codes(const void* codes, int64_t stride, const void* scale, int64_t rows, int cols) {
    STEP_REQUIRE(rows >= 0 && rows < kMostRows && cols > 0, "rows and columns must be positive, rows below 2^30");
    if (cols > kMostCols) return api_fail(VDT_ERR_UNSUPPORTED, "more than 2^30 columns");
    STEP_REQUIRE(!rows || (codes && scale), "NULL buffer");
    STEP_REQUIRE(stride >= code_bytes(cols) && stride % 16 == 0 && aligned(codes, 16), "code rows must start on 16-byte boundaries");
    STEP_REQUIRE(aligned(scale, 16), "scales must start on a 16-byte boundary");
    return VDT_OK;
}
int check_product(const uint8_t* d_w, int64_t w_stride, const uint8_t* d_w_scale, const float* d_bias, int64_t rows, int cols, int inner,
                  int out_type, const void* d_out, int64_t out_stride) {
    STEP_REQUIRE(rows >= 0 && rows < kMostRows && cols > 0 && inner > 0, "rows, cols and inner must be positive, rows below 2^30");
    if (cols >= kMostRows) return api_fail(VDT_ERR_UNSUPPORTED, "2^30 cols and more");
    if (int s = check_codes(d_w, w_stride, d_w_scale, cols, inner)) return s;
    STEP_REQUIRE(type_ok(out_type), "output type");
    STEP_REQUIRE(d_out || !rows, "NULL buffer");
    STEP_REQUIRE(out_stride >= cols || rows <= 1, "out_stride below cols");
    STEP_REQUIRE(aligned(d_out, type_size(out_type)) && aligned(d_bias, 4), "alignment of the output or the bias");
    return VDT_OK;
}

// in place: the same rows, not others that begin there
bool same_rows(const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t rows) {
    return a != b || !a || rows <= 1 || a_stride == b_stride;
}
int check_norm(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_weight, int64_t rows, int cols,
               float eps, int type, const void* d_sum, int64_t sum_stride) {
    STEP_REQUIRE(type_ok(type), "type");
    STEP_REQUIRE(rows >= 0 && rows < kMostRows && cols > 0, "rows and cols must be positive, rows below 2^30");
    if (cols > kMostCols) return api_fail(VDT_ERR_UNSUPPORTED, "more than 2^30 cols");
    STEP_REQUIRE(eps >= 0.0f && std::isfinite(eps), "eps must not be negative");
    if (!rows) return VDT_OK;
    STEP_REQUIRE(d_x && (!d_residual || d_sum), "NULL buffer");
    STEP_REQUIRE(rows == 1 || (x_stride >= cols && (!d_residual || (residual_stride >= cols && sum_stride >= cols))), "a stride below cols");
    STEP_REQUIRE(!d_residual || (same_rows(d_sum, sum_stride, d_x, x_stride, rows) && same_rows(d_sum, sum_stride, d_residual, residual_stride, rows)),
                 "a sum in place has the strides of what it replaces");
    const int e = type_size(type);
    STEP_REQUIRE(aligned(d_x, e) && aligned(d_residual, e) && aligned(d_weight, e) && aligned(d_sum, e), "alignment");
    return VDT_OK;
}
NormParams norm_params(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_weight, int64_t rows,
                       int cols, float eps, int type, void* d_sum, int64_t sum_stride, int64_t out_stride) {
    NormParams p{};
    p.x = d_x; p.residual = d_residual; p.weight = d_weight;
    p.sum = d_residual ? d_sum : nullptr;
    p.rows = rows; p.x_stride = x_stride; p.residual_stride = residual_stride; p.sum_stride = sum_stride; p.out_stride = out_stride;
    p.cols = cols; p.type = type; p.eps = eps;
    return p;
}

// a page number times the page, and a token's place in a table of `width` pages, fit what the kernels count in
int check_tables(const void* d_ring, int ring, const void* d_span, const void* d_pages, int width, const void* d_held, int seqs, int page) {
    STEP_REQUIRE(seqs >= 0 && width >= 0 && ring >= 0 && page > 0, "negative size");
    if (seqs > kMostSeqs) return api_fail(VDT_ERR_UNSUPPORTED, "more than 65535 sequences");
    if (width > kMostPages || ring > kMostPages) return api_fail(VDT_ERR_UNSUPPORTED, "more than 2^30 pages in the ring or a table's row");
    STEP_REQUIRE(d_span && (d_ring || !ring) && (!seqs || (d_held && (d_pages || !width))), "NULL buffer");
    STEP_REQUIRE(aligned(d_ring, 4) && aligned(d_span, 4) && aligned(d_pages, 4) && aligned(d_held, 4), "alignment");
    return VDT_OK;
}

}  // namespace

extern "C" size_t vdt_fp4_scale_bytes(int64_t rows, int cols) { return rows <= 0 || cols <= 0 ? 0 : scale_bytes(rows, cols); }

extern "C" int vdt_quantize_fp4(const void* d_x, int type, int64_t rows, int cols, int64_t x_stride, uint8_t* d_codes, int64_t codes_stride,
                                uint8_t* d_scale, vdt_stream stream) {
    api_clear_error();
    STEP_REQUIRE(type_ok(type), "type");
    if (int s = check_codes(d_codes, codes_stride, d_scale, rows, cols)) return s;
    if (rows == 0) return VDT_OK;
    STEP_REQUIRE(d_x && (x_stride >= cols || rows == 1), "NULL buffer, or x_stride below cols");
    STEP_REQUIRE(aligned(d_x, type_size(type)), "alignment");
    if (int s = api_check_buffers(-1, {d_x, d_codes, d_scale})) return s;
    return launched(launch_quantize_fp4(d_x, type, rows, cols, x_stride, d_codes, codes_stride, d_scale, static_cast<cudaStream_t>(stream)),
                    "quantize_fp4");
}

extern "C" int vdt_fp4_values(const uint8_t* d_codes, int64_t codes_stride, const uint8_t* d_scale, int64_t rows, int cols, int type, void* d_out,
                              int64_t out_stride, vdt_stream stream) {
    api_clear_error();
    STEP_REQUIRE(type_ok(type), "type");
    if (int s = check_codes(d_codes, codes_stride, d_scale, rows, cols)) return s;
    if (rows == 0) return VDT_OK;
    STEP_REQUIRE(d_out && (out_stride >= cols || rows == 1), "NULL buffer, or out_stride below cols");
    STEP_REQUIRE(aligned(d_out, type_size(type)), "alignment");
    if (int s = api_check_buffers(-1, {d_codes, d_scale, d_out})) return s;
    return launched(launch_fp4_values(d_codes, codes_stride, d_scale, rows, cols, type, d_out, out_stride, static_cast<cudaStream_t>(stream)),
                    "fp4_values");
}

extern "C" int vdt_fp4_matmul(const uint8_t* d_a, int64_t a_stride, const uint8_t* d_a_scale, const uint8_t* d_w, int64_t w_stride,
                              const uint8_t* d_w_scale, const float* d_bias, int64_t rows, int cols, int inner, int out_type, void* d_out,
                              int64_t out_stride, vdt_stream stream) {
    api_clear_error();
    if (int s = check_product(d_w, w_stride, d_w_scale, d_bias, rows, cols, inner, out_type, d_out, out_stride)) return s;
    if (int s = check_codes(d_a, a_stride, d_a_scale, rows, inner)) return s;
    if (rows == 0) return VDT_OK;
    if (int s = api_check_buffers(-1, {d_a, d_a_scale, d_w, d_w_scale, d_bias, d_out})) return s;
    Fp4Params p{d_a, d_a_scale, d_w, d_w_scale, d_bias, d_out, rows, a_stride, w_stride, out_stride, cols, inner, out_type, nullptr, 0};
    return launched(launch_fp4_matmul(p, false, static_cast<cudaStream_t>(stream)), "fp4_matmul");
}

extern "C" size_t vdt_fp4_linear_scratch_bytes(int64_t rows, int inner) {
    if (rows <= 0 || inner <= 0) return 0;
    return round256((size_t)rows * (size_t)code_stride(inner)) + scale_bytes(rows, inner);
}

extern "C" int vdt_fp4_linear(const void* d_x, int type, int64_t x_stride, const uint8_t* d_w, int64_t w_stride, const uint8_t* d_w_scale,
                              const float* d_bias, int64_t rows, int cols, int inner, int out_type, void* d_out, int64_t out_stride,
                              void* d_scratch, size_t scratch_bytes, vdt_stream stream) {
    api_clear_error();
    STEP_REQUIRE(type_ok(type), "type");
    if (int s = check_product(d_w, w_stride, d_w_scale, d_bias, rows, cols, inner, out_type, d_out, out_stride)) return s;
    if (rows == 0) return VDT_OK;
    STEP_REQUIRE(d_x && d_scratch, "NULL buffer");
    STEP_REQUIRE(x_stride >= inner || rows == 1, "x_stride below inner");
    STEP_REQUIRE(aligned(d_x, type_size(type)) && aligned(d_scratch, 256), "alignment (256 bytes for the scratch)");
    if (scratch_bytes < vdt_fp4_linear_scratch_bytes(rows, inner))
        return api_fail(VDT_ERR_CAPACITY, "scratch smaller than vdt_fp4_linear_scratch_bytes");
    if (int s = api_check_buffers(-1, {d_x, d_w, d_w_scale, d_bias, d_out, d_scratch})) return s;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // every CTA reads all of a few rows, so not into an output that lies over them
    const bool over = overlap(d_x, ((rows - 1) * x_stride + inner) * type_size(type), d_out, ((rows - 1) * out_stride + cols) * type_size(out_type));
    if (fp4_rounds_itself(rows) && !over) {
        Fp4Params p{nullptr, nullptr, d_w, d_w_scale, d_bias, d_out, rows, 0, w_stride, out_stride, cols, inner, out_type, d_x, x_stride};
        return launched(launch_fp4_own(p, type, st), "fp4_linear");
    }
    uint8_t* codes = static_cast<uint8_t*>(d_scratch);
    uint8_t* scale = codes + round256((size_t)rows * (size_t)code_stride(inner));
    const cudaError_t e = launch_quantize_fp4(d_x, type, rows, inner, x_stride, codes, code_stride(inner), scale, st);
    if (e != cudaSuccess) return api_cuda_fail(e, "quantize_fp4");
    Fp4Params p{codes, scale, d_w, d_w_scale, d_bias, d_out, rows, code_stride(inner), w_stride, out_stride, cols, inner, out_type, nullptr, 0};
    return launched(launch_fp4_matmul(p, true, st), "fp4_matmul");
}

extern "C" int vdt_add_rms_norm(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_weight,
                                int64_t rows, int cols, float eps, int type, void* d_sum, int64_t sum_stride, void* d_out, int64_t out_stride,
                                vdt_stream stream) {
    api_clear_error();
    if (int s = check_norm(d_x, x_stride, d_residual, residual_stride, d_weight, rows, cols, eps, type, d_sum, sum_stride)) return s;
    if (!rows) return VDT_OK;
    STEP_REQUIRE(d_out && (out_stride >= cols || rows == 1) && aligned(d_out, type_size(type)), "output");
    STEP_REQUIRE(!d_residual || d_out != d_sum, "the output over the sum");
    STEP_REQUIRE(same_rows(d_out, out_stride, d_x, x_stride, rows) && same_rows(d_out, out_stride, d_residual, residual_stride, rows),
                 "an output in place has the strides of what it replaces");
    if (int s = api_check_buffers(-1, {d_x, d_residual, d_weight, d_sum, d_out})) return s;
    NormParams p = norm_params(d_x, x_stride, d_residual, residual_stride, d_weight, rows, cols, eps, type, d_sum, sum_stride, out_stride);
    p.out = d_out;
    return launched(launch_add_rms_norm(p, static_cast<cudaStream_t>(stream)), "add_rms_norm");
}

extern "C" int vdt_add_rms_norm_int8(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_weight,
                                     int64_t rows, int cols, float eps, int type, void* d_sum, int64_t sum_stride, int8_t* d_codes,
                                     int64_t codes_stride, float* d_scale, vdt_stream stream) {
    api_clear_error();
    if (int s = check_norm(d_x, x_stride, d_residual, residual_stride, d_weight, rows, cols, eps, type, d_sum, sum_stride)) return s;
    if (!rows) return VDT_OK;
    STEP_REQUIRE(d_codes && d_scale && (codes_stride >= cols || rows == 1) && aligned(d_scale, 4), "codes or scales");
    if (int s = api_check_buffers(-1, {d_x, d_residual, d_weight, d_sum, d_codes, d_scale})) return s;
    NormParams p = norm_params(d_x, x_stride, d_residual, residual_stride, d_weight, rows, cols, eps, type, d_sum, sum_stride, codes_stride);
    p.codes = d_codes;
    p.scale = d_scale;
    return launched(launch_add_rms_norm(p, static_cast<cudaStream_t>(stream)), "add_rms_norm_int8");
}

extern "C" size_t vdt_plan_pages_scratch_bytes(int seqs) { return seqs < 0 ? 0 : round256(plan_scratch_bytes(seqs)); }

extern "C" int vdt_plan_pages(const int32_t* d_ring, int ring, const int32_t* d_span, int32_t* d_pages, int width, const int32_t* d_held,
                              const int32_t* d_new, int seqs, int page, int64_t total, int32_t* d_kept, int32_t* d_starts, int32_t* d_positions,
                              int64_t* d_slots, int32_t* d_span_out, void* d_scratch, size_t scratch_bytes, vdt_stream stream) {
    api_clear_error();
    if (int s = check_tables(d_ring, ring, d_span, d_pages, width, d_held, seqs, page)) return s;
    STEP_REQUIRE(total >= 0 && total < kMostRows, "total must be below 2^30");
    STEP_REQUIRE(d_starts && d_span_out && d_scratch && (!seqs || (d_new && d_kept)) && (!total || (d_positions && d_slots)), "NULL buffer");
    STEP_REQUIRE(aligned(d_new, 4) && aligned(d_kept, 4) && aligned(d_starts, 4) && aligned(d_positions, 4) && aligned(d_slots, 8) &&
                     aligned(d_span_out, 4) && aligned(d_scratch, 16), "alignment");
    if (scratch_bytes < vdt_plan_pages_scratch_bytes(seqs))
        return api_fail(VDT_ERR_CAPACITY, "scratch smaller than vdt_plan_pages_scratch_bytes");
    if (int s = api_check_buffers(-1, {d_ring, d_span, d_pages, d_held, d_new, d_kept, d_starts, d_positions, d_slots, d_span_out, d_scratch})) return s;
    PlanParams p{d_ring, d_span, d_pages, d_held, d_new, d_kept, d_starts, d_positions, d_span_out, d_slots, static_cast<int32_t*>(d_scratch),
                 total, ring, width, seqs, page, 0, false};
    return launched(launch_plan_pages(p, static_cast<cudaStream_t>(stream)), "plan_pages");
}

extern "C" int vdt_free_pages(int32_t* d_ring, int ring, const int32_t* d_span, const int32_t* d_pages, int width, const int32_t* d_held,
                              const uint8_t* d_done, int seqs, int page, int32_t* d_held_out, int32_t* d_span_out, vdt_stream stream) {
    api_clear_error();
    if (int s = check_tables(d_ring, ring, d_span, d_pages, width, d_held, seqs, page)) return s;
    STEP_REQUIRE(d_span_out && (!seqs || (d_done && d_held_out)), "NULL buffer");
    STEP_REQUIRE(aligned(d_held_out, 4) && aligned(d_span_out, 4), "alignment");
    if (int s = api_check_buffers(-1, {d_ring, d_span, d_pages, d_held, d_done, d_held_out, d_span_out})) return s;
    FreeParams p{d_ring, d_span, d_pages, d_held, d_done, d_held_out, d_span_out, ring, width, seqs, page, 0};
    return launched(launch_free_pages(p, static_cast<cudaStream_t>(stream)), "free_pages");
}

extern "C" int vdt_sample(const void* d_logits, int type, int64_t rows, int vocab, int64_t stride, const float* d_u, const float* d_temperature,
                          float temperature, const int32_t* d_top_k, int top_k, const float* d_top_p, float top_p, const float* d_min_p,
                          float min_p, int32_t* d_tokens, float* d_logp, vdt_stream stream) {
    api_clear_error();
    STEP_REQUIRE(type_ok(type), "type");
    STEP_REQUIRE(rows >= 0 && rows < kMostRows / 8 && vocab > 0, "rows and vocab must be positive, rows below 2^27");
    if (vocab > kMostVocab) return api_fail(VDT_ERR_UNSUPPORTED, "more than 524288 tokens");
    STEP_REQUIRE(d_temperature || (temperature >= 0.0f && std::isfinite(temperature)), "temperature must not be negative");
    STEP_REQUIRE((d_top_p || !std::isnan(top_p)) && (d_min_p || !std::isnan(min_p)), "top_p or min_p");
    if (!rows) return VDT_OK;
    STEP_REQUIRE(d_logits && d_u && d_tokens, "NULL buffer");
    STEP_REQUIRE(stride >= vocab || rows == 1, "stride below vocab");
    STEP_REQUIRE(aligned(d_logits, type_size(type)) && aligned(d_u, 4) && aligned(d_temperature, 4) && aligned(d_top_k, 4) && aligned(d_top_p, 4) &&
                     aligned(d_min_p, 4) && aligned(d_tokens, 4) && aligned(d_logp, 4), "alignment");
    if (int s = api_check_buffers(-1, {d_logits, d_u, d_temperature, d_top_k, d_top_p, d_min_p, d_tokens, d_logp})) return s;
    SampleParams p{};
    p.logits = d_logits; p.u = d_u; p.temperatures = d_temperature; p.top_ps = d_top_p; p.min_ps = d_min_p; p.top_ks = d_top_k;
    p.tokens = d_tokens; p.logp = d_logp; p.rows = rows; p.stride = stride; p.vocab = vocab; p.type = type; p.top_k = top_k;
    p.temperature = temperature; p.top_p = top_p; p.min_p = min_p;
    return launched(launch_sample(p, static_cast<cudaStream_t>(stream)), "sample");
}

// seq.cu -- entry points of the sequence operators (include/vdttfs.h): checks
// of the arguments, then one or two launches on the caller's stream.
#include <cmath>

#include "seq_internal.h"

using namespace vdt;

namespace {

constexpr int kMostHeads = 1024;
constexpr int kMostSeqs = 65535;           // grid.z
constexpr int kMostTokens = 1 << 30;       // of one sequence
constexpr int kMostCols = 1 << 30;         // kernels step past the last by up to a few thousand, in 32 bits

#define SEQ_REQUIRE(cond, text) \
    do {                        \
        if (!(cond)) return api_fail(VDT_ERR_INVALID, text); \
    } while (0)

int launched(cudaError_t e, const char* what) { return e == cudaSuccess ? VDT_OK : api_cuda_fail(e, what); }

int check_product(const int8_t* d_w, int64_t w_stride, const float* d_w_scale, const float* d_bias, int64_t rows, int cols, int inner,
                  int out_type, const void* d_out, int64_t out_stride) {
    SEQ_REQUIRE(rows >= 0 && rows < kMostTokens && cols > 0 && inner > 0, "rows, cols and inner must be positive, rows below 2^30");
    if (cols > kMostCols) return api_fail(VDT_ERR_UNSUPPORTED, "more than 2^30 cols");
    if (inner > 131072) return api_fail(VDT_ERR_UNSUPPORTED, "inner above 131072: the sums would not fit 32-bit integers");
    SEQ_REQUIRE(type_ok(out_type), "output type");
    SEQ_REQUIRE(d_w && d_w_scale && (d_out || !rows), "NULL buffer");
    SEQ_REQUIRE(w_stride >= inner && w_stride % 16 == 0 && aligned(d_w, 16), "weight rows must start on 16-byte boundaries");
    SEQ_REQUIRE(out_stride >= cols, "out_stride below cols");
    SEQ_REQUIRE(aligned(d_out, type_size(out_type)), "out alignment");
    SEQ_REQUIRE(aligned(d_w_scale, 4) && aligned(d_bias, 4), "scale or bias alignment");
    return VDT_OK;
}

// whether two buffers of rows share any byte
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}
int64_t code_stride(int inner) { return ((int64_t)inner + 15) / 16 * 16; }
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

int check_cache(const vdt_cache8* c) {
    SEQ_REQUIRE(c, "cache is NULL");
    SEQ_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "NULL cache buffer");
    SEQ_REQUIRE(c->pages > 0 && c->heads > 0 && c->heads <= kMostHeads, "cache pages or heads");
    SEQ_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "cache codes must start on a 16-byte boundary");
    SEQ_REQUIRE(aligned(c->k_scale, 4) && aligned(c->v_scale, 4), "cache scale alignment");
    if (c->page != 16 && c->page != 32 && c->page != 64) return api_fail(VDT_ERR_UNSUPPORTED, "pages of 16, 32 or 64 tokens");
    if (!attend_dim_ok(c->dim)) return api_fail(VDT_ERR_UNSUPPORTED, "head dimensions 32, 64, 96, 128, 192 and 256");
    return VDT_OK;
}

int check_rows(const int32_t* table, int width, const int32_t* held, const int32_t* starts, int seqs, int64_t total, int most) {
    SEQ_REQUIRE(seqs >= 0 && width >= 0 && total >= 0 && most >= 0, "negative size");
    SEQ_REQUIRE(total < kMostTokens && most <= total, "total below 2^30, and no run longer than it");
    if (seqs > kMostSeqs) return api_fail(VDT_ERR_UNSUPPORTED, "more than 65535 sequences");
    SEQ_REQUIRE(!seqs || (held && starts && (table || !width)), "NULL buffer");
    SEQ_REQUIRE(aligned(table, 4) && aligned(held, 4) && aligned(starts, 4), "alignment of the table or the lengths");
    return VDT_OK;
}

CacheRows cache_rows(const int32_t* table, int width, const int32_t* held, const int32_t* starts, int seqs, int64_t total, int most) {
    CacheRows r{};
    r.table = table;
    r.held = held;
    r.starts = starts;
    r.seqs = seqs;
    r.width = width;
    r.total = total;
    r.most = most;
    return r;
}

}  // namespace

extern "C" int vdt_quantize_rows(const void* d_x, int type, int64_t rows, int cols, int64_t x_stride, int8_t* d_codes,
                                 int64_t codes_stride, float* d_scale, vdt_stream stream) {
    api_clear_error();
    SEQ_REQUIRE(type_ok(type), "type");
    SEQ_REQUIRE(rows >= 0 && rows < kMostTokens && cols > 0, "rows and cols must be positive, rows below 2^30");
    if (cols > kMostCols) return api_fail(VDT_ERR_UNSUPPORTED, "more than 2^30 cols");
    if (rows == 0) return VDT_OK;
    SEQ_REQUIRE(d_x && d_codes && d_scale, "NULL buffer");
    SEQ_REQUIRE((x_stride >= cols || rows == 1) && codes_stride >= cols, "a stride below cols");
    SEQ_REQUIRE(aligned(d_x, type_size(type)) && aligned(d_scale, 4), "alignment");
    if (int s = api_check_buffers(-1, {d_x, d_codes, d_scale})) return s;
    return launched(launch_quantize_rows(d_x, type, rows, cols, x_stride, d_codes, codes_stride, d_scale,
                                         static_cast<cudaStream_t>(stream)), "quantize_rows");
}

extern "C" int vdt_int8_matmul(const int8_t* d_a, int64_t a_stride, const float* d_a_scale, const int8_t* d_w,
                               int64_t w_stride, const float* d_w_scale, const float* d_bias, int64_t rows, int cols,
                               int inner, int out_type, void* d_out, int64_t out_stride, vdt_stream stream) {
    api_clear_error();
    if (int s = check_product(d_w, w_stride, d_w_scale, d_bias, rows, cols, inner, out_type, d_out, out_stride)) return s;
    if (rows == 0) return VDT_OK;
    SEQ_REQUIRE(d_a && d_a_scale, "NULL buffer");
    SEQ_REQUIRE(aligned(d_a_scale, 4), "scale alignment");
    SEQ_REQUIRE(a_stride >= inner && a_stride % 16 == 0 && aligned(d_a, 16), "code rows must start on 16-byte boundaries");
    if (int s = api_check_buffers(-1, {d_a, d_a_scale, d_w, d_w_scale, d_bias, d_out})) return s;
    Int8Params p{d_a, d_a_scale, d_w, d_w_scale, d_bias, d_out, rows, a_stride, w_stride, out_stride, cols, inner, out_type, nullptr, 0};
    return launched(launch_int8_matmul(p, false, static_cast<cudaStream_t>(stream)), "int8_matmul");
}

extern "C" size_t vdt_int8_linear_scratch_bytes(int64_t rows, int inner) {
    if (rows <= 0 || inner <= 0) return 0;
    return round256((size_t)rows * (size_t)code_stride(inner)) + round256((size_t)rows * sizeof(float));
}

extern "C" int vdt_int8_linear(const void* d_x, int type, int64_t x_stride, const int8_t* d_w, int64_t w_stride,
                               const float* d_w_scale, const float* d_bias, int64_t rows, int cols, int inner,
                               int out_type, void* d_out, int64_t out_stride, void* d_scratch, size_t scratch_bytes,
                               vdt_stream stream) {
    api_clear_error();
    SEQ_REQUIRE(type_ok(type), "type");
    if (int s = check_product(d_w, w_stride, d_w_scale, d_bias, rows, cols, inner, out_type, d_out, out_stride)) return s;
    if (rows == 0) return VDT_OK;
    SEQ_REQUIRE(d_x && d_scratch, "NULL buffer");
    SEQ_REQUIRE(x_stride >= inner || rows == 1, "x_stride below inner");
    SEQ_REQUIRE(aligned(d_x, type_size(type)) && aligned(d_scratch, 256), "alignment (256 bytes for the scratch)");
    if (scratch_bytes < vdt_int8_linear_scratch_bytes(rows, inner))
        return api_fail(VDT_ERR_CAPACITY, "scratch smaller than vdt_int8_linear_scratch_bytes");
    if (int s = api_check_buffers(-1, {d_x, d_w, d_w_scale, d_bias, d_out, d_scratch})) return s;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // one or two rows: the scratch is not used; every CTA reads all of them, so not
    // into an output that lies over them
    const bool over = overlap(d_x, ((rows - 1) * x_stride + inner) * type_size(type), d_out,
                              ((rows - 1) * out_stride + cols) * type_size(out_type));
    if (int8_rounds_itself(rows, inner) && !over) {
        Int8Params p{nullptr, nullptr, d_w, d_w_scale, d_bias, d_out, rows, 0, w_stride, out_stride, cols, inner, out_type, d_x, x_stride};
        return launched(launch_int8_own(p, type, st), "int8_linear");
    }
    int8_t* codes = static_cast<int8_t*>(d_scratch);
    float* scale = reinterpret_cast<float*>(codes + round256((size_t)rows * (size_t)code_stride(inner)));
    cudaError_t e = launch_quantize_rows(d_x, type, rows, inner, x_stride, codes, code_stride(inner), scale, st);
    if (e != cudaSuccess) return api_cuda_fail(e, "quantize_rows");
    Int8Params p{codes, scale, d_w, d_w_scale, d_bias, d_out, rows, code_stride(inner), w_stride, out_stride, cols, inner, out_type, nullptr, 0};
    return launched(launch_int8_matmul(p, true, st), "int8_matmul");
}

extern "C" int vdt_qk_norm_rope(const void* d_q, int64_t q_token, int64_t q_head, const void* d_k, int64_t k_token,
                                int64_t k_head, const void* d_q_weight, const void* d_k_weight,
                                const int32_t* d_positions, const float* d_table, int positions, int rot, int layout,
                                int norm, float eps, int64_t tokens, int heads, int kv_heads, int dim, int type,
                                void* d_q_out, int64_t qo_token, int64_t qo_head, void* d_k_out, int64_t ko_token,
                                int64_t ko_head, vdt_stream stream) {
    api_clear_error();
    SEQ_REQUIRE(type_ok(type), "type");
    SEQ_REQUIRE(tokens >= 0 && tokens < kMostTokens && heads >= 0 && kv_heads >= 0 && heads <= kMostHeads && kv_heads <= kMostHeads,
                "tokens or heads");
    SEQ_REQUIRE(dim > 0 && dim <= 8192, "dim must be in 1..8192");
    SEQ_REQUIRE(rot >= 0 && rot <= dim && rot % 2 == 0, "rot must be even and at most dim");
    SEQ_REQUIRE(layout == VDT_ROPE_HALF || layout == VDT_ROPE_PAIRS, "layout");
    SEQ_REQUIRE(norm >= VDT_NORM_NONE && norm <= VDT_NORM_L2, "norm");
    SEQ_REQUIRE(eps >= 0.0f, "eps must not be negative");
    if (tokens == 0 || heads + kv_heads == 0) return VDT_OK;
    SEQ_REQUIRE((!heads || (d_q && d_q_out)) && (!kv_heads || (d_k && d_k_out)), "NULL buffer");
    SEQ_REQUIRE(!rot || (d_positions && d_table && positions > 0), "a rotation needs positions and a table");
    const int e = type_size(type);
    SEQ_REQUIRE(aligned(d_q, e) && aligned(d_k, e) && aligned(d_q_out, e) && aligned(d_k_out, e) && aligned(d_q_weight, e) &&
                    aligned(d_k_weight, e) && aligned(d_table, 4) && aligned(d_positions, 4), "alignment");
    if (int s = api_check_buffers(-1, {d_q, d_k, d_q_weight, d_k_weight, d_positions, d_table, d_q_out, d_k_out})) return s;
    RopeParams p{};
    p.q = d_q; p.k = d_k; p.q_out = d_q_out; p.k_out = d_k_out;
    p.q_token = q_token; p.q_head = q_head; p.k_token = k_token; p.k_head = k_head;
    p.qo_token = qo_token; p.qo_head = qo_head; p.ko_token = ko_token; p.ko_head = ko_head;
    p.wq = d_q_weight; p.wk = d_k_weight; p.at = d_positions; p.table = d_table;
    p.tokens = tokens; p.positions = positions; p.rot = rot; p.layout = layout; p.norm = norm;
    p.heads = heads; p.kv_heads = kv_heads; p.dim = dim; p.type = type; p.eps = eps;
    p.share = norm == VDT_NORM_RMS ? 1.0f / (float)dim : 1.0f;
    return launched(launch_qk_norm_rope(p, static_cast<cudaStream_t>(stream)), "qk_norm_rope");
}

extern "C" int vdt_rope_table(int positions, int rot, double base, int scaling, double factor, int trained, double fast,
                              double slow, float* d_table, vdt_stream stream) {
    api_clear_error();
    SEQ_REQUIRE(positions >= 0 && rot > 0 && rot % 2 == 0 && rot <= 8192, "positions or rot");
    SEQ_REQUIRE(base > 1.0 && std::isfinite(base), "base must be above 1");
    SEQ_REQUIRE(scaling >= VDT_SCALE_NONE && scaling <= VDT_SCALE_PARTS, "scaling");
    TableParams p{positions, rot, scaling, base, factor, 0.0, 0.0, d_table};
    if (scaling != VDT_SCALE_NONE) SEQ_REQUIRE(factor >= 1.0 && std::isfinite(factor), "factor must be at least 1");
    if (scaling == VDT_SCALE_BASE) {
        SEQ_REQUIRE(rot > 2, "VDT_SCALE_BASE needs rot above 2");
        p.base = base * std::pow(factor, (double)rot / (rot - 2));
    }
    if (scaling == VDT_SCALE_PARTS) {
        SEQ_REQUIRE(trained > 0 && slow > 0.0 && fast > slow && std::isfinite(fast), "trained, fast and slow");
        // the i whose frequency turns n times over the trained length
        auto turns = [&](double n) { return rot * std::log(trained / (n * 6.283185307179586)) / (2.0 * std::log(base)); };
        p.low = std::fmax(std::floor(turns(fast)), 0.0);
        p.high = std::fmin(std::ceil(turns(slow)), rot - 1.0);
    }
    if (!positions) return VDT_OK;
    SEQ_REQUIRE(d_table && aligned(d_table, 4), "table");
    if (int s = api_check_buffers(-1, {d_table})) return s;
    return launched(launch_rope_table(p, static_cast<cudaStream_t>(stream)), "rope_table");
}

extern "C" int vdt_cache_append(const vdt_cache8* cache, const void* d_k, int64_t k_token, int64_t k_head,
                                const void* d_v, int64_t v_token, int64_t v_head, int type, const int32_t* d_pages,
                                int width, const int32_t* d_held, const int32_t* d_starts, int seqs, int64_t total,
                                int most, vdt_stream stream) {
    api_clear_error();
    if (int s = check_cache(cache)) return s;
    SEQ_REQUIRE(type_ok(type), "type");
    if (int s = check_rows(d_pages, width, d_held, d_starts, seqs, total, most)) return s;
    if (!seqs || !total || !most) return VDT_OK;
    SEQ_REQUIRE(d_k && d_v, "NULL buffer");
    SEQ_REQUIRE(aligned(d_k, type_size(type)) && aligned(d_v, type_size(type)), "alignment");
    if (int s = api_check_buffers(-1, {cache->k, cache->v, cache->k_scale, cache->v_scale, d_k, d_v, d_pages, d_held, d_starts})) return s;
    return launched(launch_cache_append(*cache, cache_rows(d_pages, width, d_held, d_starts, seqs, total, most), d_k, d_v, type,
                                        k_token, k_head, v_token, v_head, static_cast<cudaStream_t>(stream)), "cache_append");
}

extern "C" int vdt_cache_load(const vdt_cache8* cache, const int32_t* d_pages, int width, const int32_t* d_kept,
                              const int32_t* d_starts, int seqs, int64_t total, int most, int type, void* d_k,
                              void* d_v, vdt_stream stream) {
    api_clear_error();
    if (int s = check_cache(cache)) return s;
    SEQ_REQUIRE(type_ok(type), "type");
    if (int s = check_rows(d_pages, width, d_kept, d_starts, seqs, total, most)) return s;
    if (!seqs || !total || !most) return VDT_OK;
    SEQ_REQUIRE(d_k && d_v, "NULL buffer");
    SEQ_REQUIRE(aligned(d_k, 16) && aligned(d_v, 16), "outputs must start on 16-byte boundaries");
    if (int s = api_check_buffers(-1, {cache->k, cache->v, cache->k_scale, cache->v_scale, d_k, d_v, d_pages, d_kept, d_starts})) return s;
    return launched(launch_cache_load(*cache, cache_rows(d_pages, width, d_kept, d_starts, seqs, total, most), d_k, d_v, type,
                                      static_cast<cudaStream_t>(stream)), "cache_load");
}

extern "C" size_t vdt_cache_attention_scratch_bytes(int64_t total, int heads, int kv_heads, int dim, int seqs, int most,
                                                    int most_kept) {
    if (total <= 0 || kv_heads <= 0 || heads < kv_heads || heads % kv_heads || dim <= 0 || seqs <= 0 || most <= 0 || most_kept < 0) return 0;
    return attend_scratch_bytes(total, heads, kv_heads, dim, seqs, most, most_kept);
}

extern "C" int vdt_cache_attention(const vdt_cache8* cache, const void* d_q, int64_t q_token, int64_t q_head, int heads,
                                   int type, const int32_t* d_pages, int width, const int32_t* d_kept,
                                   const int32_t* d_starts, int seqs, int64_t total, int most, int most_kept, int causal,
                                   float scale, void* d_out, int64_t out_token, int64_t out_head, void* d_scratch,
                                   size_t scratch_bytes, vdt_stream stream) {
    api_clear_error();
    if (int s = check_cache(cache)) return s;
    if (type != VDT_F16 && type != VDT_BF16)
        return api_fail(type == VDT_F32 ? VDT_ERR_UNSUPPORTED : VDT_ERR_INVALID, "attention takes f16 or bf16 queries");
    SEQ_REQUIRE(heads > 0 && heads <= kMostHeads && heads % cache->heads == 0, "heads must be a multiple of the cache's");
    if (int s = check_rows(d_pages, width, d_kept, d_starts, seqs, total, most)) return s;
    SEQ_REQUIRE(most_kept >= 0 && most_kept <= kMostTokens, "most_kept");
    SEQ_REQUIRE(std::isfinite(scale), "scale");
    if (!seqs || !total || !most) return VDT_OK;
    SEQ_REQUIRE(d_q && d_out, "NULL buffer");
    SEQ_REQUIRE(aligned(d_q, 2) && aligned(d_out, 2), "alignment");
    const size_t need = attend_scratch_bytes(total, heads, cache->heads, cache->dim, seqs, most, most_kept);
    if (need > scratch_bytes || (need && !d_scratch))
        return api_fail(VDT_ERR_CAPACITY, "scratch smaller than vdt_cache_attention_scratch_bytes");
    SEQ_REQUIRE(aligned(d_scratch, 16), "scratch alignment");
    if (!attend_fits(cache->dim, heads, cache->heads, most))
        return api_fail(VDT_ERR_UNSUPPORTED, "too many query rows in one sequence: give them in parts");
    if (int s = api_check_buffers(-1, {cache->k, cache->v, cache->k_scale, cache->v_scale, d_q, d_out, d_pages, d_kept, d_starts, d_scratch})) return s;
    AttendParams p{};
    p.c = *cache;
    p.r = cache_rows(d_pages, width, d_kept, d_starts, seqs, total, most);
    p.q = d_q; p.out = d_out;
    p.q_token = q_token; p.q_head = q_head; p.out_token = out_token; p.out_head = out_head;
    p.heads = heads; p.type = type; p.causal = causal != 0; p.most_kept = most_kept;
    p.scale = scale * 1.44269504088896340736f;       // the softmax works in powers of two
    p.scratch = static_cast<float*>(d_scratch);
    return launched(launch_cache_attention(p, static_cast<cudaStream_t>(stream)), "cache_attention");
}

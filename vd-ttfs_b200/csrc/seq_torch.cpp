// seq_torch.cpp -- vdttfs.seq's calls for torch tensors: checks of the
// tensors, room for the results, the C entry point (include/vdttfs.h).
//
// A native module and not ctypes because a decoder calls these once for every
// layer and token: the same checks and the call through ctypes took 24 us of
// host time for one token's product, whose kernels take 6.  torch provides
// memory and streams only.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>

#include "vdttfs.h"

namespace {

using at::Tensor;

const Tensor kNone;

// ------------------------------------------------------------- arguments --
const Tensor& tensor(PyObject* o, const char* what) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": a tensor is wanted, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
const Tensor& tensor_or_none(PyObject* o, const char* what) { return o == Py_None ? kNone : tensor(o, what); }

int64_t integer(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, what, ": a whole number is wanted");
    }
    return v;
}
// a number or a tensor's size as the library takes it
int size32(int64_t v, const char* what) {
    TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, what, ": out of range");
    return (int)v;
}
int small_integer(PyObject* o, const char* what) { return size32(integer(o, what), what); }
double number(PyObject* o, const char* what) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, what, ": a number is wanted");
    }
    return v;
}
bool truth(PyObject* o, const char* what) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, what, ": true or false is wanted");
    }
    return v == 1;
}

int type_of(at::ScalarType t, const char* what) {
    if (t == at::kBFloat16) return VDT_BF16;
    if (t == at::kHalf) return VDT_F16;
    TORCH_CHECK_VALUE(t == at::kFloat, what, ": float32, float16 or bfloat16 is wanted, got ", t);
    return VDT_F32;
}
at::ScalarType dtype(PyObject* o, const char* what) {
    TORCH_CHECK_TYPE(THPDtype_Check(o), what, ": a torch dtype is wanted");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

void on_device(const Tensor& t, const char* what, int64_t dims) {
    TORCH_CHECK_VALUE(t.is_cuda(), what, ": a CUDA tensor is wanted");
    TORCH_CHECK_VALUE(t.dim() == dims, what, ": ", dims, " dimensions are wanted, got ", t.sizes());
}
void flat(const Tensor& t, const char* what, at::ScalarType type, int64_t n) {
    TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == type && t.numel() == n && t.is_contiguous(), what, ": ", n,
                      " contiguous CUDA values of ", type, " are wanted, got ", t.sizes(), " of ", t.scalar_type(), " on ", t.device());
}
void heads(const Tensor& t, const char* what, int64_t dim) {
    on_device(t, what, 3);
    TORCH_CHECK_VALUE(dim < 0 || t.size(2) == dim, what, ": heads of ", dim, " are wanted, got ", t.sizes());
    TORCH_CHECK_VALUE(t.size(2) == 1 || t.stride(2) == 1, what, ": a head's values must be consecutive");
}

Tensor room(at::IntArrayRef size, at::ScalarType type, at::Device device) {
    return Tensor(at::detail::empty_cuda(size, type, device, std::nullopt));
}

// The call's stream.  One of the caller's own is torch's current one for the
// length of the call: copies that the call makes of its inputs run on it, and
// what the call allocates comes from that stream's memory.  A block of another
// stream's could still be in use by what is queued there.
class OnStream {
public:
    OnStream(PyObject* o, at::Device device) : before_(c10::cuda::getCurrentCUDAStream(device.index())), handle_(before_.stream()) {
        if (o == Py_None) return;
        handle_ = PyLong_AsVoidPtr(o);
        if (!handle_ && PyErr_Occurred()) {
            PyErr_Clear();
            TORCH_CHECK_TYPE(false, "stream: a raw handle is wanted");
        }
        if (handle_ == before_.stream()) return;
        guard_.emplace(handle_ ? c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(handle_), device.index())
                               : c10::cuda::getDefaultCUDAStream(device.index()));
    }
    void* handle() const { return handle_; }
    // A result that the call made: it may go on on the stream that was current,
    // so its memory waits for that one, too, once it is let go
    const Tensor& result(const Tensor& t) const {
        if (guard_ && t.defined() && t.numel()) t.record_stream(before_.unwrap());
        return t;
    }

private:
    c10::cuda::CUDAStream before_;
    void* handle_;
    std::optional<c10::cuda::CUDAStreamGuard> guard_;
};

template <typename T = void>
T* at_or_null(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// vdttfs._lib.VdtError for a status that is not VDT_OK
PyObject* status_error(int status, const char* what) {
    PyObject* module = PyImport_ImportModule("vdttfs._lib");
    if (!module) return nullptr;
    PyObject* type = PyObject_GetAttrString(module, "VdtError");
    Py_DECREF(module);
    if (!type) return nullptr;
    const char* detail = vdt_last_error();
    PyObject* e = PyObject_CallFunction(type, "iss", status, what, detail && *detail ? detail : vdt_strerror(status));
    if (e) {
        PyErr_SetObject(type, e);
        Py_DECREF(e);
    }
    Py_DECREF(type);
    return nullptr;
}

PyObject* pair(const Tensor& a, const Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
    PyObject* t = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

bool arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments are wanted, got %zd", want, n);
    return false;
}
#define WANT(n) \
    if (!arguments(count, n)) return nullptr

// --------------------------------------------------------- 8-bit product --
void code_rows(const Tensor& t, const char* what) {
    on_device(t, what, 2);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kChar, what, ": int8 is wanted, got ", t.scalar_type());
    const int64_t n = t.size(0), k = t.size(1);
    TORCH_CHECK_VALUE(k > 0 && t.stride(1) == 1 && (n <= 1 || t.stride(0) >= k) && t.stride(0) % 16 == 0 &&
                          reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                      what, ": rows that start on 16-byte boundaries are wanted (see quantize_rows), got ", t.sizes(), ", strides ",
                      t.strides());
    TORCH_CHECK_VALUE(!n || t.storage_offset() + (n - 1) * t.stride(0) + (k + 15) / 16 * 16 <= (int64_t)t.storage().nbytes(), what,
                      ": the last row's storage must reach to the next multiple of 16 bytes");
}
int64_t row_stride(const Tensor& t) { return std::max(t.stride(0), (t.size(1) + 15) / 16 * 16); }

// checks of what both products take; the output, new or the caller's
Tensor product_out(int64_t rows, int64_t inner, const Tensor& w, const Tensor& w_scale, const Tensor& bias, const Tensor& out,
                   at::ScalarType type) {
    code_rows(w, "w");
    const int64_t n = w.size(0);
    TORCH_CHECK_VALUE(n > 0 && inner == w.size(1), "rows of ", inner, " and weights ", w.sizes(), " do not multiply");
    flat(w_scale, "w_scale", at::kFloat, n);
    if (bias.defined()) flat(bias, "bias", at::kFloat, n);
    if (!out.defined()) return room({rows, n}, type, w.device());
    on_device(out, "out", 2);
    TORCH_CHECK_VALUE(out.size(0) == rows && out.size(1) == n && (n == 1 || out.stride(1) == 1) && (rows <= 1 || out.stride(0) >= n),
                      "out: [", rows, ", ", n, "] with consecutive columns is wanted, got ", out.sizes(), ", strides ", out.strides());
    return out;
}

PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(2);
    Tensor x = tensor(a[0], "x");
    on_device(x, "x", 2);
    const int type = type_of(x.scalar_type(), "x");
    const int64_t rows = x.size(0), cols = x.size(1);
    TORCH_CHECK_VALUE(cols > 0, "x: no columns");
    const int n = size32(cols, "x: columns");
    const OnStream on(a[1], x.device());
    if (x.stride(1) != 1 || (rows > 1 && x.stride(0) < cols)) x = x.contiguous();
    const int64_t step = (cols + 15) / 16 * 16;
    const Tensor codes = room({rows, step}, at::kChar, x.device()), scale = room({rows}, at::kFloat, x.device());
    if (const int e = vdt_quantize_rows(x.data_ptr(), type, rows, n, x.stride(0), static_cast<int8_t*>(codes.data_ptr()), step,
                                        static_cast<float*>(scale.data_ptr()), on.handle()))
        return status_error(e, "vdt_quantize_rows");
    return pair(on.result(codes).narrow(1, 0, cols), on.result(scale));
    END_HANDLE_TH_ERRORS
}

PyObject* int8_matmul(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(8);
    const Tensor &x = tensor(a[0], "a"), &xs = tensor(a[1], "a_scale"), &w = tensor(a[2], "w"), &ws = tensor(a[3], "w_scale");
    const Tensor &bias = tensor_or_none(a[4], "bias"), &given = tensor_or_none(a[6], "out");
    code_rows(x, "a");
    const OnStream on(a[7], x.device());
    const int64_t rows = x.size(0);
    flat(xs, "a_scale", at::kFloat, rows);
    const Tensor out = product_out(rows, x.size(1), w, ws, bias, given, given.defined() ? given.scalar_type() : dtype(a[5], "out_dtype"));
    const int type = type_of(out.scalar_type(), "out");
    const int n = size32(w.size(0), "w: rows");
    if (const int e = vdt_int8_matmul(static_cast<int8_t*>(x.data_ptr()), row_stride(x), at_or_null<float>(xs),
                                      static_cast<int8_t*>(w.data_ptr()), row_stride(w), at_or_null<float>(ws), at_or_null<float>(bias),
                                      rows, n, size32(x.size(1), "a: columns"), type, out.data_ptr(), std::max<int64_t>(out.stride(0), n), on.handle()))
        return status_error(e, "vdt_int8_matmul");
    return THPVariable_Wrap(given.defined() ? out : on.result(out));
    END_HANDLE_TH_ERRORS
}

PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(7);
    Tensor x = tensor(a[0], "x");
    const Tensor &w = tensor(a[1], "w"), &ws = tensor(a[2], "w_scale"), &bias = tensor_or_none(a[3], "bias");
    const Tensor& given = tensor_or_none(a[5], "out");
    on_device(x, "x", 2);
    const OnStream on(a[6], x.device());
    const int type = type_of(x.scalar_type(), "x");
    const int64_t rows = x.size(0), inner = x.size(1);
    const Tensor out = product_out(rows, inner, w, ws, bias, given,
                                   given.defined() ? given.scalar_type() : a[4] == Py_None ? x.scalar_type() : dtype(a[4], "out_dtype"));
    const int out_type = type_of(out.scalar_type(), "out");
    if ((inner > 1 && x.stride(1) != 1) || (rows > 1 && x.stride(0) < inner)) x = x.contiguous();
    const int k = size32(inner, "x: columns");
    const int64_t need = (int64_t)vdt_int8_linear_scratch_bytes(rows, k);
    const Tensor scratch = room({need}, at::kByte, x.device());
    const int n = size32(w.size(0), "w: rows");
    if (const int e = vdt_int8_linear(x.data_ptr(), type, std::max(x.stride(0), inner), static_cast<int8_t*>(w.data_ptr()), row_stride(w),
                                      at_or_null<float>(ws), at_or_null<float>(bias), rows, n, k, out_type, out.data_ptr(),
                                      std::max<int64_t>(out.stride(0), n), scratch.data_ptr(), (size_t)need, on.handle()))
        return status_error(e, "vdt_int8_linear");
    return THPVariable_Wrap(given.defined() ? out : on.result(out));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------- head norms, rotation --
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(12);
    const Tensor &q = tensor(a[0], "q"), &k = tensor_or_none(a[1], "k"), &wq = tensor_or_none(a[2], "q_weight");
    const Tensor &wk = tensor_or_none(a[3], "k_weight"), &at = tensor_or_none(a[4], "positions"), &table = tensor_or_none(a[5], "table");
    const int layout = truth(a[6], "interleaved") ? VDT_ROPE_PAIRS : VDT_ROPE_HALF, norm = small_integer(a[7], "norm");
    const Tensor &given_q = tensor_or_none(a[9], "out (q)"), &given_k = tensor_or_none(a[10], "out (k)");
    heads(q, "q", -1);
    const int64_t tokens = q.size(0), dim = q.size(2), kv = k.defined() ? k.size(1) : 0;
    const int type = type_of(q.scalar_type(), "q");
    if (k.defined()) {
        heads(k, "k", dim);
        TORCH_CHECK_VALUE(k.size(0) == tokens && k.scalar_type() == q.scalar_type(), "k: ", tokens, " tokens of ", q.scalar_type(),
                          " are wanted, got ", k.sizes(), " of ", k.scalar_type());
    }
    if (wq.defined()) flat(wq, "q_weight", q.scalar_type(), dim);
    if (wk.defined()) flat(wk, "k_weight", q.scalar_type(), dim);
    int64_t n = 0, rot = 0;
    if (table.defined()) {
        on_device(table, "table", 2);
        n = table.size(0);
        rot = table.size(1);
        flat(table, "table", at::kFloat, n * rot);
        TORCH_CHECK_VALUE(at.defined(), "positions: wanted with a table");
        flat(at, "positions", at::kInt, tokens);
    }
    const OnStream on(a[11], q.device());
    Tensor out[2];
    const Tensor* in[2] = {&q, &k};
    const Tensor* given[2] = {&given_q, &given_k};
    const bool mine = !given_q.defined();
    for (int i = 0; i < 2; ++i) {
        if (!in[i]->defined()) continue;
        if (mine) {
            out[i] = room(in[i]->sizes(), q.scalar_type(), q.device());
        } else {
            out[i] = *given[i];
            TORCH_CHECK_VALUE(out[i].defined(), "out: a pair is wanted");
            heads(out[i], "out", dim);
            TORCH_CHECK_VALUE(out[i].sizes() == in[i]->sizes() && out[i].scalar_type() == q.scalar_type(), "out: ", in[i]->sizes(), " of ",
                              q.scalar_type(), " is wanted");
        }
    }
    auto stride = [](const Tensor& t, int i) { return t.defined() ? t.stride(i) : 0; };
    if (const int e = vdt_qk_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), at_or_null(k), stride(k, 0), stride(k, 1), at_or_null(wq),
                                       at_or_null(wk), rot ? at_or_null<int32_t>(at) : nullptr, rot ? at_or_null<float>(table) : nullptr,
                                       size32(n, "table: positions"), size32(rot, "table: columns"), layout, norm, (float)number(a[8], "eps"),
                                       tokens, size32(q.size(1), "q: heads"), size32(kv, "k: heads"), size32(dim, "q: dimension"), type,
                                       out[0].data_ptr(), out[0].stride(0), out[0].stride(1), at_or_null(out[1]), stride(out[1], 0),
                                       stride(out[1], 1), on.handle()))
        return status_error(e, "vdt_qk_norm_rope");
    if (mine) {
        on.result(out[0]);
        on.result(out[1]);
    }
    if (!out[1].defined()) {
        PyObject* x = THPVariable_Wrap(out[0]);
        PyObject* t = x ? PyTuple_Pack(2, x, Py_None) : nullptr;
        Py_XDECREF(x);
        return t;
    }
    return pair(out[0], out[1]);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------- the cache --
vdt_cache8 cache_of(PyObject* o) {
    TORCH_CHECK_TYPE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4, "cache: a tuple of keys, values and their scales is wanted");
    const Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), "cache keys"), &v = tensor(PyTuple_GET_ITEM(o, 1), "cache values");
    const Tensor &ks = tensor(PyTuple_GET_ITEM(o, 2), "cache key scales"), &vs = tensor(PyTuple_GET_ITEM(o, 3), "cache value scales");
    on_device(k, "cache keys", 4);
    on_device(v, "cache values", 4);
    const int64_t pages = k.size(0), n = k.size(1), page = k.size(2), dim = k.size(3);
    flat(k, "cache keys", at::kChar, k.numel());
    flat(v, "cache values", at::kChar, k.numel());
    TORCH_CHECK_VALUE(v.size(0) == pages && v.size(1) == n && v.size(2) == dim && v.size(3) == page, "cache values: [", pages, ", ", n, ", ", dim,
                      ", ", page, "] is wanted, got ", v.sizes());
    flat(ks, "cache key scales", at::kFloat, pages * n);
    flat(vs, "cache value scales", at::kFloat, pages * n);
    TORCH_CHECK_VALUE(pages <= INT32_MAX && n <= INT32_MAX && page <= INT32_MAX && dim <= INT32_MAX, "cache: too large");
    return {static_cast<int8_t*>(k.data_ptr()), static_cast<int8_t*>(v.data_ptr()), static_cast<float*>(ks.data_ptr()),
            static_cast<float*>(vs.data_ptr()), (int)pages, (int)page, (int)n, (int)dim};
}

struct Rows {
    const int32_t *pages, *held, *starts;
    int seqs, width;
};
Rows rows_of(PyObject* pages, PyObject* held, PyObject* starts) {
    const Tensor& p = tensor(pages, "pages");
    on_device(p, "pages", 2);
    flat(p, "pages", at::kInt, p.numel());
    const int64_t n = p.size(0);
    const Tensor &h = tensor(held, "tokens held"), &s = tensor(starts, "starts");
    flat(h, "tokens held", at::kInt, n);
    flat(s, "starts", at::kInt, n + 1);
    TORCH_CHECK_VALUE(n <= INT32_MAX && p.size(1) <= INT32_MAX, "pages: too large");
    return {static_cast<int32_t*>(p.data_ptr()), static_cast<int32_t*>(h.data_ptr()), static_cast<int32_t*>(s.data_ptr()), (int)n, (int)p.size(1)};
}

PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(8);
    const vdt_cache8 c = cache_of(a[0]);
    const Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    const Rows r = rows_of(a[3], a[4], a[5]);
    heads(k, "k", c.dim);
    heads(v, "v", c.dim);
    const int type = type_of(k.scalar_type(), "k");
    const int64_t total = k.size(0);
    TORCH_CHECK_VALUE(k.size(1) == c.heads && v.size(1) == c.heads && v.size(0) == total && v.scalar_type() == k.scalar_type(),
                      "k and v: [tokens, ", c.heads, ", ", c.dim, "] of one type are wanted, got ", k.sizes(), " of ", k.scalar_type(), " and ",
                      v.sizes(), " of ", v.scalar_type());
    const OnStream on(a[7], k.device());
    const int most = (int)std::min<int64_t>(small_integer(a[6], "most"), total);
    if (const int e = vdt_cache_append(&c, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), type, r.pages,
                                       r.width, r.held, r.starts, r.seqs, total, most, on.handle()))
        return status_error(e, "vdt_cache_append");
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject* cache_load(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(8);
    const vdt_cache8 c = cache_of(a[0]);
    const Rows r = rows_of(a[1], a[2], a[3]);
    const int64_t total = integer(a[4], "total");
    TORCH_CHECK_VALUE(total >= 0, "total: negative");
    const int most = (int)std::min<int64_t>(small_integer(a[5], "most"), total);
    const at::ScalarType type = dtype(a[6], "dtype");
    const int kind = type_of(type, "dtype");
    const at::Device device = tensor(PyTuple_GET_ITEM(a[0], 0), "cache keys").device();
    const OnStream on(a[7], device);
    const Tensor k = room({total, c.heads, c.dim}, type, device), v = room({total, c.heads, c.dim}, type, device);
    if (const int e = vdt_cache_load(&c, r.pages, r.width, r.held, r.starts, r.seqs, total, most, kind, k.data_ptr(), v.data_ptr(), on.handle()))
        return status_error(e, "vdt_cache_load");
    return pair(on.result(k), on.result(v));
    END_HANDLE_TH_ERRORS
}

PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    WANT(11);
    const Tensor& q = tensor(a[0], "q");
    const vdt_cache8 c = cache_of(a[1]);
    const Rows r = rows_of(a[2], a[3], a[4]);
    heads(q, "q", c.dim);
    const int64_t total = q.size(0);
    const int n = size32(q.size(1), "q: heads");
    const int type = type_of(q.scalar_type(), "q");
    const int most = (int)std::min<int64_t>(small_integer(a[5], "most"), total), most_kept = small_integer(a[6], "most_kept");
    const Tensor& given = tensor_or_none(a[9], "out");
    const OnStream on(a[10], q.device());
    const Tensor out = given.defined() ? given : room(q.sizes(), q.scalar_type(), q.device());
    if (given.defined()) {
        heads(out, "out", c.dim);
        TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), "out: ", q.sizes(), " of ", q.scalar_type(), " is wanted");
    }
    const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)c.dim) : number(a[8], "scale");
    const size_t need = vdt_cache_attention_scratch_bytes(total, n, c.heads, c.dim, r.seqs, most, most_kept);
    const Tensor scratch = need ? room({(int64_t)need}, at::kByte, q.device()) : Tensor();
    if (const int e = vdt_cache_attention(&c, q.data_ptr(), q.stride(0), q.stride(1), n, type, r.pages, r.width, r.held, r.starts, r.seqs,
                                          total, most, most_kept, truth(a[7], "causal"), (float)scale, out.data_ptr(), out.stride(0), out.stride(1),
                                          at_or_null(scratch), need, on.handle()))
        return status_error(e, "vdt_cache_attention");
    return THPVariable_Wrap(given.defined() ? out : on.result(out));
    END_HANDLE_TH_ERRORS
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(quantize_rows), METHOD(int8_matmul), METHOD(int8_linear), METHOD(qk_norm_rope),
                          METHOD(cache_append), METHOD(cache_load), METHOD(cache_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_seq", "The sequence operators for torch tensors (see vdttfs.seq).", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__seq(void) { return PyModule_Create(&kModule); }

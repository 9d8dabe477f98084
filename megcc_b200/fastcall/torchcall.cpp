// Operator calls on tensors without their Python attributes. Looking over the tensors of one product and making
// its result takes a Python function 5 us, twice as long as the launch of its kernel and longer than the kernel
// itself for one token; here it takes 1. The calls are the C ABI's: this module only checks, allocates on the
// current stream and passes addresses.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <exception>
#include <string>

#include "../../include/megcc_b200.h"

namespace {

// The library's functions, and what raises an error for a status (set once by bind())
struct Abi {
    decltype(&mb200_quantize_rows_s8) quantize_rows;
    decltype(&mb200_matmul_s8_scaled_workspace_bytes) matmul_workspace;
    decltype(&mb200_matmul_s8_scaled) matmul;
    decltype(&mb200_linear_s8_workspace_bytes) linear_workspace;
    decltype(&mb200_linear_s8) linear;
    decltype(&mb200_moe_s8_workspace_bytes) moe_workspace;
    decltype(&mb200_moe_s8) moe;
    decltype(&mb200_kv_append_s8) kv_append;
    decltype(&mb200_kv_read_s8) kv_read;
    decltype(&mb200_attention_cache_s8_workspace_bytes) cache_workspace;
    decltype(&mb200_attention_cache_s8) attention_cache;
    decltype(&mb200_attention_prompt) attention_prompt;
} abi;
PyObject* on_status = nullptr;
PyObject* out_of_memory = nullptr;  // torch.OutOfMemoryError

// A refused argument: ValueError with this text
struct Refused : std::exception {
    std::string text;
    const char* what() const noexcept override {
        return text.c_str();
    }
};
[[noreturn]] void refuse(const std::string& text) {
    Refused r;
    r.text = text;
    throw r;
}
std::string shown(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i)
        s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ") of " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o))
        refuse(std::string(name) + ": a tensor, not " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? MB200_DTYPE_F32 : t == at::kHalf ? MB200_DTYPE_F16 : t == at::kBFloat16 ? MB200_DTYPE_BF16 : -1;
}

// A matrix of the current device whose rows' elements are neighbours
struct Matrix {
    int m, k;
    long long ld;
    void* p;
};
Matrix rows_of(const at::Tensor& t, bool floats, const char* name) {
    const bool kind = floats ? dtype_code(t.scalar_type()) >= 0 : t.scalar_type() == at::kChar;
    if (!kind || t.dim() != 2 || !t.is_cuda() || t.layout() != at::kStrided)
        refuse(std::string(name) + ": a CUDA matrix of " + (floats ? "fp32, fp16 or bf16" : "int8") + ", not " + shown(t));
    if (t.get_device() != c10::cuda::current_device())
        refuse(std::string(name) + " is on " + t.device().str() + ", not on the current device");
    const int64_t m = t.size(0), k = t.size(1);
    if (k > 1 && t.stride(1) != 1)
        refuse(std::string(name) + ": elements of a row must be neighbours");
    if (m > INT32_MAX || k > INT32_MAX)
        refuse(std::string(name) + ": extents beyond an int, " + shown(t));
    // (torch gives an expanded row stride 0, which the library refuses as overlapping)
    return {(int)m, (int)k, (long long)t.stride(0), t.data_ptr()};
}
const float* vector_of(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* name) {
    if (t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous() || t.device() != like.device())
        refuse(std::string(name) + ": " + std::to_string(n) + " contiguous fp32 values on " + like.device().str() +
               ", not " + shown(t));
    return (const float*)t.data_ptr();
}
const int8_t* weights_of(const at::Tensor& t, int dims, const at::Tensor& like, const char* name) {
    if (t.scalar_type() != at::kChar || t.dim() != dims || !t.is_contiguous() || t.device() != like.device())
        refuse(std::string(name) + ": a contiguous int8 tensor of " + std::to_string(dims) + " dimensions on " +
               like.device().str() + ", not " + shown(t));
    for (int i = 0; i < dims; ++i)
        if (t.size(i) > INT32_MAX)
            refuse(std::string(name) + ": extents beyond an int, " + shown(t));
    return (const int8_t*)t.data_ptr();
}
at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}
// 256-byte aligned device scratch of at least `bytes`. It may be dropped as soon as the kernels are launched: torch
// hands freed memory out again in the order of the stream.
struct Scratch {
    at::Tensor keep;
    void* p = nullptr;
    Scratch(size_t bytes, const at::Tensor& like) {
        if (bytes) {
            keep = make({(int64_t)bytes + 256}, at::kByte, like);
            p = (void*)(((uintptr_t)keep.data_ptr() + 255) & ~(uintptr_t)255);
        }
    }
};
void* stream_of(const at::Tensor& t) {
    return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// false with an error set
bool done(int status) {
    if (status == 0)
        return true;
    PyObject* r = PyObject_CallFunction(on_status, "i", status);
    if (r) {
        Py_DECREF(r);
        PyErr_Format(PyExc_RuntimeError, "TinyNNStatus %d", status);
    }
    return false;
}
bool counted(Py_ssize_t n, Py_ssize_t want) {
    if (n != want)
        PyErr_Format(PyExc_TypeError, "the function takes %zd arguments (%zd given)", want, n);
    return n == want;
}
// C++ exceptions end here
template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(out_of_memory, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
// (an exception on its way to guarded() takes the lock again too)
struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() {
        PyEval_RestoreThread(state);
    }
};
template <class F>
int without_gil(F f) {
    const WithoutGil released;
    return f();
}

PyObject* quantize_rows_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!counted(n, 1))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(args[0], "x");
        const Matrix a = rows_of(x, true, "x");
        at::Tensor q = make({a.m, a.k}, at::kChar, x), scales = make({a.m}, at::kFloat, x);
        const int status = without_gil([&] {
            return abi.quantize_rows(a.p, dtype_code(x.scalar_type()), a.m, a.k, a.ld, (int8_t*)q.data_ptr(), a.k,
                                     (float*)scales.data_ptr(), stream_of(x));
        });
        if (!done(status))
            return nullptr;
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(scales)));
    });
}

PyObject* matmul_s8_scaled(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!counted(n, 6))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &at = tensor(args[0], "a"), &bt = tensor(args[1], "b_packed");
        const Matrix a = rows_of(at, false, "a");
        const int8_t* b = weights_of(bt, 2, at, "b_packed");
        if (bt.size(1) != a.k)
            refuse("b_packed: [n, " + std::to_string(a.k) + "], not " + shown(bt));
        const int cols = (int)bt.size(0);
        const float* sa = vector_of(tensor(args[2], "a_scales"), a.m, at, "a_scales");
        const float* sb = vector_of(tensor(args[3], "b_scales"), cols, at, "b_scales");
        const float* bias = args[4] == Py_None ? nullptr : vector_of(tensor(args[4], "bias"), cols, at, "bias");
        const int type = THPDtype_Check(args[5]) ? dtype_code(((THPDtype*)args[5])->scalar_type) : -1;
        if (type < 0)
            refuse("results are fp32, fp16 or bf16");
        at::Tensor c = make({a.m, cols}, ((THPDtype*)args[5])->scalar_type, at);
        const size_t bytes = abi.matmul_workspace(a.m, cols, a.k, (const int8_t*)a.p, a.ld, b);
        const Scratch ws(bytes, at);
        const int status = without_gil([&] {
            return abi.matmul(a.m, cols, a.k, (const int8_t*)a.p, a.ld, b, sa, sb, bias, c.data_ptr(), type, cols, ws.p,
                              bytes, stream_of(at));
        });
        return done(status) ? THPVariable_Wrap(std::move(c)) : nullptr;
    });
}

PyObject* linear_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!counted(n, 4))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &x = tensor(args[0], "x"), &bt = tensor(args[1], "b_packed");
        const Matrix a = rows_of(x, true, "x");
        const int8_t* b = weights_of(bt, 2, x, "b_packed");
        if (bt.size(1) != a.k)
            refuse("b_packed: [n, " + std::to_string(a.k) + "], not " + shown(bt));
        const int cols = (int)bt.size(0);
        const float* sb = vector_of(tensor(args[2], "b_scales"), cols, x, "b_scales");
        const float* bias = args[3] == Py_None ? nullptr : vector_of(tensor(args[3], "bias"), cols, x, "bias");
        at::Tensor y = make({a.m, cols}, x.scalar_type(), x);
        const size_t bytes = abi.linear_workspace(a.m, cols, a.k, b);
        const Scratch ws(bytes, x);
        const int status = without_gil([&] {
            return abi.linear(a.m, cols, a.k, a.p, dtype_code(x.scalar_type()), a.ld, b, sb, bias, y.data_ptr(), cols,
                              ws.p, bytes, stream_of(x));
        });
        return done(status) ? THPVariable_Wrap(std::move(y)) : nullptr;
    });
}

PyObject* moe_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!counted(n, 8))
        return nullptr;
    const long top = PyLong_AsLong(args[6]);
    const int renormalize = PyObject_IsTrue(args[7]);
    if ((top == -1 && PyErr_Occurred()) || renormalize < 0)
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &x = tensor(args[0], "x"), &logits = tensor(args[1], "logits");
        const at::Tensor &w1 = tensor(args[2], "w1"), &w2 = tensor(args[4], "w2");
        const Matrix a = rows_of(x, true, "x");
        if (logits.dim() != 2 || logits.size(0) != a.m)
            refuse("logits: [" + std::to_string(a.m) + ", experts], not " + shown(logits));
        const int64_t e = logits.size(1);
        const float* pl = vector_of(logits, a.m * e, x, "logits");
        const int8_t *p1 = weights_of(w1, 3, x, "w1"), *p2 = weights_of(w2, 3, x, "w2");
        const int64_t f = w2.size(2);
        if (w1.size(0) != e || w2.size(0) != e || w1.size(1) != 2 * f || w1.size(2) != a.k || w2.size(1) != a.k)
            refuse("w1: [experts, 2 f, d] and w2: [experts, d, f] over rows of " + std::to_string(a.k) + " and " +
                   std::to_string(e) + " experts, not " + shown(w1) + " and " + shown(w2));
        const float* s1 = vector_of(tensor(args[3], "w1_scales"), e * 2 * f, x, "w1_scales");
        const float* s2 = vector_of(tensor(args[5], "w2_scales"), e * a.k, x, "w2_scales");
        if (e > INT32_MAX || top > INT32_MAX || top < INT32_MIN)
            refuse("moe_s8: " + std::to_string(top) + " of " + std::to_string(e) + " experts");
        const mb200_moe_param p = {a.m, a.k, (int)f, (int)e, (int)top, renormalize, dtype_code(x.scalar_type())};
        at::Tensor y = make({a.m, a.k}, x.scalar_type(), x);
        const size_t bytes = abi.moe_workspace(&p);
        const Scratch ws(bytes, x);
        const int status = without_gil([&] {
            return abi.moe(&p, a.p, a.ld, pl, p1, s1, p2, s2, y.data_ptr(), a.k, ws.p, bytes, stream_of(x));
        });
        return done(status) ? THPVariable_Wrap(std::move(y)) : nullptr;
    });
}

// ---- attention with the int8 cache ----
// A whole number of Python's that an int holds, or an error
bool int_of(PyObject* o, int* v) {
    const long n = PyLong_AsLong(o);
    if (n == -1 && PyErr_Occurred())
        return false;
    if (n > INT32_MAX || n < INT32_MIN) {
        PyErr_Format(PyExc_ValueError, "%ld is beyond an int", n);
        return false;
    }
    *v = (int)n;
    return true;
}
void on_current_device(const at::Tensor& t, const char* name) {
    if (!t.is_cuda() || t.layout() != at::kStrided)
        refuse(std::string(name) + ": a CUDA tensor, not " + shown(t));
    if (t.get_device() != c10::cuda::current_device())
        refuse(std::string(name) + " is on " + t.device().str() + ", not on the current device");
}
int extent(const at::Tensor& t, int dim, const char* name) {
    if (t.size(dim) > INT32_MAX)
        refuse(std::string(name) + ": extents beyond an int, " + shown(t));
    return (int)t.size(dim);
}
// The cache's tensors k, v, k_scales, v_scales and the block table
mb200_kv_cache cache_of(PyObject* const* args) {
    const at::Tensor &k = tensor(args[0], "cache.k"), &v = tensor(args[1], "cache.v"), &ks = tensor(args[2], "cache.k_scales"),
                     &vs = tensor(args[3], "cache.v_scales"), &table = tensor(args[4], "block_table");
    on_current_device(k, "cache.k");
    weights_of(k, 4, k, "cache.k");
    weights_of(v, 4, k, "cache.v");
    if (v.sizes() != k.sizes())
        refuse("cache.v: of the shape of cache.k, not " + shown(v));
    mb200_kv_cache c{};
    c.pages = extent(k, 0, "cache.k"), c.kv_heads = extent(k, 1, "cache.k");
    c.page_tokens = extent(k, 2, "cache.k"), c.d = extent(k, 3, "cache.k");
    if (c.page_tokens % MB200_KV_BLOCK)
        refuse("cache.k: pages of a multiple of " + std::to_string(MB200_KV_BLOCK) + " positions, not " + shown(k));
    for (const at::Tensor* s : {&ks, &vs}) {
        const char* name = s == &ks ? "cache.k_scales" : "cache.v_scales";
        if (s->dim() != 3 || s->size(0) != c.pages || s->size(1) != c.kv_heads ||
            s->size(2) != c.page_tokens / MB200_KV_BLOCK)
            refuse(std::string(name) + ": a scale for each block of " + std::to_string(MB200_KV_BLOCK) +
                   " positions of a page and head, not " + shown(*s));
        vector_of(*s, s->numel(), k, name);
    }
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.device() != k.device() ||
        (table.size(1) > 1 && table.stride(1) != 1))
        refuse("block_table: [sequences, pages] int32 on " + k.device().str() + ", rows' elements neighbours, not " +
               shown(table));
    c.batch = extent(table, 0, "block_table"), c.table_pages = extent(table, 1, "block_table");
    c.table_stride = table.stride(0);
    c.k = (int8_t*)k.data_ptr(), c.v = (int8_t*)v.data_ptr();
    c.k_scales = (float*)ks.data_ptr(), c.v_scales = (float*)vs.data_ptr();
    c.block_table = (const int32_t*)table.data_ptr();
    return c;
}
const int32_t* ints_of(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* name) {
    if (t.scalar_type() != at::kInt || t.numel() != n || !t.is_contiguous() || t.device() != like.device())
        refuse(std::string(name) + ": " + std::to_string(n) + " contiguous int32 values on " + like.device().str() +
               ", not " + shown(t));
    return (const int32_t*)t.data_ptr();
}
// [tokens, heads, d] of fp16 or bf16 whose heads' elements are neighbours
mb200_heads heads_of(const at::Tensor& t, const at::Tensor& like, const char* name) {
    if (dtype_code(t.scalar_type()) <= 0 || t.dim() != 3 || t.scalar_type() != like.scalar_type())
        refuse(std::string(name) + ": [tokens, heads, elements] of fp16 or bf16, all operands alike, not " + shown(t));
    on_current_device(t, name);
    if (t.size(2) > 1 && t.stride(2) != 1)
        refuse(std::string(name) + ": elements of a head must be neighbours");
    extent(t, 0, name), extent(t, 1, name), extent(t, 2, name);
    return {t.data_ptr(), (long long)t.stride(0), (long long)t.stride(1)};
}
mb200_heads heads_of(const at::Tensor& t, int64_t tokens, int64_t heads, int64_t d, const at::Tensor& like, const char* name) {
    const mb200_heads h = heads_of(t, like, name);
    if (t.size(0) != tokens || t.size(1) != heads || t.size(2) != d)
        refuse(std::string(name) + ": [" + std::to_string(tokens) + ", " + std::to_string(heads) + ", " + std::to_string(d) +
               "], not " + shown(t));
    return h;
}
PyObject* wrapped_or_none(at::Tensor&& t) {
    if (!t.defined())
        Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(t));
}

PyObject* kv_append_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!counted(n, 14))
        return nullptr;
    const int interleaved = PyObject_IsTrue(args[12]), turned_keys = PyObject_IsTrue(args[13]);
    if (interleaved < 0 || turned_keys < 0)
        return nullptr;
    return guarded([&]() -> PyObject* {
        const mb200_kv_cache c = cache_of(args);
        const at::Tensor& k = tensor(args[6], "k");
        mb200_kv_append_param p{};
        const int64_t tokens = k.dim() ? k.size(0) : 0;
        p.k = heads_of(k, tokens, c.kv_heads, c.d, k, "k");
        p.v = heads_of(tensor(args[7], "v"), tokens, c.kv_heads, c.d, k, "v");
        p.tokens = (int)tokens, p.dtype = dtype_code(k.scalar_type());
        p.lengths = ints_of(tensor(args[5], "lengths"), c.batch, k, "lengths");
        if (args[11] != Py_None)
            p.cu = ints_of(tensor(args[11], "cu_tokens"), (int64_t)c.batch + 1, k, "cu_tokens");
        else if (tokens != c.batch)
            refuse("k: a token for each of " + std::to_string(c.batch) + " sequences (or cu_tokens), not " + shown(k));
        if ((args[9] == Py_None) != (args[10] == Py_None))
            refuse("cos and sin: both or none");
        if (args[9] != Py_None) {
            const at::Tensor& cosines = tensor(args[9], "cos");
            if (cosines.dim() != 2)
                refuse("cos: [positions, turned elements / 2], not " + shown(cosines));
            p.positions = extent(cosines, 0, "cos");
            const int64_t half = cosines.size(1);
            if (half > INT32_MAX / 2)
                refuse("cos: extents beyond an int, " + shown(cosines));
            p.rot_dims = (int)(2 * half);
            p.cosines = vector_of(cosines, p.positions * half, k, "cos");
            const at::Tensor& sines = tensor(args[10], "sin");
            if (sines.sizes() != cosines.sizes())
                refuse("sin: of the shape of cos, not " + shown(sines));
            p.sines = vector_of(sines, p.positions * half, k, "sin");
        }
        p.interleaved = interleaved;
        at::Tensor q_out, k_out;
        if (args[8] != Py_None) {
            const at::Tensor& q = tensor(args[8], "q");
            if (q.dim() != 3)
                refuse("q: [tokens, heads, elements], not " + shown(q));
            if (args[9] == Py_None)
                refuse("q is only turned, which needs cos and sin");
            p.q = heads_of(q, tokens, q.size(1), c.d, k, "q");
            p.heads = extent(q, 1, "q");
            q_out = make({tokens, p.heads, c.d}, k.scalar_type(), k);
            p.q_out = {q_out.data_ptr(), (long long)p.heads * c.d, c.d};
        }
        if (turned_keys) {
            k_out = make({tokens, c.kv_heads, c.d}, k.scalar_type(), k);
            p.k_out = {k_out.data_ptr(), (long long)c.kv_heads * c.d, c.d};
        }
        const int status = without_gil([&] { return abi.kv_append(&c, &p, stream_of(k)); });
        if (!done(status))
            return nullptr;
        return Py_BuildValue("NN", wrapped_or_none(std::move(q_out)), wrapped_or_none(std::move(k_out)));
    });
}

PyObject* kv_read_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    int tokens;
    if (!counted(n, 9) || !int_of(args[7], &tokens))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const mb200_kv_cache c = cache_of(args);
        const at::Tensor& like = tensor(args[0], "cache.k");
        const int32_t* starts = args[5] == Py_None ? nullptr : ints_of(tensor(args[5], "starts"), c.batch, like, "starts");
        const int32_t* cu = ints_of(tensor(args[6], "cu_tokens"), (int64_t)c.batch + 1, like, "cu_tokens");
        const int type = THPDtype_Check(args[8]) ? dtype_code(((THPDtype*)args[8])->scalar_type) : -1;
        if (type <= 0)
            refuse("results are fp16 or bf16");
        if (tokens < 0)
            refuse("kv_read_s8: " + std::to_string(tokens) + " tokens");
        at::Tensor k = make({tokens, c.kv_heads, c.d}, ((THPDtype*)args[8])->scalar_type, like);
        at::Tensor v = make({tokens, c.kv_heads, c.d}, ((THPDtype*)args[8])->scalar_type, like);
        const mb200_heads hk = {k.data_ptr(), (long long)c.kv_heads * c.d, c.d};
        const mb200_heads hv = {v.data_ptr(), (long long)c.kv_heads * c.d, c.d};
        const int status = without_gil([&] { return abi.kv_read(&c, starts, cu, tokens, type, &hk, &hv, stream_of(like)); });
        if (!done(status))
            return nullptr;
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
    });
}

// scale, or 1 / sqrt(d) for None; false with an error set
bool scale_of(PyObject* o, double* scale) {
    *scale = o == Py_None ? 0.0 : PyFloat_AsDouble(o);
    return !(*scale == -1.0 && PyErr_Occurred());
}
// The result that the caller brought, or a new one like q
at::Tensor result_for(PyObject* o, const at::Tensor& q) {
    if (o == Py_None)
        return make(q.sizes(), q.scalar_type(), q);
    const at::Tensor& out = tensor(o, "out");
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || out.device() != q.device())
        refuse("out: a tensor like q, not " + shown(out));
    return out;
}

PyObject* attention_cache_s8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    double scale;
    if (!counted(n, 9) || !scale_of(args[7], &scale))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const mb200_kv_cache c = cache_of(args + 1);
        const at::Tensor& q = tensor(args[0], "q");
        at::Tensor out = result_for(args[8], q);
        if ((q.dim() != 3 && q.dim() != 4) || q.size(0) != c.batch)
            refuse("q: [" + std::to_string(c.batch) + ", heads, elements] or [" + std::to_string(c.batch) +
                   ", queries, heads, elements], not " + shown(q));
        const int queries = q.dim() == 4 ? extent(q, 1, "q") : 1;
        // all queries as one line of tokens
        auto line = [&](const at::Tensor& t, const char* name) {
            if (t.dim() == 3)
                return heads_of(t, q, name);
            if (t.size(0) > 1 && t.size(1) > 1 && t.stride(0) != t.stride(1) * t.size(1))
                refuse(std::string(name) + ": sequences must lie as far apart as their queries take");
            const mb200_heads h = heads_of(t.select(1, 0), q, name);
            return mb200_heads{h.p, (long long)(t.size(1) > 1 ? t.stride(1) : t.stride(0)), h.head_stride};
        };
        if (queries == 0 || q.size(q.dim() - 2) == 0 || q.size(q.dim() - 1) != c.d)
            refuse("q: heads of " + std::to_string(c.d) + " elements, not " + shown(q));
        const mb200_heads hq = line(q, "q"), ho = line(out, "out");
        const int heads = extent(q, q.dim() - 2, "q");
        const at::Tensor& lt = tensor(args[6], "lengths");
        const int32_t* lengths = ints_of(lt, c.batch, q, "lengths");
        if (args[7] == Py_None)
            scale = 1 / std::sqrt((double)c.d);
        const size_t bytes = abi.cache_workspace(&c, heads, queries);
        const Scratch ws(bytes, q);
        const int status = without_gil([&] {
            return abi.attention_cache(&c, lengths, heads, queries, dtype_code(q.scalar_type()), &hq, (float)scale, &ho,
                                       ws.p, bytes, stream_of(q));
        });
        return done(status) ? THPVariable_Wrap(std::move(out)) : nullptr;
    });
}

PyObject* attention_prompt(PyObject*, PyObject* const* args, Py_ssize_t n) {
    double scale;
    if (!counted(n, 8) || !scale_of(args[6], &scale))
        return nullptr;
    const int causal = PyObject_IsTrue(args[5]);
    if (causal < 0)
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(args[0], "q"), &k = tensor(args[1], "k"), &cu = tensor(args[3], "cu_q");
        const mb200_heads hq = heads_of(q, q, "q"), hk = heads_of(k, q, "k");
        const int64_t d = q.size(2);
        if (k.size(2) != d)
            refuse("k: heads of " + std::to_string(d) + " elements, not " + shown(k));
        const mb200_heads hv = heads_of(tensor(args[2], "v"), k.size(0), k.size(1), d, q, "v");
        at::Tensor out = result_for(args[7], q);
        const mb200_heads ho = heads_of(out, q, "out");
        if (cu.numel() < 1 || cu.numel() > INT32_MAX)
            refuse("cu_q: sequences + 1 int32 values, not " + shown(cu));
        const int32_t* cu_q = ints_of(cu, cu.numel(), q, "cu_q");
        const int32_t* cu_k = args[4] == Py_None ? nullptr : ints_of(tensor(args[4], "cu_k"), cu.numel(), q, "cu_k");
        if (!cu_k && k.size(0) != q.size(0))
            refuse("k: of as many tokens as q (or cu_k), not " + shown(k));
        if (args[6] == Py_None)
            scale = 1 / std::sqrt((double)d);
        const int status = without_gil([&] {
            return abi.attention_prompt((int)cu.numel() - 1, cu_q, cu_k, (int)q.size(0), (int)k.size(0), (int)q.size(1),
                                        (int)k.size(1), (int)d, dtype_code(q.scalar_type()), &hq, &hk, &hv, causal,
                                        (float)scale, &ho, stream_of(q));
        });
        return done(status) ? THPVariable_Wrap(std::move(out)) : nullptr;
    });
}

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long at[7];
    PyObject *fail, *memory;
    if (!PyArg_ParseTuple(args, "OOKKKKKKK", &fail, &memory, at, at + 1, at + 2, at + 3, at + 4, at + 5, at + 6))
        return nullptr;
    abi.quantize_rows = (decltype(abi.quantize_rows))(uintptr_t)at[0];
    abi.matmul_workspace = (decltype(abi.matmul_workspace))(uintptr_t)at[1];
    abi.matmul = (decltype(abi.matmul))(uintptr_t)at[2];
    abi.linear_workspace = (decltype(abi.linear_workspace))(uintptr_t)at[3];
    abi.linear = (decltype(abi.linear))(uintptr_t)at[4];
    abi.moe_workspace = (decltype(abi.moe_workspace))(uintptr_t)at[5];
    abi.moe = (decltype(abi.moe))(uintptr_t)at[6];
    Py_INCREF(fail);
    Py_XSETREF(on_status, fail);
    Py_INCREF(memory);
    Py_XSETREF(out_of_memory, memory);
    Py_RETURN_NONE;
}

PyObject* bind_attention(PyObject*, PyObject* args) {
    unsigned long long at[5];
    if (!PyArg_ParseTuple(args, "KKKKK", at, at + 1, at + 2, at + 3, at + 4))
        return nullptr;
    abi.kv_append = (decltype(abi.kv_append))(uintptr_t)at[0];
    abi.kv_read = (decltype(abi.kv_read))(uintptr_t)at[1];
    abi.cache_workspace = (decltype(abi.cache_workspace))(uintptr_t)at[2];
    abi.attention_cache = (decltype(abi.attention_cache))(uintptr_t)at[3];
    abi.attention_prompt = (decltype(abi.attention_prompt))(uintptr_t)at[4];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
        {"bind", bind, METH_VARARGS, "bind(raises for a status, torch.OutOfMemoryError, addresses of the library's functions)"},
        {"bind_attention", bind_attention, METH_VARARGS, "bind_attention(addresses of the library's functions), behind bind"},
        {"quantize_rows_s8", (PyCFunction)(void*)quantize_rows_s8, METH_FASTCALL, "(x) -> (q, scales)"},
        {"matmul_s8_scaled", (PyCFunction)(void*)matmul_s8_scaled, METH_FASTCALL,
         "(a, b_packed, a_scales, b_scales, bias, dtype) -> c"},
        {"linear_s8", (PyCFunction)(void*)linear_s8, METH_FASTCALL, "(x, b_packed, b_scales, bias) -> y"},
        {"moe_s8", (PyCFunction)(void*)moe_s8, METH_FASTCALL,
         "(x, logits, w1, w1_scales, w2, w2_scales, top_k, renormalize) -> y"},
        {"kv_append_s8", (PyCFunction)(void*)kv_append_s8, METH_FASTCALL,
         "(cache.k, .v, .k_scales, .v_scales, block_table, lengths, k, v, q, cos, sin, cu_tokens, interleaved, turned_keys) "
         "-> (q, k)"},
        {"kv_read_s8", (PyCFunction)(void*)kv_read_s8, METH_FASTCALL,
         "(cache.k, .v, .k_scales, .v_scales, block_table, starts, cu_tokens, tokens, dtype) -> (k, v)"},
        {"attention_cache_s8", (PyCFunction)(void*)attention_cache_s8, METH_FASTCALL,
         "(q, cache.k, .v, .k_scales, .v_scales, block_table, lengths, scale, out) -> out"},
        {"attention_prompt", (PyCFunction)(void*)attention_prompt, METH_FASTCALL,
         "(q, k, v, cu_q, cu_k, causal, scale, out) -> out"},
        {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "made_for", MADE_FOR) < 0)
        Py_CLEAR(m);
    return m;
}

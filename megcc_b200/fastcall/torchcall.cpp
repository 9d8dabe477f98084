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

PyMethodDef methods[] = {
        {"bind", bind, METH_VARARGS, "bind(raises for a status, torch.OutOfMemoryError, addresses of the library's functions)"},
        {"quantize_rows_s8", (PyCFunction)(void*)quantize_rows_s8, METH_FASTCALL, "(x) -> (q, scales)"},
        {"matmul_s8_scaled", (PyCFunction)(void*)matmul_s8_scaled, METH_FASTCALL,
         "(a, b_packed, a_scales, b_scales, bias, dtype) -> c"},
        {"linear_s8", (PyCFunction)(void*)linear_s8, METH_FASTCALL, "(x, b_packed, b_scales, bias) -> y"},
        {"moe_s8", (PyCFunction)(void*)moe_s8, METH_FASTCALL,
         "(x, logits, w1, w1_scales, w2, w2_scales, top_k, renormalize) -> y"},
        {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "made_for", MADE_FOR) < 0)
        Py_CLEAR(m);
    return m;
}

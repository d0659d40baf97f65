// Python entry of the stand-alone operators: checks of the tensors, outputs and
// scratch from torch's allocator, the device and stream of the call, and the C
// ABI (include/sparsemoe_b200.h), whose functions bind() takes from the library
// that the package has loaded.
//
// Native because a decode step calls these with a few tokens: through ctypes a
// call cost the host 10.7 us (routing) and 15.6 us (a product in two launches),
// of which the launches themselves were 3.5 us each.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <cstdarg>

#include "../../include/sparsemoe_b200.h"

namespace {

decltype(&moe_route_experts) f_route;
decltype(&moe_int8_quantize_tokens) f_quantize;
decltype(&moe_int8_matmul) f_matmul;
decltype(&moe_int8_linear) f_linear;
decltype(&moe_int8_linear_scratch_bytes) f_linear_scratch;
decltype(&moe_int8_shared_expert) f_shared;
decltype(&moe_int8_shared_expert_scratch_bytes) f_shared_scratch;
PyObject* f_check;   // Python: raises for a status that is not MOE_OK

using at::Tensor;

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    va_list ap;
    va_start(ap, format);
    PyErr_FormatV(type, format, ap);
    va_end(ap);
    throw python_error();
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MOE_TYPE_F32;
        case at::kHalf: return MOE_TYPE_F16;
        case at::kBFloat16: return MOE_TYPE_BF16;
        default: return -1;
    }
}

const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}

struct Rows {
    int64_t n, cols, ld;
};
// Shape and row stride of a matrix whose rows are contiguous.
Rows rows_of(const Tensor& t, const char* name) {
    if (t.dim() != 2) refuse(PyExc_ValueError, "%s must be 2-D, got %d dimensions", name, (int)t.dim());
    Rows r{t.size(0), t.size(1), t.stride(0)};
    if (r.cols > 1 && t.stride(1) != 1) refuse(PyExc_ValueError, "%s: the elements of a row must be contiguous", name);
    if (r.ld < r.cols) {
        if (r.n > 1)
            refuse(PyExc_ValueError, "%s: rows overlap (stride %lld for %lld columns)", name, (long long)r.ld,
                                    (long long)r.cols);
        r.ld = r.cols;
    }
    return r;
}

const float* vector_of(PyObject* o, int64_t n, const char* name, at::Device dev) {
    if (o == Py_None) return nullptr;
    const Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1) ||
        t.device() != dev)
        refuse(PyExc_ValueError, "%s must be a contiguous f32 vector of %lld on cuda:%d", name, (long long)n, dev.index());
    return static_cast<const float*>(t.data_ptr());
}

Tensor fresh(at::IntArrayRef size, at::ScalarType type, at::Device dev) {
    return at::detail::empty_cuda(size, type, dev, std::nullopt);
}

// The int8 matrix [K, N] in the C ABI's terms.
MoeInt8Weight weight_of(PyObject* o, PyObject* scale, const char* name, int64_t K, at::Device dev, int64_t* N) {
    const Tensor& w = tensor(o, name);
    if (w.scalar_type() != at::kChar || w.dim() != 2 || w.size(0) != K || w.device() != dev)
        refuse(PyExc_ValueError, "%s must be int8 [K=%lld, N] on cuda:%d", name, (long long)K, dev.index());
    *N = w.size(1);
    const int64_t sk = w.stride(0), sn = w.stride(1);
    MoeInt8Weight r{static_cast<const int8_t*>(w.data_ptr()), 0, nullptr, MOE_WEIGHT_KN};
    // the stride of an axis of one element says nothing
    if (sn == 1 && (K == 1 || (sk % 16 == 0 && sk >= *N))) {
        r.row_stride = K > 1 ? sk : (*N + 15) / 16 * 16;
    } else if (sk == 1 && (*N == 1 || (sn % 16 == 0 && sn >= K))) {
        r.order = MOE_WEIGHT_NK;
        r.row_stride = *N > 1 ? sn : (K + 15) / 16 * 16;
    } else {
        refuse(PyExc_ValueError, 
            "%s: one axis must be contiguous and the other's stride a multiple of 16 bytes, got strides (%lld, %lld); "
            "int8_weight() lays a matrix out so",
            name, (long long)sk, (long long)sn);
    }
    r.scale = vector_of(scale, *N, "weight scales", dev);
    if (!r.scale) refuse(PyExc_ValueError, "%s needs its scales", name);
    return r;
}

// `out`, or a new tensor of `type`.
Tensor output_of(PyObject* o, int64_t n, int64_t cols, at::ScalarType type, at::Device dev, int* kind, int64_t* ld) {
    if (o == Py_None) {
        Tensor t = fresh({n, cols}, type, dev);
        *kind = type_of(t);
        *ld = cols;
        if (*kind < 0) refuse(PyExc_ValueError, "the output must be f32, f16 or bf16");
        return t;
    }
    const Tensor& t = tensor(o, "out");
    *kind = type_of(t);
    if (*kind < 0 || t.dim() != 2 || t.size(0) != n || t.size(1) != cols || t.device() != dev)
        refuse(PyExc_ValueError, "out must be f32, f16 or bf16 of shape (%lld, %lld) on cuda:%d", (long long)n,
                                (long long)cols, dev.index());
    *ld = rows_of(t, "out").ld;
    return t;
}

// The tensors' device as the current one, and torch's current stream there.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit On(at::Device dev) {
        if (c10::cuda::current_device() != dev.index()) guard.set_index(dev.index());
        stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    }
};

void check(int rc) {
    if (rc == MOE_OK) return;
    PyObject* r = PyObject_CallFunction(f_check, "i", rc);
    Py_XDECREF(r);
    throw python_error();
}

int as_int(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < INT_MIN || v > INT_MAX) refuse(PyExc_ValueError, "a number is out of range");
    return (int)v;
}
int to_int(int64_t v, const char* name) {
    if (v > INT_MAX) refuse(PyExc_ValueError, "%s: a dimension of %lld", name, (long long)v);
    return (int)v;
}

at::ScalarType dtype_of(PyObject* o, at::ScalarType none) {
    if (o == Py_None) return none;
    if (!THPDtype_Check(o)) refuse(PyExc_TypeError, "out_dtype must be a torch.dtype");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

void expect(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) refuse(PyExc_TypeError, "%d arguments for %d", (int)n, (int)want);
}

// route(logits, top_k, address of a MoeRouting, bias, out or None) -> (indices, weights)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    const Tensor& x = tensor(a[0], "logits");
    const int kind = type_of(x);
    if (kind < 0 || !x.is_cuda()) refuse(PyExc_ValueError, "logits must be f32, f16 or bf16 on a GPU");
    const at::Device dev = x.device();
    const Rows r = rows_of(x, "logits");
    const int k = as_int(a[1]), E = to_int(r.cols, "logits");
    const auto* spec = static_cast<const MoeRouting*>(PyLong_AsVoidPtr(a[2]));
    if (PyErr_Occurred()) throw python_error();
    const float* bias = vector_of(a[3], E, "bias", dev);
    Tensor idx, w;
    if (a[4] == Py_None) {
        const int64_t cols = k < 0 ? 0 : k;   // (a k out of range is refused below)
        idx = fresh({r.n, cols}, at::kInt, dev);
        w = fresh({r.n, cols}, at::kFloat, dev);
    } else {
        if (!PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 2)
            refuse(PyExc_TypeError, "out must be a tuple (indices, weights)");
        idx = tensor(PyTuple_GET_ITEM(a[4], 0), "out");
        w = tensor(PyTuple_GET_ITEM(a[4], 1), "out");
        auto fits = [&](const Tensor& t, at::ScalarType type) {
            return t.scalar_type() == type && t.dim() == 2 && t.size(0) == r.n && t.size(1) == k && t.is_contiguous() &&
                   t.device() == dev;
        };
        if (!fits(idx, at::kInt) || !fits(w, at::kFloat))
            refuse(PyExc_ValueError, "out must be contiguous int32 and f32 tensors of shape (%lld, %d) on cuda:%d",
                                    (long long)r.n, k, dev.index());
    }
    On on(dev);
    check(f_route(x.data_ptr(), kind, r.n, E, r.ld, k, spec, bias, static_cast<int*>(idx.data_ptr()),
                  static_cast<float*>(w.data_ptr()), on.stream));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw python_error();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(idx));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(w));
    return pair;
    END_HANDLE_TH_ERRORS
}

// quantize(x) -> (codes with rows on 16-byte boundaries, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 1);
    const Tensor& x = tensor(a[0], "x");
    const int kind = type_of(x);
    if (kind < 0 || !x.is_cuda()) refuse(PyExc_ValueError, "x must be f32, f16 or bf16 on a GPU");
    const at::Device dev = x.device();
    const Rows r = rows_of(x, "x");
    const int64_t kp = (r.cols + 15) / 16 * 16;
    Tensor q = fresh({r.n, kp}, at::kChar, dev), s = fresh({r.n}, at::kFloat, dev);
    On on(dev);
    check(f_quantize(x.data_ptr(), kind, r.n, to_int(r.cols, "x"), r.ld, static_cast<int8_t*>(q.data_ptr()), kp,
                     static_cast<float*>(s.data_ptr()), on.stream));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw python_error();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(q.narrow(1, 0, r.cols)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(s));
    return pair;
    END_HANDLE_TH_ERRORS
}

// matmul(q, scale, w, w_scale, bias, out_dtype, out)
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7);
    const Tensor& q = tensor(a[0], "q");
    if (q.scalar_type() != at::kChar || !q.is_cuda()) refuse(PyExc_ValueError, "q must be int8 on a GPU");
    const at::Device dev = q.device();
    Rows r = rows_of(q, "q");
    if (r.n <= 1) r.ld = (r.ld + 15) / 16 * 16;
    int64_t N;
    const MoeInt8Weight w = weight_of(a[2], a[3], "w", r.cols, dev, &N);
    const float* bias = vector_of(a[4], N, "bias", dev);
    const float* scale = vector_of(a[1], r.n, "scale", dev);
    int kind;
    int64_t ld;
    Tensor out = output_of(a[6], r.n, N, dtype_of(a[5], at::kBFloat16), dev, &kind, &ld);
    On on(dev);
    check(f_matmul(static_cast<const int8_t*>(q.data_ptr()), r.ld, scale, r.n, to_int(r.cols, "q"), &w, to_int(N, "w"),
                   bias, out.data_ptr(), kind, ld, on.stream));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// linear(x, w, w_scale, bias, out_dtype, out)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6);
    const Tensor& x = tensor(a[0], "x");
    const int xkind = type_of(x);
    if (xkind < 0 || !x.is_cuda()) refuse(PyExc_ValueError, "x must be f32, f16 or bf16 on a GPU");
    const at::Device dev = x.device();
    const Rows r = rows_of(x, "x");
    int64_t N;
    const MoeInt8Weight w = weight_of(a[1], a[2], "w", r.cols, dev, &N);
    const float* bias = vector_of(a[3], N, "bias", dev);
    int kind;
    int64_t ld;
    Tensor out = output_of(a[5], r.n, N, dtype_of(a[4], x.scalar_type()), dev, &kind, &ld);
    const int K = to_int(r.cols, "x");
    const size_t bytes = f_linear_scratch(r.n, K, N);
    Tensor scratch;
    if (bytes) scratch = fresh({(int64_t)bytes}, at::kByte, dev);
    On on(dev);
    check(f_linear(x.data_ptr(), xkind, r.n, K, r.ld, &w, to_int(N, "w"), bias, out.data_ptr(), kind, ld,
                   bytes ? scratch.data_ptr() : nullptr, bytes, on.stream));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// shared(x, w_gate, s_gate, w_up, s_up, w_down, s_down, residual, out)
PyObject* shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    const Tensor& x = tensor(a[0], "x");
    const int xkind = type_of(x);
    if (xkind < 0 || !x.is_cuda()) refuse(PyExc_ValueError, "x must be f32, f16 or bf16 on a GPU");
    const at::Device dev = x.device();
    const Rows r = rows_of(x, "x");
    int64_t f, fu, d;
    const MoeInt8Weight g = weight_of(a[1], a[2], "w_gate", r.cols, dev, &f);
    const MoeInt8Weight u = weight_of(a[3], a[4], "w_up", r.cols, dev, &fu);
    const MoeInt8Weight dn = weight_of(a[5], a[6], "w_down", f, dev, &d);
    if (fu != f || d != r.cols)
        refuse(PyExc_ValueError, "w_up must be [%lld, %lld] and w_down [%lld, %lld]", (long long)r.cols, (long long)f,
                                (long long)f, (long long)r.cols);
    const void* res = nullptr;
    int64_t ld_res = 0;
    if (a[7] != Py_None) {
        const Tensor& t = tensor(a[7], "residual");
        if (!t.sizes().equals(x.sizes()) || t.scalar_type() != x.scalar_type() || t.device() != dev)
            refuse(PyExc_ValueError, "residual must have x's shape, type and device");
        ld_res = rows_of(t, "residual").ld;
        res = t.data_ptr();
    }
    int kind;
    int64_t ld;
    Tensor out = output_of(a[8], r.n, d, x.scalar_type(), dev, &kind, &ld);
    const int di = to_int(d, "x"), fi = to_int(f, "w_gate");
    const size_t bytes = f_shared_scratch(r.n, di, fi);
    Tensor scratch = fresh({(int64_t)bytes}, at::kByte, dev);
    On on(dev);
    check(f_shared(x.data_ptr(), xkind, r.n, di, r.ld, &g, &u, &dn, fi, res, ld_res, out.data_ptr(), kind, ld,
                   scratch.data_ptr(), bytes, on.stream));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// bind(check, addresses of the library's functions in the order below)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject* chk;
    unsigned long long p[7];
    if (!PyArg_ParseTuple(args, "OKKKKKKK", &chk, &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6])) return nullptr;
    Py_INCREF(chk);
    Py_XDECREF(f_check);
    f_check = chk;
    f_route = reinterpret_cast<decltype(f_route)>(p[0]);
    f_quantize = reinterpret_cast<decltype(f_quantize)>(p[1]);
    f_matmul = reinterpret_cast<decltype(f_matmul)>(p[2]);
    f_linear = reinterpret_cast<decltype(f_linear)>(p[3]);
    f_linear_scratch = reinterpret_cast<decltype(f_linear_scratch)>(p[4]);
    f_shared = reinterpret_cast<decltype(f_shared)>(p[5]);
    f_shared_scratch = reinterpret_cast<decltype(f_shared_scratch)>(p[6]);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, {"route", FAST(route)},   {"quantize", FAST(quantize)},
                         {"matmul", FAST(matmul)},              {"linear", FAST(linear)}, {"shared", FAST(shared)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators(void) { return PyModule_Create(&module); }

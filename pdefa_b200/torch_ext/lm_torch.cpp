// Binding of the language-model operators for torch tensors: argument checks, output
// tensors, torch's current stream, and the call into the C ABI (whose addresses lm.py
// hands over, so this module is not linked against the engine).
//
// In Python those steps cost 8 to 11 us a call, more than most small calls take on the
// GPU; here they cost about 2.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/pdefa_b200_ext.h"

namespace {

constexpr int64_t kBlock = 128;

decltype(&engine_rms_norm_device) g_rms_norm = nullptr;
decltype(&engine_matmul_fp8_device) g_matmul = nullptr;
decltype(&engine_matmul_grouped_fp8_device) g_grouped = nullptr;
decltype(&engine_sample_device) g_sample = nullptr;
PyObject* g_error = nullptr;       // PdefaError
PyObject* g_check = nullptr;       // raises PdefaError for a status other than 0

struct Refused {
    PyObject* type;
    std::string what;
};
[[noreturn]] void type_error(const char* op, const std::string& m) { throw Refused{PyExc_TypeError, std::string(op) + ": " + m}; }
[[noreturn]] void refuse(const char* op, const std::string& m) { throw Refused{g_error, std::string(op) + ": " + m}; }

std::string text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}

const at::Tensor& tensor(PyObject* o, const char* op, const char* name) {
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
        type_error(op, std::string(name) + ": a CUDA torch.Tensor is needed");
    return THPVariable_Unpack(o);
}

// `t` is of `type`, has `dims` dimensions, the last of them dense, and is on GPU `device`.
void need(const at::Tensor& t, const char* op, const char* name, at::ScalarType type, int64_t dims, int device) {
    if (t.scalar_type() != type)
        type_error(op, std::string(name) + ": " + c10::toString(type) + " is needed, got " + c10::toString(t.scalar_type()));
    if (t.dim() != dims) refuse(op, std::string(name) + ": " + std::to_string(dims) + " dimensions are needed, got " + text(t.sizes()));
    if (t.get_device() != device) refuse(op, std::string(name) + ": is on another GPU");
    if (dims && t.size(-1) > 1 && t.stride(-1) != 1)
        refuse(op, std::string(name) + ": the last dimension has to be dense, strides are " + text(t.strides()));
}

int float_code(at::ScalarType t) {
    return t == at::kFloat ? ENGINE_F32 : t == at::kHalf ? ENGINE_F16 : t == at::kBFloat16 ? ENGINE_BF16 : -1;
}
int need_float(const at::Tensor& t, const char* op, const char* name) {
    const int code = float_code(t.scalar_type());
    if (code < 0)
        type_error(op, std::string(name) + " must be float32, float16 or bfloat16, got " + c10::toString(t.scalar_type()));
    return code;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// t as evenly spaced rows: their number, length and distance.
struct Rows {
    int64_t rows = 1, cols = 0, stride = 0;
};
Rows rows_of(const at::Tensor& t, const char* op, const char* name) {
    Rows r;
    const int64_t d = t.dim();
    r.cols = t.size(-1);
    for (int64_t i = 0; i + 1 < d; ++i) r.rows *= t.size(i);
    if (r.rows <= 1 || r.cols == 0) { r.stride = r.cols; return r; }
    int64_t i = d - 2;
    while (t.size(i) == 1) --i;                  // the innermost dimension of rows with more than one
    r.stride = t.stride(i);
    int64_t next = r.stride * t.size(i);
    for (--i; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (t.stride(i) != next)
            refuse(op, std::string(name) + ": rows of shape " + text(t.sizes()) + ", strides " + text(t.strides()) + " are not evenly spaced");
        next *= t.size(i);
    }
    return r;
}

PyObject* status(int rc, const char* op) {
    PyObject* r = PyObject_CallFunction(g_check, "is", rc, op);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(g_error, op);
    return nullptr;
}

// Runs a binding, with its refusals and torch's exceptions (allocation, ...) as Python's.
template <class F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.what.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// Calls a C entry point without the interpreter's lock. The arguments are made before: pointers
// of tensors without storage (fake ones, under tracing) and streams throw, which needs the lock.
template <class F, class... A>
int unlocked(F f, A... a) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = (int)f(a...);
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a, b, c, d;
    PyObject *error, *check;
    if (!PyArg_ParseTuple(args, "KKKKOO", &a, &b, &c, &d, &error, &check)) return nullptr;
    g_rms_norm = reinterpret_cast<decltype(g_rms_norm)>(a);
    g_matmul = reinterpret_cast<decltype(g_matmul)>(b);
    g_grouped = reinterpret_cast<decltype(g_grouped)>(c);
    g_sample = reinterpret_cast<decltype(g_sample)>(d);
    Py_INCREF(error);
    Py_INCREF(check);
    g_error = error;
    g_check = check;
    Py_RETURN_NONE;
}

// rms_norm(x, weight, residual, eps, fp8) -> y | (y, h) | (q, scales) | (q, scales, h)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 5) type_error("rms_norm", "5 arguments");
        const bool fp8 = args[4] == Py_True;
        const char* op = fp8 ? "ops_rms_norm_fp8" : "ops_rms_norm";
        const double eps = PyFloat_AsDouble(args[3]);
        if (eps == -1.0 && PyErr_Occurred()) return nullptr;
        const at::Tensor& x = tensor(args[0], op, "x");
        const int code = need_float(x, op, "x");
        const int device = x.get_device();
        if (x.dim() == 0) refuse(op, "x needs a dimension");
        need(x, op, "x", x.scalar_type(), x.dim(), device);
        const Rows rx = rows_of(x, op, "x");
        const at::Tensor& w = tensor(args[1], op, "weight");
        need(w, op, "weight", w.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type(), 1, device);
        if (w.size(0) != rx.cols) refuse(op, "weight of " + std::to_string(w.size(0)) + " for rows of " + std::to_string(rx.cols));
        at::Tensor h, y, scales;
        const at::Tensor* res = nullptr;
        Rows rr;
        if (args[2] != Py_None) {
            res = &tensor(args[2], op, "residual");
            if (res->sizes() != x.sizes()) refuse(op, "the residual needs x's shape " + text(x.sizes()));
            need(*res, op, "residual", x.scalar_type(), x.dim(), device);
            rr = rows_of(*res, op, "residual");
            h = at::empty(x.sizes(), x.options().requires_grad(false));
        }
        const int64_t nb = (rx.cols + kBlock - 1) / kBlock;
        if (fp8) {
            y = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));
            c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
            shape.back() = nb;
            scales = at::empty(shape, x.options().dtype(at::kFloat).requires_grad(false));
        } else {
            y = at::empty(x.sizes(), x.options().requires_grad(false));
        }
        if (rx.rows > 0 && rx.cols > 0) {
            const int rc = unlocked(g_rms_norm, x.const_data_ptr(), rx.stride, res ? res->const_data_ptr() : nullptr, rr.stride,
                                    w.const_data_ptr(), res ? h.mutable_data_ptr() : nullptr, rx.cols, y.mutable_data_ptr(), rx.cols,
                                    fp8 ? scales.mutable_data_ptr<float>() : nullptr, nb, rx.rows, rx.cols, code,
                                    float_code(w.scalar_type()), (float)eps, device, stream_of(device));
            if (rc) return status(rc, op);
        } else if (!(eps >= 0.0 && eps <= 3.4e38)) {
            refuse(op, "eps must be finite and >= 0");
        }
        if (fp8) return res ? Py_BuildValue("NNN", THPVariable_Wrap(y), THPVariable_Wrap(scales), THPVariable_Wrap(h))
                            : Py_BuildValue("NN", THPVariable_Wrap(y), THPVariable_Wrap(scales));
        return res ? Py_BuildValue("NN", THPVariable_Wrap(y), THPVariable_Wrap(h)) : THPVariable_Wrap(y);
    });
}

at::ScalarType out_type(PyObject* o, const char* op, int* code) {
    if (o == Py_None) { *code = ENGINE_BF16; return at::kBFloat16; }
    if (!THPDtype_Check(o)) type_error(op, "out_dtype must be a torch.dtype");
    const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
    *code = float_code(t);
    if (*code < 0) type_error(op, std::string("out_dtype must be float32, float16 or bfloat16, got ") + c10::toString(t));
    return t;
}

// matmul(a, a_scales, b, b_scales, out_dtype) and grouped(a, a_scales, b, b_scales, offsets, out_dtype)
template <bool GROUPED>
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* op = GROUPED ? "ops_matmul_grouped_fp8" : "ops_matmul_fp8";
        if (n != (GROUPED ? 6 : 5)) type_error(op, "wrong number of arguments");
        constexpr int64_t D = GROUPED ? 3 : 2;
        const at::Tensor& a = tensor(args[0], op, "a");
        const at::Tensor& sa = tensor(args[1], op, "a_scales");
        const at::Tensor& b = tensor(args[2], op, "b");
        const at::Tensor& sb = tensor(args[3], op, "b_scales");
        const int device = a.get_device();
        need(a, op, "a", at::kFloat8_e4m3fn, 2, device);
        need(b, op, "b", at::kFloat8_e4m3fn, D, device);
        need(sa, op, "a_scales", at::kFloat, 2, device);
        need(sb, op, "b_scales", at::kFloat, D, device);
        const int64_t m = a.size(0), k = a.size(1), nn = b.size(D - 2), kb = (k + kBlock - 1) / kBlock, nb = (nn + kBlock - 1) / kBlock;
        bool fits = b.size(D - 1) == k && sa.size(0) == m && sa.size(1) == kb && sb.size(D - 2) == nb && sb.size(D - 1) == kb;
        const at::Tensor* off = nullptr;
        const int64_t experts = GROUPED ? b.size(0) : 1;
        if (GROUPED) {
            off = &tensor(args[4], op, "offsets");
            need(*off, op, "offsets", at::kInt, 1, device);
            fits = fits && sb.size(0) == experts && off->size(0) == experts + 1;
        }
        if (!fits)
            refuse(op, "shapes do not fit: a " + text(a.sizes()) + ", a_scales " + text(sa.sizes()) + ", b " + text(b.sizes()) +
                           ", b_scales " + text(sb.sizes()) + (GROUPED ? ", offsets " + text(off->sizes()) : std::string()));
        int code = 0;
        const at::ScalarType type = out_type(args[GROUPED ? 5 : 4], op, &code);
        if (GROUPED && experts == 0) return THPVariable_Wrap(at::zeros({m, nn}, a.options().dtype(type)));
        at::Tensor out = at::empty({m, nn}, a.options().dtype(type).requires_grad(false));
        int rc;
        if constexpr (GROUPED)
            rc = unlocked(g_grouped, a.const_data_ptr(), a.stride(0), sa.const_data_ptr<float>(), sa.stride(0), b.const_data_ptr(),
                          b.stride(1), b.stride(0), sb.const_data_ptr<float>(), sb.stride(1), sb.stride(0),
                          off->const_data_ptr<int32_t>(), experts, out.mutable_data_ptr(), nn, code, m, nn, k, device, stream_of(device));
        else
            rc = unlocked(g_matmul, a.const_data_ptr(), a.stride(0), sa.const_data_ptr<float>(), sa.stride(0), b.const_data_ptr(),
                          b.stride(0), sb.const_data_ptr<float>(), sb.stride(0), out.mutable_data_ptr(), nn, code, m, nn, k, device,
                          stream_of(device));
        if (rc) return status(rc, op);
        return THPVariable_Wrap(std::move(out));
    });
}

// sample(logits, noise, temperature, top_k, top_p, min_p) -> (tokens, probs)
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* op = "ops_sample";
        if (n != 6) type_error(op, "6 arguments");
        const at::Tensor& x = tensor(args[0], op, "logits");
        const at::Tensor& e = tensor(args[1], op, "noise");
        const int code = need_float(x, op, "logits");
        const int device = x.get_device();
        need(x, op, "logits", x.scalar_type(), 2, device);
        need(e, op, "noise", at::kFloat, 2, device);
        if (e.sizes() != x.sizes()) refuse(op, "noise " + text(e.sizes()) + " for logits " + text(x.sizes()));
        const int64_t rows = x.size(0), vocab = x.size(1);
        static const char* const names[] = {"temperature", "top_k", "top_p", "min_p"};
        const void* per_row[4] = {};
        for (int i = 0; i < 4; ++i) {
            if (args[2 + i] == Py_None) continue;
            const at::Tensor& t = tensor(args[2 + i], op, names[i]);
            need(t, op, names[i], i == 1 ? at::kInt : at::kFloat, 1, device);
            if (t.size(0) != rows) refuse(op, std::string(names[i]) + " of " + std::to_string(t.size(0)) + " for " + std::to_string(rows) + " rows");
            per_row[i] = t.const_data_ptr();
        }
        at::Tensor tokens = at::empty({rows}, x.options().dtype(at::kInt).requires_grad(false));
        at::Tensor probs = at::empty({rows}, x.options().dtype(at::kFloat).requires_grad(false));
        const int rc = unlocked(g_sample, x.const_data_ptr(), x.stride(0), code, e.const_data_ptr<float>(), e.stride(0),
                                static_cast<const float*>(per_row[0]), static_cast<const int32_t*>(per_row[1]),
                                static_cast<const float*>(per_row[2]), static_cast<const float*>(per_row[3]), rows, vocab,
                                tokens.mutable_data_ptr<int32_t>(), probs.mutable_data_ptr<float>(), device, stream_of(device));
        if (rc) return status(rc, op);
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(tokens)), THPVariable_Wrap(std::move(probs)));
    });
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "C entry points, PdefaError and the status check."},
    {"rms_norm", FAST(rms_norm), ""},
    {"matmul", FAST(matmul<false>), ""},
    {"grouped", FAST(matmul<true>), ""},
    {"sample", FAST(sample), ""},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lm_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_lm_torch() { return PyModule_Create(&module); }

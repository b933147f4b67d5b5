// The W8A8 operators' front end for torch tensors: checks, output allocation, stream, call of the C entry (include/dynscaler_hip.h) -- in C++
// because a call on a few rows is over on the GPU before Python has gone through that (gemm_i8 of one token 8.8 us a call from Python,
// the kernel 4.3).  dynamicscaler_amd/ops.py holds the documented functions; the entries' addresses come from the library it has loaded.
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/ops/empty_cuda_dispatch.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <optional>
#include <string>
#include "../../include/dynscaler_hip.h"

namespace {

decltype(&ds_gemm_i8_workspace_bytes) c_gemm_workspace;
decltype(&ds_gemm_i8) c_gemm;
decltype(&ds_rmsnorm_rows) c_rmsnorm;
decltype(&ds_quantize_rows_i8) c_quantize;
decltype(&ds_dequantize_rows_i8) c_dequantize;
decltype(&ds_last_error) c_last_error;
PyObject *ds_error = nullptr, *out_of_memory = nullptr;

struct Refused { std::string says; };
struct Raised {};                      // a Python error is set

[[noreturn]] void refuse(const std::string& says) { throw Refused{says}; }

const char* name_of(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return "torch.float16";
        case at::kFloat: return "torch.float32";
        case at::kChar: return "torch.int8";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kDouble: return "torch.float64";
        default: return c10::toString(t);
    }
}

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

enum : unsigned { F16 = 1, F32 = 2, I8 = 4 };
unsigned kind(at::ScalarType t) { return t == at::kHalf ? F16 : t == at::kFloat ? F32 : t == at::kChar ? I8 : 0; }
int ds_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? DS_F16 : t.scalar_type() == at::kFloat ? DS_F32 : DS_I8; }

struct What { const char *op, *arg; std::string str() const { return std::string(op) + "(" + arg + ")"; } };

const at::Tensor& tensor(PyObject* o, What w) {
    if (!THPVariable_Check(o)) refuse(w.str() + ": is not a tensor");
    return THPVariable_Unpack(o);
}

struct Rows { int64_t m, n, ld; };

// a 2-D tensor with unit column stride and rows that do not overlap
Rows rows_of(const at::Tensor& t, What w, unsigned kinds, int64_t rows = -1, int64_t cols = -1) {
    if (!(kind(t.scalar_type()) & kinds))
        refuse(w.str() + ": " + name_of(t.scalar_type()) + " is not one of" + (kinds & F16 ? " torch.float16" : "") + (kinds & F32 ? " torch.float32" : "") + (kinds & I8 ? " torch.int8" : ""));
    if (t.dim() != 2) refuse(w.str() + ": has to be [rows, columns], got " + shape_of(t));
    const int64_t m = t.size(0), n = t.size(1), ld = t.stride(0), step = t.stride(1);
    if ((rows >= 0 && m != rows) || (cols >= 0 && n != cols))
        refuse(w.str() + ": is " + std::to_string(m) + " x " + std::to_string(n) + ", expected " + std::to_string(rows < 0 ? m : rows) + " x " + std::to_string(cols < 0 ? n : cols));
    if (m > INT32_MAX || n > INT32_MAX) refuse(w.str() + ": " + shape_of(t) + " is too large");
    if (n > 1 && step != 1) refuse(w.str() + ": the columns of a row have to be contiguous (strides " + std::to_string(ld) + ", " + std::to_string(step) + ")");
    if (m <= 1) return {m, n, n};
    if (ld < n) refuse(w.str() + ": rows overlap (row stride " + std::to_string(ld) + ", " + std::to_string(n) + " columns)");
    return {m, n, ld};
}

void vector_of(const at::Tensor& t, What w, int64_t n) {
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        refuse(w.str() + ": has to be a contiguous fp32 vector of " + std::to_string(n) + " values, got " + name_of(t.scalar_type()) + " " + shape_of(t));
}

at::ScalarType rows_type(PyObject* o, const char* what) {
    const bool is = THPDtype_Check(o);
    const at::ScalarType t = is ? reinterpret_cast<THPDtype*>(o)->scalar_type : at::kDouble;
    if (!(kind(t) & (F16 | F32))) refuse(std::string(what) + " " + (is ? name_of(t) : "given") + " is not torch.float16 or torch.float32");
    return t;
}

// The call's device is the first tensor's, the others have to be on it, and it has to be the current one.
struct Call {
    c10::Device dev;
    explicit Call(const at::Tensor& first) : dev(first.device()) {}
    void with(const at::Tensor& t) const {
        if (t.device() != dev) refuse("tensors on " + dev.str() + " and " + t.device().str() + " in one call");
    }
    void on_current_device() const {
        if (dev.type() != c10::DeviceType::CUDA) refuse("tensors are on " + dev.str() + "; the DynamicScaler hot path has no CPU fallback");
        const int now = c10::hip::current_device();
        if (dev.index() != now)
            refuse("tensors are on " + dev.str() + ", the current device is cuda:" + std::to_string(now) + ": call under torch.cuda.device(" + std::to_string(dev.index()) + ")");
    }
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType t) const {
        return at::cuda::empty(sizes, t, c10::kStrided, dev, c10::nullopt, c10::nullopt);
    }
};

// The stream of a call: the current one, or the one that the caller names by its handle.  A named stream is the current one while the call lasts, so
// what the call allocates (outputs, workspace) is that stream's, as under torch.cuda.stream(): the allocator hands a block of the stream that
// was current before to nobody else's kernels, and the other way round.
class Stream {
    std::optional<c10::hip::HIPStream> before;
    hipStream_t handle;
public:
    Stream(const Call& call, PyObject* given) {
        call.on_current_device();
        const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream(call.dev.index());
        handle = now.stream();
        if (given == Py_None) return;
        const uintptr_t named = reinterpret_cast<uintptr_t>(PyLong_AsVoidPtr(given));
        if (PyErr_Occurred()) throw Raised{};
        handle = reinterpret_cast<hipStream_t>(named);
        if (handle == now.stream()) return;
        before = now;                         // (1 is the default stream's other name; odd numbers mean pool streams to torch)
        c10::hip::setCurrentHIPStream(c10::hip::getStreamFromExternal(reinterpret_cast<hipStream_t>(named & 1 ? 0 : named), call.dev.index()));
    }
    ~Stream() {
        if (before) c10::hip::setCurrentHIPStream(*before);
    }
    Stream(const Stream&) = delete;
    Stream& operator=(const Stream&) = delete;
    operator void*() const { return handle; }
};

void done(int rc, const char* what) {
    if (rc != DS_OK) refuse(std::string(what) + " failed (code " + std::to_string(rc) + "): " + c_last_error());
}

// an output given by the caller is handed back as it is
PyObject* handed(PyObject* given, const at::Tensor& t) {
    if (given == Py_None) return THPVariable_Wrap(t);
    Py_INCREF(given);
    return given;
}

PyObject* tuple(std::initializer_list<PyObject*> items) {
    PyObject* r = PyTuple_New((Py_ssize_t)items.size());
    Py_ssize_t i = 0;
    for (PyObject* o : items) PyTuple_SET_ITEM(r, i++, o);
    return r;
}

long integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t expected, F&& f) {
    if (n != expected || !ds_error) {
        PyErr_SetString(PyExc_TypeError, ds_error ? "wrong number of arguments" : "bind() comes first");
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(ds_error, r.says.c_str());
    } catch (const Raised&) {
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(out_of_memory, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// A, W, a_scale, w_scale, bias, residual, out, out_dtype, epilogue, stream -> out
PyObject* gemm_i8(PyObject*, PyObject* const* arg, Py_ssize_t nargs) {
    return guarded(nargs, 10, [&]() -> PyObject* {
        const char* op = "gemm_i8";
        const at::Tensor &A = tensor(arg[0], {op, "A"}), &W = tensor(arg[1], {op, "W"}), &sa = tensor(arg[2], {op, "a_scale"}), &sw = tensor(arg[3], {op, "w_scale"});
        const Rows a = rows_of(A, {op, "A"}, I8), w = rows_of(W, {op, "W"}, I8, -1, a.n);
        vector_of(sa, {op, "a_scale"}, a.m);
        vector_of(sw, {op, "w_scale"}, w.m);
        const Call call(A);
        call.with(W);
        call.with(sa);
        call.with(sw);
        const float* bias = nullptr;
        if (arg[4] != Py_None) {
            const at::Tensor& b = tensor(arg[4], {op, "bias"});
            vector_of(b, {op, "bias"}, w.m);
            call.with(b);
            bias = static_cast<const float*>(b.const_data_ptr());
        }
        const long epilogue = integer(arg[8]);
        // (the types of `out` and `residual` set the other flags: a flag that says otherwise would write past a buffer)
        if (epilogue & ~(long)(DS_EPI_GEGLU | DS_EPI_SILU)) refuse("gemm_i8: epilogue " + std::to_string(epilogue) + " is not DS_EPI_GEGLU or DS_EPI_SILU");
        const int64_t cols = epilogue & DS_EPI_GEGLU ? w.m / 2 : w.m;
        ds_gemm_i8_desc d{};
        d.lda = a.ld; d.ldw = w.ld; d.M = (int)a.m; d.N = (int)w.m; d.K = (int)a.n;
        d.epilogue = (int)epilogue;
        const void* residual = nullptr;
        if (arg[5] != Py_None) {
            const at::Tensor& r = tensor(arg[5], {op, "residual"});
            d.ldr = rows_of(r, {op, "residual"}, F16 | F32, a.m, cols).ld;
            call.with(r);
            if (r.scalar_type() == at::kFloat) d.epilogue |= DS_EPI_RES_F32;
            residual = r.const_data_ptr();
        }
        at::Tensor out;
        if (arg[6] != Py_None) {
            out = tensor(arg[6], {op, "out"});
            d.ldc = rows_of(out, {op, "out"}, F16 | F32, a.m, cols).ld;
            call.with(out);
        }
        const at::ScalarType type = out.defined() ? out.scalar_type() : rows_type(arg[7], "gemm_i8: out_dtype");
        if (type == at::kFloat) d.epilogue |= DS_EPI_OUT_F32;
        const Stream st(call, arg[9]);
        if (!out.defined()) {
            out = call.empty({a.m, cols}, type);
            d.ldc = cols;
        }
        const int8_t *pa = static_cast<const int8_t*>(A.const_data_ptr()), *pw = static_cast<const int8_t*>(W.const_data_ptr());
        at::Tensor room;                       // back to the allocator with the call: the next block of the same stream
        const size_t bytes = c_gemm_workspace(pa, pw, &d);
        if (bytes) {
            try {
                room = call.empty({(int64_t)bytes}, at::kChar);
            } catch (const c10::OutOfMemoryError&) {      // slower without
            }
        }
        done(c_gemm(pa, pw, static_cast<const float*>(sa.const_data_ptr()), static_cast<const float*>(sw.const_data_ptr()), bias, residual, out.data_ptr(), &d,
                    room.defined() ? room.data_ptr() : nullptr, room.defined() ? bytes : 0, st), "ds_gemm_i8");
        return handed(arg[6], out);
    });
}

// name, 8-bit?, x, gamma, eps, residual, sum_out, out, out_dtype, scale, stream -> (out, scale | None, sum | None)
PyObject* rmsnorm(PyObject*, PyObject* const* arg, Py_ssize_t nargs) {
    return guarded(nargs, 11, [&]() -> PyObject* {
        const char* op = PyUnicode_AsUTF8(arg[0]);
        const double eps = PyFloat_AsDouble(arg[4]);
        if (!op || (eps == -1.0 && PyErr_Occurred())) throw Raised{};
        const bool i8 = arg[1] == Py_True;
        const at::Tensor &x = tensor(arg[2], {op, "x"}), &gamma = tensor(arg[3], {op, "gamma"});
        const Rows r = rows_of(x, {op, "x"}, F16 | F32);
        if (r.n < 1) refuse(std::string(op) + ": rows without values");
        vector_of(gamma, {op, "gamma"}, r.n);
        const Call call(x);
        call.with(gamma);
        ds_rmsnorm_desc d{};
        d.ldx = r.ld; d.rows = (int)r.m; d.C = (int)r.n; d.x_dtype = ds_type(x); d.eps = (float)eps;
        const at::Tensor *res = nullptr, *given_scale = nullptr;
        at::Tensor sum, y, scale;
        if (arg[5] != Py_None) {
            res = &tensor(arg[5], {op, "residual"});
            d.ldr = rows_of(*res, {op, "residual"}, F16 | F32, r.m, r.n).ld;
            d.r_dtype = ds_type(*res);
            call.with(*res);
            if (arg[6] != Py_None) {
                sum = tensor(arg[6], {op, "sum_out"});
                d.lds = rows_of(sum, {op, "sum_out"}, kind(res->scalar_type()), r.m, r.n).ld;
                call.with(sum);
            }
        } else if (arg[6] != Py_None) {
            refuse(std::string(op) + ": sum_out without a residual");
        }
        const at::ScalarType type = i8 ? at::kChar : rows_type(arg[8], "rmsnorm: out_dtype");
        if (arg[7] != Py_None) {
            y = tensor(arg[7], {op, "out"});
            d.ldy = rows_of(y, {op, "out"}, i8 ? I8 : F16 | F32, r.m, r.n).ld;
            call.with(y);
        }
        if (i8 && arg[9] != Py_None) {
            given_scale = &tensor(arg[9], {op, "scale"});
            vector_of(*given_scale, {op, "scale"}, r.m);
            call.with(*given_scale);
            scale = *given_scale;
        }
        const Stream st(call, arg[10]);
        if (res && !sum.defined()) {
            sum = call.empty({r.m, r.n}, res->scalar_type());
            d.lds = r.n;
        }
        if (!y.defined()) {
            y = call.empty({r.m, r.n}, type);
            d.ldy = r.n;
        }
        if (i8 && !scale.defined()) scale = call.empty({r.m}, at::kFloat);
        d.y_dtype = ds_type(y);
        done(c_rmsnorm(x.const_data_ptr(), res ? res->const_data_ptr() : nullptr, static_cast<const float*>(gamma.const_data_ptr()), res ? sum.data_ptr() : nullptr, y.data_ptr(),
                       i8 ? static_cast<float*>(scale.data_ptr()) : nullptr, &d, st), "ds_rmsnorm_rows");
        return tuple({handed(arg[7], y), i8 ? handed(arg[9], scale) : (Py_INCREF(Py_None), Py_None), res ? handed(arg[6], sum) : (Py_INCREF(Py_None), Py_None)});
    });
}

// x, out, scale, stream -> (out, scale)
PyObject* quantize_rows_i8(PyObject*, PyObject* const* arg, Py_ssize_t nargs) {
    return guarded(nargs, 4, [&]() -> PyObject* {
        const char* op = "quantize_rows_i8";
        const at::Tensor& x = tensor(arg[0], {op, "x"});
        const Rows r = rows_of(x, {op, "x"}, F16 | F32);
        if (r.n < 1) refuse("quantize_rows_i8: rows without values");
        const Call call(x);
        at::Tensor q, scale;
        int64_t ldq = r.n;
        if (arg[1] != Py_None) {
            q = tensor(arg[1], {op, "out"});
            ldq = rows_of(q, {op, "out"}, I8, r.m, r.n).ld;
            call.with(q);
        }
        if (arg[2] != Py_None) {
            scale = tensor(arg[2], {op, "scale"});
            vector_of(scale, {op, "scale"}, r.m);
            call.with(scale);
        }
        const Stream st(call, arg[3]);
        if (!q.defined()) q = call.empty({r.m, r.n}, at::kChar);
        if (!scale.defined()) scale = call.empty({r.m}, at::kFloat);
        done(c_quantize(x.const_data_ptr(), ds_type(x), r.ld, static_cast<int8_t*>(q.data_ptr()), ldq, static_cast<float*>(scale.data_ptr()), (int)r.m, (int)r.n, st), "ds_quantize_rows_i8");
        return tuple({handed(arg[1], q), handed(arg[2], scale)});
    });
}

// q, scale, out, dtype, stream -> out
PyObject* dequantize_rows_i8(PyObject*, PyObject* const* arg, Py_ssize_t nargs) {
    return guarded(nargs, 5, [&]() -> PyObject* {
        const char* op = "dequantize_rows_i8";
        const at::Tensor &q = tensor(arg[0], {op, "q"}), &scale = tensor(arg[1], {op, "scale"});
        const Rows r = rows_of(q, {op, "q"}, I8);
        if (r.n < 1) refuse("dequantize_rows_i8: rows without values");
        vector_of(scale, {op, "scale"}, r.m);
        const Call call(q);
        call.with(scale);
        at::Tensor y;
        int64_t ldy = r.n;
        if (arg[2] != Py_None) {
            y = tensor(arg[2], {op, "out"});
            ldy = rows_of(y, {op, "out"}, F16 | F32, r.m, r.n).ld;
            call.with(y);
        }
        const at::ScalarType type = y.defined() ? y.scalar_type() : rows_type(arg[3], "dequantize_rows_i8: dtype");
        const Stream st(call, arg[4]);
        if (!y.defined()) y = call.empty({r.m, r.n}, type);
        done(c_dequantize(static_cast<const int8_t*>(q.const_data_ptr()), r.ld, static_cast<const float*>(scale.const_data_ptr()), y.data_ptr(), ds_type(y), ldy, (int)r.m, (int)r.n, st),
             "ds_dequantize_rows_i8");
        return handed(arg[2], y);
    });
}

// the classes of refusals and of failed allocations, and the entries' addresses (gemm's workspace, gemm, rmsnorm, quantize, dequantize, last_error)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *cls, *oom;
    unsigned long long f[6];
    if (!PyArg_ParseTuple(args, "OOKKKKKK", &cls, &oom, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5])) return nullptr;
    c_gemm_workspace = reinterpret_cast<decltype(c_gemm_workspace)>(f[0]);
    c_gemm = reinterpret_cast<decltype(c_gemm)>(f[1]);
    c_rmsnorm = reinterpret_cast<decltype(c_rmsnorm)>(f[2]);
    c_quantize = reinterpret_cast<decltype(c_quantize)>(f[3]);
    c_dequantize = reinterpret_cast<decltype(c_dequantize)>(f[4]);
    c_last_error = reinterpret_cast<decltype(c_last_error)>(f[5]);
    Py_INCREF(cls);
    Py_INCREF(oom);
    Py_XDECREF(ds_error);
    Py_XDECREF(out_of_memory);
    ds_error = cls;
    out_of_memory = oom;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"gemm_i8", (PyCFunction)(void*)gemm_i8, METH_FASTCALL, nullptr},
                         {"rmsnorm", (PyCFunction)(void*)rmsnorm, METH_FASTCALL, nullptr},
                         {"quantize_rows_i8", (PyCFunction)(void*)quantize_rows_i8, METH_FASTCALL, nullptr},
                         {"dequantize_rows_i8", (PyCFunction)(void*)dequantize_rows_i8, METH_FASTCALL, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_w8a8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__w8a8(void) { return PyModule_Create(&module); }

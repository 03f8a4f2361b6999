// The layers' forward passes as the interpreter calls them.  The library itself (librptc_b200.so) knows no tensors; what lies
// between a module's `forward` and its entry points -- reading the module's attributes, checks, the result and the
// workspace, device and stream -- cost 12 us of Python and ctypes per call, as much as the kernels of a one-token pass.
// Functions return the result, or the rptc_status of the entry point as an int (the caller raises).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <optional>
#include <string>
#include <vector>

#include "../../include/rptc_b200.h"

namespace {

// Entry points of the library that the Python side has loaded.
struct {
    decltype(&rptc_linear_workspace_bytes) linear_workspace_bytes;
    decltype(&rptc_linear_forward) linear_forward;
    decltype(&rptc_packed_workspace_bytes) packed_workspace_bytes;
    decltype(&rptc_packed_forward) packed_forward;
    decltype(&rptc_gemv_timed) gemv_timed;
    decltype(&rptc_dequantize) dequantize;
    decltype(&rptc_decompress) decompress;
    decltype(&rptc_attn_prompt) attn_prompt;
    decltype(&rptc_qkv_append) qkv_append;
    decltype(&rptc_kv4_values) kv4_values;
    decltype(&rptc_attn_decode_kv4_workspace_bytes) attn_decode_kv4_workspace_bytes;
    decltype(&rptc_attn_decode_kv4) attn_decode_kv4;
    decltype(&rptc_token_logprobs) token_logprobs;
} g_lib;

#define RPTC_NAMES(X) X(in_features) X(out_features) X(block_in) X(block_out) X(scale) X(fmt) X(_buffers) X(codes) X(lut) X(carry_in) \
    X(signs_in) X(signs_out) X(num_banks) X(bank_blocks) X(L) X(alphabets) X(biases_out) X(biases_in) X(scales_out) X(scales_in) X(bias)
struct Names {
#define RPTC_FIELD(n) PyObject *n;
    RPTC_NAMES(RPTC_FIELD)
} g_names;

struct PyError : std::exception {};      // the interpreter's error is set
[[noreturn]] void fail(const char *what) {
    PyErr_SetString(PyExc_RuntimeError, what);
    throw PyError();
}

// A module's instance attributes and buffers, where they usually lie without the module's __getattr__; what lies elsewhere (a buffer
// that was replaced by a parameter, a property of a subclass) is asked of the module.
class Attributes {
public:
    explicit Attributes(PyObject *module) : module_(module), dict_(PyObject_GenericGetDict(module, nullptr)) {
        if (!dict_) throw PyError();
        buffers_ = get(dict_, g_names._buffers);
    }
    Attributes(const Attributes &) = delete;
    ~Attributes() {
        for (PyObject *o : owned_) Py_DECREF(o);
        Py_XDECREF(dict_);
    }
    PyObject *object(PyObject *name) { return get(dict_, name); }
    int64_t integer(PyObject *name) {
        const long long v = PyLong_AsLongLong(get(dict_, name));
        if (v == -1 && PyErr_Occurred()) throw PyError();
        return v;
    }
    double number(PyObject *name) {
        const double v = PyFloat_AsDouble(get(dict_, name));
        if (v == -1.0 && PyErr_Occurred()) throw PyError();
        return v;
    }
    // A buffer as a kernel reads it: `count` values of `type`, contiguous, and (device_with) on one GPU with the others; null for
    // None where the layer may do without.  (`.half()` and the like change buffers of a module, `.to()` may have been missed.)
    const void *pointer(PyObject *name, at::ScalarType type, int64_t count, bool optional = false) {
        PyObject *o = get(buffers_, name);
        if (o == Py_None && optional) return nullptr;
        if (!THPVariable_Check(o)) refuse(name, "must be a tensor");
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() != type) refuse(name, (std::string("must have dtype ") + c10::toString(type) + ", got " + c10::toString(t.scalar_type())).c_str());
        if (t.numel() != count) refuse(name, ("must have " + std::to_string(count) + " elements, got " + std::to_string(t.numel())).c_str());
        if (!t.is_contiguous()) refuse(name, "must be contiguous");
        if (held_n_ == sizeof(held_) / sizeof(held_[0])) fail("too many buffers");
        held_[held_n_++] = t;
        if (!device_) device_ = t.device();
        if (!elsewhere_ && (!t.is_cuda() || *device_ != t.device())) elsewhere_ = name;
        return t.data_ptr();
    }
    // The device of all buffers asked for; x has to be there too.
    c10::Device device_with(const at::Tensor &x) const {
        if (elsewhere_) refuse(elsewhere_, "must be a CUDA tensor on the GPU of the layer's other buffers");
        if (!x.is_cuda()) fail("x must be a CUDA tensor");
        if (x.device() != *device_) fail("x is on another GPU than the layer");
        return *device_;
    }

private:
    PyObject *get(PyObject *dict, PyObject *name) {
        PyObject *o = PyDict_GetItemWithError(dict, name);
        if (o) return o;
        if (!PyErr_Occurred()) o = PyObject_GetAttr(module_, name);
        if (!o) throw PyError();
        owned_.push_back(o);
        return o;
    }
    [[noreturn]] static void refuse(PyObject *name, const char *what) {
        const char *n = PyUnicode_AsUTF8(name);
        fail((std::string(n ? n : "a buffer") + " " + what).c_str());
    }
    PyObject *module_, *dict_, *buffers_ = nullptr, *elsewhere_ = nullptr;
    std::vector<PyObject *> owned_;
    at::Tensor held_[7];      // a launch lets other threads run, and they may give the module new buffers
    size_t held_n_ = 0;
    std::optional<c10::Device> device_;
};

const at::Tensor &unpack(PyObject *o, const char *what) {
    if (!THPVariable_Check(o)) fail(what);
    return THPVariable_Unpack(o);
}

rptc_format format_of(PyObject *structure) {      // the ctypes mirror of rptc_format
    rptc_format f;
    Py_buffer view;
    if (PyObject_GetBuffer(structure, &view, PyBUF_SIMPLE)) throw PyError();
    const bool fits = view.len == (Py_ssize_t)sizeof(f);
    if (fits) memcpy(&f, view.buf, sizeof(f));
    PyBuffer_Release(&view);
    if (!fits) fail("fmt is not a Format");
    return f;
}

// The activations as the kernels read them: contiguous, 16-byte aligned.
at::Tensor ready(const at::Tensor &x) {
    at::Tensor t = x.contiguous();
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) t = t.clone(at::MemoryFormat::Contiguous);
    return t;
}

at::Tensor result_like(const at::Tensor &x, int64_t columns) {
    at::DimVector shape(x.sizes());
    shape.back() = columns;
    return at::empty(shape, x.options().requires_grad(false));
}

template <typename F>
PyObject *guarded(F &&f) {
    try {
        return f();
    } catch (const PyError &) {
    } catch (...) {      // torch's own classes: out of memory is torch.OutOfMemoryError here too
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

cudaStream_t current_stream(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// linear_forward(module, x)
PyObject *linear_forward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 2) fail("linear_forward(module, x)");
        Attributes a(args[0]);
        const at::Tensor &x_in = unpack(args[1], "x must be a tensor");
        rptc_linear l;
        l.m = a.integer(g_names.out_features);
        l.n = a.integer(g_names.in_features);
        l.fmt = format_of(a.object(g_names.fmt));
        if (x_in.dim() < 1 || x_in.size(-1) != l.n || x_in.numel() == 0) fail("x must have in_features columns and at least one row");
        if (l.fmt.L < 1 || l.fmt.L > 16 || l.fmt.S < 0 || l.fmt.S > 16) fail("fmt has no such code");
        l.codes = a.pointer(g_names.codes, at::kInt, l.m * l.n * l.fmt.K / 32);
        l.lut = a.pointer(g_names.lut, at::kHalf, l.fmt.code == RPTC_CODE_LUT ? int64_t(1) << l.fmt.L : int64_t(2) << l.fmt.S);
        l.carry_in = static_cast<const uint32_t *>(a.pointer(g_names.carry_in, at::kInt, l.m, true));
        l.signs_in = a.pointer(g_names.signs_in, at::kHalf, l.n, true);
        l.signs_out = a.pointer(g_names.signs_out, at::kHalf, l.m, true);
        l.block_in = (int32_t)a.integer(g_names.block_in);
        l.block_out = (int32_t)a.integer(g_names.block_out);
        l.scale = (float)a.number(g_names.scale);
        const c10::cuda::OptionalCUDAGuard guard(a.device_with(x_in));
        const at::Tensor x = ready(x_in.scalar_type() == at::kHalf ? x_in : x_in.to(at::kHalf));
        const int64_t rows = x.numel() / l.n;
        at::Tensor y = result_like(x, l.m);
        const int64_t need = g_lib.linear_workspace_bytes(&l, rows);
        at::Tensor ws = at::empty({need > 0 ? need : 1}, x.options().dtype(at::kByte));
        const cudaStream_t s = current_stream(x);
        int status;
        Py_BEGIN_ALLOW_THREADS                                        // a launch waits where the stream's queue is full
        status = g_lib.linear_forward(&l, x.data_ptr(), y.data_ptr(), rows, ws.data_ptr(), need, s);
        Py_END_ALLOW_THREADS
        if (status != RPTC_OK) return PyLong_FromLong(status);
        // beyond 64 rows the product of a layer without transforms leaves the scale to be applied
        if (!l.signs_in && rows > 64 && l.scale != 1.f) y = y * a.number(g_names.scale);
        return THPVariable_Wrap(std::move(y));
    });
}

// packed_forward(module, x)
PyObject *packed_forward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 2) fail("packed_forward(module, x)");
        Attributes a(args[0]);
        const at::Tensor &x_in = unpack(args[1], "x must be a tensor");
        rptc_packed l;
        l.m = a.integer(g_names.out_features);
        l.n = a.integer(g_names.in_features);
        l.banks = (int32_t)a.integer(g_names.num_banks);
        l.bank_blocks = (int32_t)a.integer(g_names.bank_blocks);
        l.L = (int32_t)a.integer(g_names.L);
        if (x_in.dim() < 1 || x_in.size(-1) != l.n) fail("x must have in_features columns");
        if (l.L < 1 || l.L > 16) fail("L must be 1 to 16");
        l.codes = a.pointer(g_names.codes, at::kInt, (int64_t)l.banks * l.bank_blocks * 32 * l.n / 16);
        l.alphabets = a.pointer(g_names.alphabets, at::kHalf, (int64_t)l.banks << l.L);
        l.biases_out = static_cast<const float *>(a.pointer(g_names.biases_out, at::kFloat, l.m));
        l.biases_in = static_cast<const float *>(a.pointer(g_names.biases_in, at::kFloat, l.n));
        l.scales_out = static_cast<const float *>(a.pointer(g_names.scales_out, at::kFloat, l.m));
        l.scales_in = static_cast<const float *>(a.pointer(g_names.scales_in, at::kFloat, l.n));
        l.bias = static_cast<const float *>(a.pointer(g_names.bias, at::kFloat, l.m, true));
        const at::ScalarType type = x_in.scalar_type();
        const int dtype = type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : 2;
        const c10::cuda::OptionalCUDAGuard guard(a.device_with(x_in));
        const at::Tensor x = ready(dtype == 2 && type != at::kFloat ? x_in.to(at::kFloat) : x_in);
        at::Tensor y = result_like(x, l.m);
        const int64_t tokens = x.numel() / l.n;
        if (tokens > 0) {
            const int64_t most = tokens < 65535 ? tokens : 65535;      // tokens per native call
            const int64_t need = g_lib.packed_workspace_bytes(&l, most);
            if (need < 0) return PyLong_FromLong(RPTC_ERR_SHAPE);
            at::Tensor ws = at::empty({need}, x.options().dtype(at::kByte));
            const char *xp = static_cast<const char *>(x.data_ptr());
            char *yp = static_cast<char *>(y.data_ptr());
            const int64_t width = x.element_size();
            const cudaStream_t s = current_stream(x);
            int status = RPTC_OK;
            Py_BEGIN_ALLOW_THREADS
            for (int64_t t = 0; t < tokens && status == RPTC_OK; t += most)
                status = g_lib.packed_forward(&l, xp + t * l.n * width, dtype, yp + t * l.m * width, most < tokens - t ? most : tokens - t, ws.data_ptr(), need, s);
            Py_END_ALLOW_THREADS
            if (status != RPTC_OK) return PyLong_FromLong(status);
        }
        if (y.scalar_type() != type) y = y.to(type);
        return THPVariable_Wrap(std::move(y));
    });
}

// gemv_timed(codes, lut, x, acc, y, m, n, x_order, accumulate, fmt): milliseconds, or the status
PyObject *gemv_timed(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 10) fail("gemv_timed(codes, lut, x, acc, y, m, n, x_order, accumulate, fmt)");
        const at::Tensor *t[5];
        for (int i = 0; i < 5; ++i) t[i] = &unpack(args[i], "expected a tensor");
        long long v[4];
        for (int i = 0; i < 4; ++i) {
            v[i] = PyLong_AsLongLong(args[5 + i]);
            if (v[i] == -1 && PyErr_Occurred()) throw PyError();
        }
        const rptc_format fmt = format_of(args[9]);
        const c10::cuda::OptionalCUDAGuard guard(t[4]->device());
        const cudaStream_t s = current_stream(*t[4]);
        float ms = 0.f;
        int status;
        Py_BEGIN_ALLOW_THREADS                                        // waits for the result
        status = g_lib.gemv_timed(t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), static_cast<float *>(t[3]->data_ptr()), t[4]->data_ptr(),
                                  v[0], v[1], (int)v[2], (int)v[3], &fmt, &ms, s);
        Py_END_ALLOW_THREADS
        return status == RPTC_OK ? PyFloat_FromDouble(ms) : PyLong_FromLong(status);
    });
}

bool plain(const at::Tensor &t, at::ScalarType type) { return t.is_cuda() && t.scalar_type() == type && t.is_contiguous(); }

// dequantize(alphabet, symbols): symbols to weights, or None for what is not as the kernel reads it (the caller converts it, or refuses it)
PyObject *dequantize(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 2) fail("dequantize(alphabet, symbols)");
        if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
        const at::Tensor &alphabet = THPVariable_Unpack(args[0]), &symbols = THPVariable_Unpack(args[1]);
        const bool f32 = alphabet.scalar_type() == at::kFloat;
        const int64_t entries = alphabet.numel(), dims = symbols.dim();
        if (!plain(alphabet, f32 ? at::kFloat : at::kHalf) || !plain(symbols, at::kInt) || alphabet.device() != symbols.device() || alphabet.dim() != 1 ||
            entries < 8 || entries > 65536 || (entries & (entries - 1)) || dims < 1 || dims > 2 || symbols.numel() == 0)
            Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(symbols.device());
        at::Tensor out = at::empty(symbols.sizes(), alphabet.options().requires_grad(false));
        int L = 0;
        while ((int64_t(1) << L) < entries) ++L;
        const cudaStream_t s = current_stream(symbols);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.dequantize(alphabet.data_ptr(), static_cast<const int32_t *>(symbols.data_ptr()), out.data_ptr(), f32, dims == 2 ? symbols.size(0) : 1,
                                  symbols.size(-1), L, s);
        Py_END_ALLOW_THREADS
        return status == RPTC_OK ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(status);
    });
}

// decompress(codes, lut, m, n, fmt, out): 0 when done, None for what is not as the kernel reads it (the caller refuses it)
PyObject *decompress(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 6) fail("decompress(codes, lut, m, n, fmt, out)");
        if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[5])) Py_RETURN_NONE;
        const at::Tensor &codes = THPVariable_Unpack(args[0]), &lut = THPVariable_Unpack(args[1]), &out = THPVariable_Unpack(args[5]);
        const long long m = PyLong_AsLongLong(args[2]), n = PyLong_AsLongLong(args[3]);
        if (PyErr_Occurred()) throw PyError();
        const rptc_format fmt = format_of(args[4]);
        if (fmt.L < 1 || fmt.L > 16 || fmt.S < 0 || fmt.S > 16 || m <= 0 || n <= 0 || m > (1 << 30) || n > (1 << 30)) Py_RETURN_NONE;
        if (!plain(codes, at::kInt) || !plain(lut, at::kHalf) || codes.device() != lut.device() || codes.device() != out.device() ||
            lut.numel() != (fmt.code == RPTC_CODE_LUT ? int64_t(1) << fmt.L : int64_t(2) << fmt.S) || codes.numel() * 32 != m * n * fmt.K ||
            out.scalar_type() != at::kHalf || out.dim() != 2 || out.size(0) != m || out.size(1) != n || out.stride(1) != 1)
            Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(codes.device());
        const cudaStream_t s = current_stream(codes);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.decompress(codes.data_ptr(), lut.data_ptr(), nullptr, out.data_ptr(), out.stride(0), m, n, &fmt, s);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(status);
    });
}

// ---- the serving operators.  None for what is not as the kernels read it: the caller refuses it, and says why. ----
const at::Tensor *tensor_or_null(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
// A tensor on `device` of `type`, contiguous in `shape`.
bool is(const at::Tensor *t, c10::Device device, at::ScalarType type, at::IntArrayRef shape) {
    return t && t->device() == device && t->scalar_type() == type && t->sizes() == shape && t->is_contiguous();
}
// Rows of at least `width` values with unit column stride; `ld` what is between them.
bool is_rows(const at::Tensor *t, c10::Device device, int64_t rows, int64_t width, int64_t &ld) {
    if (!t || t->device() != device || t->dim() != 2 || t->size(0) != rows || t->size(1) < width || (t->stride(1) != 1 && t->size(1) > 1)) return false;
    ld = rows > 1 ? t->stride(0) : std::max(t->size(1), t->stride(0));
    return true;
}
bool whole(PyObject *o, int64_t &v) {
    if (!PyLong_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyError();
    return true;
}
bool number(PyObject *o, double none, float &v) {
    const double d = o == Py_None ? none : PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) throw PyError();
    v = (float)d;
    return true;
}
// (k, v) in fp16, or (k codes, k scales, v codes, v scales).
bool cache_of(PyObject *o, rptc_kv_cache &c, const at::Tensor *(&t)[4]) {
    if (!PyTuple_Check(o)) return false;
    const Py_ssize_t n = PyTuple_GET_SIZE(o);
    if (n != 2 && n != 4) return false;
    for (Py_ssize_t i = 0; i < n; ++i)
        if (!(t[i] = tensor_or_null(PyTuple_GET_ITEM(o, i)))) return false;
    const at::Tensor &k = *t[0];
    if (!k.is_cuda() || k.dim() != 4 || k.numel() == 0) return false;
    if (n == 2) {
        if (k.size(3) != 128 || !is(t[0], k.device(), at::kHalf, k.sizes()) || !is(t[1], k.device(), at::kHalf, k.sizes())) return false;
        c = {t[0]->data_ptr(), nullptr, t[1]->data_ptr(), nullptr, k.size(0), k.size(1), (int32_t)k.size(2), 16};
        return true;
    }
    const int64_t shape[5] = {k.size(0), k.size(1), k.size(2), 4, 2};
    if (k.size(3) != 64) return false;
    for (int i = 0; i < 4; ++i)
        if (i % 2 ? !is(t[i], k.device(), at::kHalf, at::IntArrayRef(shape, 5)) : !is(t[i], k.device(), at::kByte, k.sizes())) return false;
    c = {t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), t[3]->data_ptr(), k.size(0), k.size(2), (int32_t)k.size(1), 4};
    return true;
}

// attn_prompt(q, k, v, starts, kv_first, kv_len, out, scale)
PyObject *attn_prompt(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 8) fail("attn_prompt(q, k, v, starts, kv_first, kv_len, out, scale)");
        const at::Tensor *q = tensor_or_null(args[0]), *k = tensor_or_null(args[1]), *v = tensor_or_null(args[2]), *starts = tensor_or_null(args[3]);
        if (!q || !k || !v || !starts || !q->is_cuda() || q->dim() != 3 || k->dim() != 3 || v->sizes() != k->sizes() || k->size(2) != q->size(2) ||
            q->size(0) == 0 || k->size(0) == 0 || q->stride(2) != 1 || k->stride(2) != 1 || v->stride(2) != 1)
            Py_RETURN_NONE;
        const at::ScalarType type = q->scalar_type();
        const c10::Device device = q->device();
        if ((type != at::kHalf && type != at::kBFloat16) || k->scalar_type() != type || v->scalar_type() != type || k->device() != device || v->device() != device) Py_RETURN_NONE;
        if (starts->dim() != 1 || starts->size(0) < 2 || !is(starts, device, at::kInt, starts->sizes())) Py_RETURN_NONE;
        rptc_prompt_attention a = {};
        a.sequences = starts->size(0) - 1;
        a.starts = static_cast<const int32_t *>(starts->data_ptr());
        if ((args[4] == Py_None) != (args[5] == Py_None)) Py_RETURN_NONE;
        if (args[4] != Py_None) {
            const at::Tensor *first = tensor_or_null(args[4]), *count = tensor_or_null(args[5]);
            if (!is(first, device, at::kInt, {a.sequences}) || !is(count, device, at::kInt, {a.sequences})) Py_RETURN_NONE;
            a.kv_first = static_cast<const int32_t *>(first->data_ptr()), a.kv_len = static_cast<const int32_t *>(count->data_ptr());
        }
        const at::Tensor *given = args[6] == Py_None ? nullptr : tensor_or_null(args[6]);
        if (args[6] != Py_None && (!given || given->device() != device || given->scalar_type() != type || given->sizes() != q->sizes() || given->stride(2) != 1)) Py_RETURN_NONE;
        a.tokens = q->size(0), a.kv_tokens = k->size(0), a.heads = (int32_t)q->size(1), a.kv_heads = (int32_t)k->size(1), a.d = (int32_t)q->size(2);
        a.dtype = type == at::kBFloat16;
        if (!number(args[7], 1.0 / std::sqrt((double)std::max(a.d, 1)), a.scale)) Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor out = given ? *given : at::empty(q->sizes(), at::TensorOptions().dtype(type).device(device));
        const auto strides = [&](const at::Tensor &t, int64_t &row, int64_t &head) {      // of an axis of one element any
            row = t.size(0) > 1 ? t.stride(0) : t.size(1) * a.d, head = t.size(1) > 1 ? t.stride(1) : a.d;
        };
        strides(*q, a.q_row, a.q_head), strides(*k, a.k_row, a.k_head), strides(*v, a.v_row, a.v_head), strides(out, a.out_row, a.out_head);
        a.q = q->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr(), a.out = out.data_ptr();
        const cudaStream_t s = current_stream(*q);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.attn_prompt(&a, s);
        Py_END_ALLOW_THREADS
        return status == RPTC_OK ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(status);
    });
}

// qkv_append(x, pos, angles, cache, heads, kv_heads, slots, signs_out, scale, transform, out, clear)
PyObject *qkv_append(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 12) fail("qkv_append(x, pos, angles, cache, heads, kv_heads, slots, signs_out, scale, transform, out, clear)");
        rptc_append a = {};
        const at::Tensor *held[4], *x = tensor_or_null(args[0]), *angles = tensor_or_null(args[2]);
        int64_t heads, kv_heads;
        if (!x || !x->is_cuda() || x->dim() != 2 || x->size(0) == 0 || !cache_of(args[3], a.cache, held) || !whole(args[4], heads) || !whole(args[5], kv_heads)) Py_RETURN_NONE;
        const c10::Device device = x->device();
        if (held[0]->device() != device || heads <= 0 || heads > 4096 || kv_heads != a.cache.kv_heads) Py_RETURN_NONE;
        const int64_t width = (heads + 2 * kv_heads) * 128;
        a.tokens = x->size(0), a.heads = (int32_t)heads;
        a.x_is_f32 = x->scalar_type() == at::kFloat;
        if ((!a.x_is_f32 && x->scalar_type() != at::kHalf) || !is_rows(x, device, a.tokens, width, a.ld_x)) Py_RETURN_NONE;
        const at::Tensor *pos = tensor_or_null(args[1]);
        if (!is(pos, device, at::kInt, {a.tokens}) || !angles || angles->dim() != 3 || angles->size(0) < a.cache.max_pos ||
            !is(angles, device, at::kFloat, {angles->size(0), 64, 2}))
            Py_RETURN_NONE;
        a.pos = static_cast<const int32_t *>(pos->data_ptr()), a.angles = static_cast<const float *>(angles->data_ptr());
        if (args[6] != Py_None) {
            const at::Tensor *slots = tensor_or_null(args[6]);
            if (!is(slots, device, at::kInt, {a.tokens})) Py_RETURN_NONE;
            a.slots = static_cast<const int32_t *>(slots->data_ptr());
        }
        if (args[7] != Py_None) {
            const at::Tensor *signs = tensor_or_null(args[7]);
            if (!is(signs, device, at::kHalf, {width})) Py_RETURN_NONE;
            a.signs_out = signs->data_ptr();
        }
        if (!number(args[8], 1.0, a.scale)) Py_RETURN_NONE;
        const int transform = PyObject_IsTrue(args[9]), clear = PyObject_IsTrue(args[11]);
        if (transform < 0 || clear < 0) throw PyError();
        a.transform = transform, a.clear = clear;
        const at::Tensor *given = args[10] == Py_None ? nullptr : tensor_or_null(args[10]);
        if (args[10] != Py_None && (!given || given->scalar_type() != at::kHalf || !is_rows(given, device, a.tokens, heads * 128, a.ld_out))) Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor out = given ? *given : at::empty({a.tokens, width}, at::TensorOptions().dtype(at::kHalf).device(device));
        if (!given) a.ld_out = width;
        a.out_kv = out.size(1) >= width;
        a.x = x->data_ptr(), a.out = out.data_ptr();
        const cudaStream_t s = current_stream(*x);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.qkv_append(&a, s);
        Py_END_ALLOW_THREADS
        return status == RPTC_OK ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(status);
    });
}

// kv4_values(cache, count, out): (k, v)
PyObject *kv4_values(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 3) fail("kv4_values(cache, count, out)");
        rptc_kv_cache c;
        const at::Tensor *held[4], *count = tensor_or_null(args[1]);
        if (!cache_of(args[0], c, held) || c.bits != 4) Py_RETURN_NONE;
        const c10::Device device = held[0]->device();
        if (!is(count, device, at::kInt, {c.rows})) Py_RETURN_NONE;
        const int64_t shape[4] = {c.rows, c.max_pos, c.kv_heads, 128};
        at::Tensor out[2];
        const c10::cuda::OptionalCUDAGuard guard(device);
        for (int i = 0; i < 2; ++i) {
            if (args[2] == Py_None) {
                out[i] = at::empty(at::IntArrayRef(shape, 4), at::TensorOptions().dtype(at::kHalf).device(device));
            } else {
                if (!PyTuple_Check(args[2]) || PyTuple_GET_SIZE(args[2]) != 2) Py_RETURN_NONE;
                const at::Tensor *t = tensor_or_null(PyTuple_GET_ITEM(args[2], i));
                if (!is(t, device, at::kHalf, at::IntArrayRef(shape, 4))) Py_RETURN_NONE;
                out[i] = *t;
            }
        }
        const cudaStream_t s = current_stream(*held[0]);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.kv4_values(&c, static_cast<const int32_t *>(count->data_ptr()), out[0].data_ptr(), out[1].data_ptr(), s);
        Py_END_ALLOW_THREADS
        if (status != RPTC_OK) return PyLong_FromLong(status);
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])));
    });
}

// attn_decode_kv4(q, pos, cache, heads, out, scale, signs_in)
PyObject *attn_decode_kv4(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 7) fail("attn_decode_kv4(q, pos, cache, heads, out, scale, signs_in)");
        rptc_kv_cache c;
        const at::Tensor *held[4], *q = tensor_or_null(args[0]), *pos = tensor_or_null(args[1]);
        int64_t heads, ld_q, ld_out = 0;
        if (!cache_of(args[2], c, held) || c.bits != 4 || !whole(args[3], heads) || heads <= 0 || heads > 4096) Py_RETURN_NONE;
        const c10::Device device = held[0]->device();
        if (!is_rows(q, device, c.rows, heads * 128, ld_q) || q->scalar_type() != at::kHalf || !is(pos, device, at::kInt, {c.rows})) Py_RETURN_NONE;
        const at::Tensor *given = args[4] == Py_None ? nullptr : tensor_or_null(args[4]), *signs = args[6] == Py_None ? nullptr : tensor_or_null(args[6]);
        if (args[4] != Py_None && (!given || given->scalar_type() != at::kHalf || !is_rows(given, device, c.rows, heads * 128, ld_out))) Py_RETURN_NONE;
        if (args[6] != Py_None && !is(signs, device, at::kHalf, {heads * 128})) Py_RETURN_NONE;
        float scale;
        if (!number(args[5], 0.08838834764831845, scale)) Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor out = given ? *given : at::empty({c.rows, heads * 128}, at::TensorOptions().dtype(at::kHalf).device(device));
        if (!given) ld_out = heads * 128;
        const int64_t need = g_lib.attn_decode_kv4_workspace_bytes(&c, (int)heads);
        at::Tensor ws;
        if (need > 0) ws = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(device));
        const cudaStream_t s = current_stream(*q);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.attn_decode_kv4(q->data_ptr(), ld_q, static_cast<const int32_t *>(pos->data_ptr()), &c, out.data_ptr(), ld_out, (int)heads, scale,
                                       signs ? signs->data_ptr() : nullptr, need > 0 ? ws.data_ptr() : nullptr, need, s);
        Py_END_ALLOW_THREADS
        return status == RPTC_OK ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(status);
    });
}

// token_logprobs(logits, targets, top): (logprob or None, entropy, top_logprobs, top_ids)
PyObject *token_logprobs(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 3) fail("token_logprobs(logits, targets, top)");
        const at::Tensor *x = tensor_or_null(args[0]), *targets = args[1] == Py_None ? nullptr : tensor_or_null(args[1]);
        int64_t top, ld;
        if (!x || !x->is_cuda() || x->dim() != 2 || x->size(0) == 0 || x->size(1) == 0 || !whole(args[2], top)) Py_RETURN_NONE;
        const c10::Device device = x->device();
        const int64_t rows = x->size(0), n = x->size(1);
        const at::ScalarType type = x->scalar_type();
        const int dtype = type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : type == at::kFloat ? 2 : -1;
        if (dtype < 0 || top < 0 || top > 32 || top > n || !is_rows(x, device, rows, n, ld) || (args[1] != Py_None && !is(targets, device, at::kLong, {rows}))) Py_RETURN_NONE;
        const c10::cuda::OptionalCUDAGuard guard(device);
        const auto f32 = at::TensorOptions().dtype(at::kFloat).device(device);
        at::Tensor logprob, entropy = at::empty({rows}, f32), best = at::empty({rows, top}, f32), ids = at::empty({rows, top}, f32.dtype(at::kLong));
        if (targets) logprob = at::empty({rows}, f32);
        const cudaStream_t s = current_stream(*x);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_lib.token_logprobs(x->data_ptr(), dtype, ld, targets ? static_cast<const int64_t *>(targets->data_ptr()) : nullptr,
                                      targets ? static_cast<float *>(logprob.data_ptr()) : nullptr, static_cast<float *>(entropy.data_ptr()),
                                      top ? static_cast<float *>(best.data_ptr()) : nullptr, top ? static_cast<int64_t *>(ids.data_ptr()) : nullptr, rows, n, (int)top, s);
        Py_END_ALLOW_THREADS
        if (status != RPTC_OK) return PyLong_FromLong(status);
        PyObject *first = targets ? THPVariable_Wrap(std::move(logprob)) : Py_NewRef(Py_None);
        return Py_BuildValue("(NNNN)", first, THPVariable_Wrap(std::move(entropy)), THPVariable_Wrap(std::move(best)), THPVariable_Wrap(std::move(ids)));
    });
}

// bind(addresses of the entry points, in the order of g_lib)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        constexpr Py_ssize_t kEntries = sizeof(g_lib) / sizeof(void *);
        if (nargs != kEntries) fail("bind(an address per entry point)");
        void *p[kEntries];
        for (Py_ssize_t i = 0; i < kEntries; ++i) {
            p[i] = PyLong_AsVoidPtr(args[i]);
            if (!p[i]) {
                if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "null address");
                throw PyError();
            }
        }
        static_assert(sizeof(g_lib) == sizeof(p), "addresses alone");
        memcpy(&g_lib, p, sizeof(p));
        Py_RETURN_NONE;
    });
}

#define RPTC_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {RPTC_METHOD(bind), RPTC_METHOD(linear_forward), RPTC_METHOD(packed_forward), RPTC_METHOD(gemv_timed),
                           RPTC_METHOD(dequantize), RPTC_METHOD(decompress), RPTC_METHOD(attn_prompt), RPTC_METHOD(qkv_append), RPTC_METHOD(kv4_values),
                           RPTC_METHOD(attn_decode_kv4), RPTC_METHOD(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
#define RPTC_INTERN(n) \
    g_names.n = PyUnicode_InternFromString(#n); \
    if (!g_names.n) return nullptr;
    RPTC_NAMES(RPTC_INTERN)
    return PyModule_Create(&g_module);
}

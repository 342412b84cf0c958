// torch_shim.cpp - the Python layer's checks and argument structures for the
// layer ops (layer_ops.py), in C++.
//
// A single-token call runs for a few microseconds on the GPU; checking a dozen
// tensors and filling a ctypes structure in Python took 17-27 us a call. This
// module reads the tensors directly, keeps every check and message on the host
// side of the C ABI (include/fds_b200.h), allocates what the caller did not
// give, and calls the ABI's entry points by the addresses that Python loaded.
// It holds no state but those, the error class and, per device, the two status
// words.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <sstream>
#include <string>

#include "fds_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

PyObject* g_error = nullptr;         // FdsError
PyObject* g_status = nullptr;        // device index -> (status word, mirror word) addresses
PyObject* g_raise_timeout = nullptr; // device index: raises with the recorded bits
using LastError = const char* (*)();
LastError g_last_error = nullptr;
int (*g_linear_int8)(const FdsLinearInt8Args*, void*) = nullptr;
int (*g_residual_norm)(const FdsResidualNormArgs*, void*) = nullptr;
int (*g_window)(const FdsWindowArgs*, void*) = nullptr;

struct Refused {
    std::string what;
};
struct PythonError {};  // the Python error indicator is set

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw Refused{s.str()};
}
// the message is only built on failure
#define FDS_REQUIRE(cond, ...)                                     \
    do {                                                           \
        if (__builtin_expect(!(cond), 0)) refuse(__VA_ARGS__);     \
    } while (0)

std::string shape_of(const Tensor& t) {
    std::ostringstream s;
    s << '(';
    for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
    s << ')';
    return s.str();
}

const char* name_of(ScalarType t) {
    switch (t) {
        case ScalarType::Half: return "torch.float16";
        case ScalarType::BFloat16: return "torch.bfloat16";
        case ScalarType::Float: return "torch.float32";
        case ScalarType::Char: return "torch.int8";
        case ScalarType::Int: return "torch.int32";
        default: return c10::toString(t);
    }
}

bool is16(ScalarType t) { return t == ScalarType::Half || t == ScalarType::BFloat16; }
int dtype_code(ScalarType t) { return t == ScalarType::Half ? FDS_DTYPE_FP16 : FDS_DTYPE_BF16; }

// A tensor argument, or null for None.
const Tensor* optional(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    FDS_REQUIRE(THPVariable_Check(o), name, " must be a torch.Tensor");
    return &THPVariable_Unpack(o);
}
const Tensor& required(PyObject* o, const char* name) {
    FDS_REQUIRE(THPVariable_Check(o), name, " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw PythonError{};
        PyErr_Clear();
        refuse(name, " is out of range");
    }
    return v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
}
// None, torch.float16 or torch.bfloat16
ScalarType dtype_or(PyObject* o, ScalarType otherwise) {
    ScalarType t = otherwise;
    if (o != Py_None) {
        FDS_REQUIRE(THPDtype_Check(o), "dtype must be a torch.dtype");
        t = reinterpret_cast<THPDtype*>(o)->scalar_type;
    }
    FDS_REQUIRE(is16(t), "dtype must be torch.float16 or torch.bfloat16, got ", name_of(t));
    return t;
}

void type_is(const Tensor& t, const char* name, ScalarType a) {
    FDS_REQUIRE(t.scalar_type() == a, name, " must be ", name_of(a), ", got ", name_of(t.scalar_type()));
}
void type_is16(const Tensor& t, const char* name) {
    FDS_REQUIRE(is16(t.scalar_type()), name, " must be torch.float16 or torch.bfloat16, got ", name_of(t.scalar_type()));
}
void on_cuda(const Tensor& t, const char* name) {
    FDS_REQUIRE(t.is_cuda(), name, " must be on a CUDA device (there is no CPU fallback)");
}
void on_device(const Tensor& t, const char* name, c10::Device dev) {
    FDS_REQUIRE(t.device() == dev, name, " must be on ", dev.str(), ", got ", t.device().str());
}

uintptr_t address(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

// 2-D, contiguous columns, rows on `align`-byte boundaries that do not overlap
void rows_2d(const Tensor& t, const char* name, uintptr_t align) {
    FDS_REQUIRE(t.dim() == 2, name, " must be 2-D [rows, columns], got ", shape_of(t));
    const int64_t rows = t.size(0), cols = t.size(1);
    FDS_REQUIRE(cols <= 1 || t.stride(1) == 1, name, " columns must be contiguous (stride(1) == 1)");
    FDS_REQUIRE(address(t) % align == 0 &&
              (rows <= 1 || (t.stride(0) >= cols && t.stride(0) * static_cast<int64_t>(t.element_size()) % static_cast<int64_t>(align) == 0)),
          name, " rows must be ", align, "-byte aligned and not overlap");
}
// Row stride in elements; that of a single row is never stepped over: any valid value.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }

void shape_is(const Tensor& t, const char* name, int64_t rows, int64_t cols) {
    FDS_REQUIRE(t.size(0) == rows && t.size(1) == cols, name, " must be [", rows, ", ", cols, "], got ", shape_of(t));
}

void vector_1d(const Tensor& t, const char* name, int64_t n, uintptr_t align) {
    FDS_REQUIRE(t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1) && address(t) % align == 0, name,
          " must be a contiguous, ", align, "-byte aligned [", n, "] tensor, got ", shape_of(t));
}

Tensor make(at::IntArrayRef shape, ScalarType t, c10::Device dev) {
    return at::empty(shape, at::TensorOptions().dtype(t).device(dev));
}

struct StatusWords {
    int32_t* status = nullptr;
    int32_t* mirror = nullptr;
};
StatusWords g_words[64];

// The device's status words; raises if an earlier kernel on it timed out.
StatusWords status_words(c10::Device dev) {
    const int idx = dev.index();
    FDS_REQUIRE(idx >= 0 && idx < 64, "device index ", idx, " out of range");
    StatusWords& w = g_words[idx];
    if (w.mirror == nullptr) {
        PyObject* pair = PyObject_CallFunction(g_status, "i", idx);
        if (pair == nullptr) throw PythonError{};
        unsigned long long a = 0, b = 0;
        const int ok = PyArg_ParseTuple(pair, "KK", &a, &b);
        Py_DECREF(pair);
        if (!ok) throw PythonError{};
        w.status = reinterpret_cast<int32_t*>(a);
        w.mirror = reinterpret_cast<int32_t*>(b);
    }
    if (__builtin_expect(*static_cast<volatile int32_t*>(w.mirror) != 0, 0)) {
        PyObject* r = PyObject_CallFunction(g_raise_timeout, "i", idx);
        if (r == nullptr) throw PythonError{};
        Py_DECREF(r);
    }
    return w;
}

template <typename Args>
void launch(int (*fn)(const Args*, void*), const Args& args, c10::Device dev, const char* name) {
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const int rc = fn(&args, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    FDS_REQUIRE(rc == FDS_OK, name, " failed (code ", rc, "): ", g_last_error());
}

PyObject* pair_of(const Tensor& a, const Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = THPVariable_Wrap(b);
    PyObject* r = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

// ---------------------------------------------------------------- window attention

void heads_4d(const Tensor& t, const char* name, c10::Device dev, ScalarType dt) {
    type_is(t, name, dt);
    on_device(t, name, dev);
    FDS_REQUIRE(t.dim() == 4, name, " must be 4-D [batch, length, heads, 64], got ", shape_of(t));
    FDS_REQUIRE(t.stride(3) == 1 || t.size(3) <= 1, name, " heads must be contiguous (stride(3) == 1)");
}

void batch_vector(const Tensor* t, const char* name, c10::Device dev, int64_t batch) {
    if (t == nullptr) return;
    type_is(*t, name, ScalarType::Int);
    on_device(*t, name, dev);
    vector_1d(*t, name, batch, 4);
}

// (q, k, v, left, right, sinks, q_start, kv_len, out, scale, timeout_ns, debug_flags)
PyObject* window_attention(PyObject* const* a) {
    const Tensor& q = required(a[0], "q");
    type_is16(q, "q");
    on_cuda(q, "q");
    const Tensor& k = required(a[1], "k");
    const Tensor& v = required(a[2], "v");
    const c10::Device dev = q.device();
    const ScalarType dt = q.scalar_type();
    heads_4d(q, "q", dev, dt);
    heads_4d(k, "k", dev, dt);
    heads_4d(v, "v", dev, dt);
    const int64_t batch = q.size(0), q_len = q.size(1), heads = q.size(2), k_len = k.size(1), kv_heads = k.size(2);
    FDS_REQUIRE(q.size(3) == 64, "head_dim must be 64, got ", q.size(3));
    FDS_REQUIRE(k.size(0) == batch && k.size(3) == 64 && k.sizes() == v.sizes(), "k and v must be [", batch,
          ", length, heads, 64], got ", shape_of(k), " and ", shape_of(v));
    FDS_REQUIRE(batch >= 1 && batch <= 65535 && kv_heads >= 1 && kv_heads <= 65535 && heads >= 1 && heads % kv_heads == 0, "heads (",
          heads, ") must be a positive multiple of the key heads (", kv_heads, "), batch and key heads in [1, 65535]");
    const int64_t top = int64_t{1} << 28;
    FDS_REQUIRE(q_len <= top && k_len <= top && heads <= top, "q, k and v are too long");
    const int64_t left = integer(a[3], "left"), right = integer(a[4], "right"), sinks = integer(a[5], "sinks");
    FDS_REQUIRE(left >= 0 && right >= 0 && sinks >= 0, "left, right and sinks must be >= 0");
    const Tensor* q_start = optional(a[6], "q_start");
    const Tensor* kv_len = optional(a[7], "kv_len");
    batch_vector(q_start, "q_start", dev, batch);
    batch_vector(kv_len, "kv_len", dev, batch);
    Tensor out;
    if (a[8] == Py_None) {
        out = make(q.sizes(), dt, dev);
    } else {
        out = required(a[8], "out");
        heads_4d(out, "out", dev, dt);
        FDS_REQUIRE(out.sizes() == q.sizes(), "out must be ", shape_of(q), ", got ", shape_of(out));
    }
    const double scale = a[9] == Py_None ? 0.125 : real(a[9]);
    const StatusWords words = status_words(dev);
    if (q_len > 0 && k_len == 0) {
        out.zero_();
    } else if (q_len > 0) {
        FdsWindowArgs w{};
        w.q = q.data_ptr(), w.k = k.data_ptr(), w.v = v.data_ptr(), w.out = out.data_ptr();
        for (int i = 0; i < 3; ++i) {
            w.q_stride[i] = q.stride(i), w.k_stride[i] = k.stride(i);
            w.v_stride[i] = v.stride(i), w.out_stride[i] = out.stride(i);
        }
        w.q_start = q_start != nullptr ? q_start->data_ptr<int32_t>() : nullptr;
        w.kv_len = kv_len != nullptr ? kv_len->data_ptr<int32_t>() : nullptr;
        w.status = words.status, w.status_host = words.mirror;
        w.batch = static_cast<int32_t>(batch), w.heads = static_cast<int32_t>(heads), w.kv_heads = static_cast<int32_t>(kv_heads);
        w.q_len = static_cast<int32_t>(q_len), w.k_len = static_cast<int32_t>(k_len), w.head_dim = 64, w.dtype = dtype_code(dt);
        w.left = static_cast<int32_t>(std::min(left, top)), w.right = static_cast<int32_t>(std::min(right, top));
        w.sinks = static_cast<int32_t>(std::min(sinks, top));
        w.scale = static_cast<float>(scale);
        w.timeout_ns = integer(a[10], "timeout_ns");
        w.debug_flags = static_cast<int32_t>(integer(a[11], "debug_flags"));
        launch(g_window, w, dev, "fds_window_attn_fwd");
    }
    return THPVariable_Wrap(out);
}

// ---------------------------------------------------------------- 8-bit projections

// out and scale of a quantised [rows, c], allocated when None
void int8_rows(PyObject* o, PyObject* s, int64_t rows, int64_t c, c10::Device dev, Tensor& out, Tensor& scale) {
    if (o == Py_None) {
        out = make({rows, c}, ScalarType::Char, dev);
    } else {
        out = required(o, "out");
        type_is(out, "out", ScalarType::Char);
        on_device(out, "out", dev);
        rows_2d(out, "out", 8);
        shape_is(out, "out", rows, c);
    }
    if (s == Py_None) {
        scale = make({rows}, ScalarType::Float, dev);
    } else {
        scale = required(s, "scale");
        type_is(scale, "scale", ScalarType::Float);
        on_device(scale, "scale", dev);
        vector_1d(scale, "scale", rows, 4);
    }
}

// (x, out, scale)
PyObject* quantize_rows(PyObject* const* a) {
    const Tensor& x = required(a[0], "x");
    type_is16(x, "x");
    on_cuda(x, "x");
    rows_2d(x, "x", 16);
    const int64_t rows = x.size(0), c = x.size(1);
    const c10::Device dev = x.device();
    FDS_REQUIRE(c % 8 == 0 && c >= 8 && c <= 16384, "columns must be a multiple of 8, at most 16384 (got ", c, ")");
    FDS_REQUIRE(rows <= 0x7fffffff, "too many rows");
    Tensor out, scale;
    int8_rows(a[1], a[2], rows, c, dev, out, scale);
    if (rows > 0) {
        FdsResidualNormArgs n{};
        n.x = x.data_ptr(), n.x_stride = row_stride(x);
        n.h = out.data_ptr(), n.h_stride = row_stride(out), n.h_scale = scale.data_ptr<float>();
        n.rows = static_cast<int32_t>(rows), n.c = static_cast<int32_t>(c), n.length = n.rows;
        n.dtype = dtype_code(x.scalar_type());
        n.post = n.norm = FDS_NORM_NONE;
        n.alpha = 1.f;
        launch(g_residual_norm, n, dev, "fds_residual_norm_fwd");
    }
    return pair_of(out, scale);
}

// (x, x_scale, w, w_scale, b, out, dtype, epilogue, cos, sin, length, heads, cta_pair, tile_n)
PyObject* linear_int8(PyObject* const* a) {
    const Tensor& x = required(a[0], "x");
    type_is(x, "x", ScalarType::Char);
    on_cuda(x, "x");
    rows_2d(x, "x", 16);
    const c10::Device dev = x.device();
    const Tensor& w = required(a[2], "w");
    type_is(w, "w", ScalarType::Char);
    on_device(w, "w", dev);
    rows_2d(w, "w", 16);
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    FDS_REQUIRE(w.size(1) == k, "w is ", shape_of(w), " but x has ", k, " columns");
    FDS_REQUIRE(k % 16 == 0 && k > 0 && k <= 65536, "in_features must be a multiple of 16, at most 65536 (got ", k, ")");
    FDS_REQUIRE(n % 8 == 0 && n > 0 && n <= 0x7fffffff && m <= 0x7fffffff, "out_features must be a multiple of 8 (got ", n, ")");
    const Tensor& xs = required(a[1], "x_scale");
    const Tensor& ws = required(a[3], "w_scale");
    type_is(xs, "x_scale", ScalarType::Float);
    type_is(ws, "w_scale", ScalarType::Float);
    on_device(xs, "x_scale", dev);
    on_device(ws, "w_scale", dev);
    vector_1d(xs, "x_scale", m, 4);
    vector_1d(ws, "w_scale", n, 16);
    const Tensor* b = optional(a[4], "b");
    const int epilogue = static_cast<int>(integer(a[7], "epilogue"));
    const ScalarType dt = dtype_or(a[6], b != nullptr ? b->scalar_type() : ScalarType::Half);
    if (b != nullptr) {
        type_is(*b, "b", dt);
        on_device(*b, "b", dev);
        vector_1d(*b, "b", n, 16);
    }
    const bool accum = epilogue == FDS_EPILOGUE_ACCUMULATE_F32;
    const ScalarType ot = accum ? ScalarType::Float : dt;
    Tensor out;
    if (a[5] == Py_None && !accum) {
        out = make({m, n}, ot, dev);
    } else {
        const char* name = accum ? "the residual" : "out";
        out = required(a[5], name);
        type_is(out, name, ot);
        on_device(out, name, dev);
        rows_2d(out, name, 16);
        shape_is(out, name, m, n);
    }
    FdsLinearInt8Args f{};
    if (epilogue == FDS_EPILOGUE_ROPE) {
        const Tensor& cos = required(a[8], "cos");
        const Tensor& sin = required(a[9], "sin");
        const int64_t length = integer(a[10], "length"), heads = integer(a[11], "heads");
        FDS_REQUIRE(heads >= 1 && heads <= 0x7fffffff && n == 192 * heads, "w must have 3*heads*64 = ", 192 * heads, " rows (got ", n, ")");
        FDS_REQUIRE(length >= 1, "length must be >= 1");
        // positions past the last row do not occur: neither do their table rows
        const int64_t seq = std::min(length, std::max<int64_t>(1, m));
        for (const Tensor* t : {&cos, &sin})
            FDS_REQUIRE(t->scalar_type() == ScalarType::Float && t->dim() == 2 && t->size(1) == 64 && t->size(0) >= seq &&
                      t->is_contiguous() && t->device() == dev && address(*t) % 16 == 0,
                  "cos and sin must be contiguous fp32 [>= ", seq, ", 64] tables on ", dev.str());
        f.cos = cos.data_ptr<float>(), f.sin = sin.data_ptr<float>();
        f.seq_len = static_cast<int32_t>(seq), f.rope_cols = static_cast<int32_t>(128 * heads);
    }
    const StatusWords words = status_words(dev);
    if (m > 0) {
        f.a = x.data_ptr(), f.a_row_stride = row_stride(x), f.a_scale = xs.data_ptr<float>();
        f.w = w.data_ptr(), f.w_row_stride = row_stride(w), f.w_scale = ws.data_ptr<float>();
        f.bias = b != nullptr ? b->data_ptr() : nullptr;
        f.out = out.data_ptr(), f.out_row_stride = m > 1 ? out.stride(0) : n;
        f.status = words.status, f.status_host = words.mirror;
        f.m = static_cast<int32_t>(m), f.n = static_cast<int32_t>(n), f.k = static_cast<int32_t>(k);
        f.dtype = dtype_code(dt), f.epilogue = epilogue;
        f.cta_pair = static_cast<int32_t>(integer(a[12], "pair")), f.tile_n = static_cast<int32_t>(integer(a[13], "tile_n"));
        launch(g_linear_int8, f, dev, "fds_linear_int8_fwd");
    }
    return THPVariable_Wrap(out);
}

// ---------------------------------------------------------------- between two blocks

int norm_kind(PyObject* o, const char* name) {
    if (PyUnicode_Check(o)) {
        if (PyUnicode_CompareWithASCIIString(o, "none") == 0) return FDS_NORM_NONE;
        if (PyUnicode_CompareWithASCIIString(o, "layer") == 0) return FDS_NORM_LAYER;
        if (PyUnicode_CompareWithASCIIString(o, "rms") == 0) return FDS_NORM_RMS;
    }
    refuse(name, " must be 'none', 'layer' or 'rms'");
}

// A parameter vector [c], or with `windows` > 0 also [>= windows, c]; its
// address, and the elements between the rows of windows in `stride` (0: one for all)
const void* parameter(const Tensor* t, const char* name, int64_t c, int64_t windows, ScalarType pt, c10::Device dev,
                      int64_t* stride) {
    if (t == nullptr) return nullptr;
    type_is(*t, name, pt);
    on_device(*t, name, dev);
    if (windows > 0 && t->dim() == 2) {
        rows_2d(*t, name, 16);
        FDS_REQUIRE(t->size(1) == c && t->size(0) >= windows, name, " must be [", c, "] or [", windows, ", ", c, "], got ", shape_of(*t));
        *stride = t->size(0) > 1 ? t->stride(0) : 0;
    } else {
        vector_1d(*t, name, c, 16);
    }
    return t->data_ptr();
}

// (x, y, gate, residual_scale, post, post_weight, post_bias, norm, weight, bias, scale, shift, length, eps, dtype,
//  residual_out, out, quantize, out_scale)
PyObject* residual_norm(PyObject* const* a) {
    const Tensor& x = required(a[0], "x");
    on_cuda(x, "x");
    rows_2d(x, "x", 16);
    const c10::Device dev = x.device();
    const int64_t rows = x.size(0), c = x.size(1);
    const Tensor* y = optional(a[1], "y");
    const ScalarType xt = x.scalar_type();
    const ScalarType dt = dtype_or(a[14], y != nullptr ? y->scalar_type() : (is16(xt) ? xt : ScalarType::Half));
    FDS_REQUIRE(xt == ScalarType::Float || xt == dt, "x must be torch.float32 or ", name_of(dt), ", got ", name_of(xt));
    FDS_REQUIRE(c % 8 == 0 && c >= 8 && c <= 16384, "columns must be a multiple of 8, at most 16384 (got ", c, ")");
    FDS_REQUIRE(rows <= 0x7fffffff, "too many rows");
    const Tensor *gate = optional(a[2], "gate"), *post_w = optional(a[5], "post_weight"), *post_b = optional(a[6], "post_bias"),
                 *weight = optional(a[8], "weight"), *bias = optional(a[9], "bias"), *scale = optional(a[10], "scale"),
                 *shift = optional(a[11], "shift");
    const double alpha = real(a[3]), eps = real(a[13]);
    const int64_t length = a[12] == Py_None ? std::max<int64_t>(1, rows) : integer(a[12], "length");
    FDS_REQUIRE(length >= 1, "length must be >= 1");
    FdsResidualNormArgs n{};
    n.post = norm_kind(a[4], "post");
    n.norm = norm_kind(a[7], "norm");
    Tensor x_new = x;
    if (y != nullptr) {
        type_is(*y, "y", dt);
        on_device(*y, "y", dev);
        rows_2d(*y, "y", 16);
        shape_is(*y, "y", rows, c);
        if (a[15] != Py_None) {
            x_new = required(a[15], "residual_out");
            type_is(x_new, "residual_out", xt);
            on_device(x_new, "residual_out", dev);
            rows_2d(x_new, "residual_out", 16);
            shape_is(x_new, "residual_out", rows, c);
        }
        n.y = y->data_ptr(), n.y_stride = row_stride(*y);
        n.x_out = x_new.data_ptr(), n.x_out_stride = row_stride(x_new);
    } else {
        FDS_REQUIRE(gate == nullptr && n.post == FDS_NORM_NONE && post_w == nullptr && post_b == nullptr && alpha == 1.0 && a[15] == Py_None,
              "gate, residual_scale, residual_out and the norm after the block need y");
    }
    ScalarType pt = dt;
    for (const Tensor* t : {gate, post_w, post_b, weight, bias, scale, shift})
        if (t != nullptr) {
            pt = t->scalar_type();
            break;
        }
    FDS_REQUIRE(pt == ScalarType::Float || pt == dt, "parameter vectors must be torch.float32 or ", name_of(dt), ", got ", name_of(pt));
    const int64_t windows = std::max<int64_t>(1, (rows + length - 1) / length);
    int64_t shift_stride = 0, none = 0;
    n.post_w = parameter(post_w, "post_weight", c, 0, pt, dev, &none);
    n.post_b = parameter(post_b, "post_bias", c, 0, pt, dev, &none);
    n.w = parameter(weight, "weight", c, 0, pt, dev, &none);
    n.b = parameter(bias, "bias", c, 0, pt, dev, &none);
    n.gate = parameter(gate, "gate", c, windows, pt, dev, &n.gate_stride);
    n.scale = parameter(scale, "scale", c, windows, pt, dev, &n.mod_stride);
    n.shift = parameter(shift, "shift", c, windows, pt, dev, &shift_stride);
    if (scale == nullptr)
        n.mod_stride = shift_stride;
    else
        FDS_REQUIRE(shift == nullptr || shift_stride == n.mod_stride || windows == 1, "scale and shift must have the same layout");
    if (windows == 1) n.gate_stride = n.mod_stride = 0;
    const int quantize = PyObject_IsTrue(a[17]);
    if (quantize < 0) throw PythonError{};
    Tensor out, out_scale;
    if (quantize) {
        int8_rows(a[16], a[18], rows, c, dev, out, out_scale);
    } else {
        FDS_REQUIRE(a[18] == Py_None, "out_scale is for quantize=True");
        if (a[16] == Py_None) {
            out = make({rows, c}, dt, dev);
        } else {
            out = required(a[16], "out");
            type_is(out, "out", dt);
            on_device(out, "out", dev);
            rows_2d(out, "out", 16);
            shape_is(out, "out", rows, c);
        }
    }
    if (rows > 0) {
        n.x = x.data_ptr(), n.x_stride = row_stride(x);
        n.h = out.data_ptr(), n.h_stride = row_stride(out);
        n.h_scale = quantize ? out_scale.data_ptr<float>() : nullptr;
        n.rows = static_cast<int32_t>(rows), n.c = static_cast<int32_t>(c);
        n.length = static_cast<int32_t>(std::min<int64_t>(length, 0x7fffffff));
        n.dtype = dtype_code(dt), n.x_f32 = xt == ScalarType::Float, n.param_f32 = pt == ScalarType::Float;
        n.alpha = static_cast<float>(alpha), n.eps = static_cast<float>(eps);
        launch(g_residual_norm, n, dev, "fds_residual_norm_fwd");
    }
    PyObject* h = quantize ? pair_of(out, out_scale) : THPVariable_Wrap(out);
    PyObject* xn = THPVariable_Wrap(x_new);
    PyObject* r = h != nullptr && xn != nullptr ? PyTuple_Pack(2, xn, h) : nullptr;
    Py_XDECREF(h);
    Py_XDECREF(xn);
    return r;
}

// ---------------------------------------------------------------- module

template <PyObject* (*fn)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
        return nullptr;
    }
    try {
        if (g_window == nullptr) refuse("the native library is not bound");
        return fn(args);
    } catch (const Refused& e) {
        PyErr_SetString(g_error, e.what.c_str());
    } catch (const PythonError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// (FdsError, status callback, timeout callback, addresses of fds_last_error and the three entry points)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *error, *status, *raise_timeout;
    unsigned long long last, linear, norm, window;
    if (!PyArg_ParseTuple(args, "OOOKKKK", &error, &status, &raise_timeout, &last, &linear, &norm, &window)) return nullptr;
    Py_INCREF(error);
    Py_INCREF(status);
    Py_INCREF(raise_timeout);
    g_error = error, g_status = status, g_raise_timeout = raise_timeout;
    g_last_error = reinterpret_cast<LastError>(last);
    g_linear_int8 = reinterpret_cast<decltype(g_linear_int8)>(linear);
    g_residual_norm = reinterpret_cast<decltype(g_residual_norm)>(norm);
    g_window = reinterpret_cast<decltype(g_window)>(window);
    Py_RETURN_NONE;
}

template <PyObject* (*fn)(PyObject* const*), int kArgs>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<fn, kArgs>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    method<window_attention, 12>("window_attention"),
    method<quantize_rows, 3>("quantize_rows"),
    method<linear_int8, 14>("linear_int8"),
    method<residual_norm, 19>("residual_norm"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fds_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fds_torch() { return PyModule_Create(&g_module); }

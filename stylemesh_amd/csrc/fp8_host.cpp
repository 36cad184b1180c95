// Host side of the 8-bit operators (runtime/fp8.py): a call's checks, allocations and the library call in native code. The
// smallest calls are bound by the host: quantising 16 x 4096 takes 2.6 us of kernel and took 9.3 us of interpreter (two allocations
// at 1.4 us each, fifteen attribute reads, the foreign-function call); from here it takes 5.8, of which 3.2 are the launch's own.
// What is not in order comes back as None, and the Python side says why.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>

#include <algorithm>

#include "../../include/stylemesh_hip.h"

namespace {

constexpr int64_t BLOCK = 128, MAX_DIM = 65535 * 128;
constexpr at::ScalarType TYPES[] = {at::kFloat, at::kBFloat16, at::kHalf};                 // SM_TYPE_*
constexpr at::ScalarType FORMATS[] = {at::kFloat8_e4m3fn, at::kFloat8_e5m2};               // SM_FP8_*

at::Tensor room(at::IntArrayRef size, at::ScalarType type, int device) {
    return at::empty(size, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (at::DeviceIndex)device)));
}

// a float32 / bfloat16 / float16 matrix of `device` with unit column stride and rows that do not overlap
struct Matrix {
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, stride = 0;
    int type = -1;
    bool take(PyObject* o, int device, bool in_graph) {      // in_graph: the result would belong to its autograd graph
        if (!THPVariable_Check(o)) return false;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (in_graph && t.requires_grad() && at::GradMode::is_enabled()) return false;
        if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() != 2 || t.get_device() != device || t.is_neg()) return false;
        for (int i = 0; i < 3; ++i)
            if (t.scalar_type() == TYPES[i]) type = i;
        rows = t.size(0), cols = t.size(1);
        if (type < 0 || rows > MAX_DIM || cols > MAX_DIM || (cols > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < cols)) return false;
        stride = rows > 1 ? t.stride(0) : std::max<int64_t>(cols, 1);
        p = t.const_data_ptr();
        return true;
    }
};

// A matrix of 8-bit codes as its Fp8Matrix keeps it: its addresses are read at every call. False where its tensors no longer hold
// what the matrix was made of (memory given up or exchanged since: a weight that was moved away, for one).
bool holds(const at::Tensor& t, int64_t bytes, int device) {
    return t.is_cuda() && t.get_device() == device && t.is_contiguous() && (int64_t)t.nbytes() == bytes &&
           t.storage_offset() * (int64_t)t.itemsize() + bytes <= (int64_t)t.storage().nbytes();
}
struct Coded {
    const void *codes = nullptr, *scale = nullptr;
    bool take(PyObject* data, PyObject* scales, int64_t rows, int64_t pitch, int tiles, int f32, int device) {
        if (!THPVariable_Check(data) || !THPVariable_Check(scales)) return false;
        const at::Tensor &d = THPVariable_Unpack(data), &s = THPVariable_Unpack(scales);
        const int64_t kb = pitch / BLOCK, sr = tiles ? (rows + BLOCK - 1) / BLOCK : rows;
        if (!holds(d, rows * pitch, device) || !holds(s, f32 ? kb * sr * 4 : (kb + 3) / 4 * sr * 4, device)) return false;
        codes = d.const_data_ptr(), scale = s.const_data_ptr();
        return (uintptr_t)codes % 16 == 0 && (uintptr_t)scale % 4 == 0;
    }
};

// The arguments of a call, taken in order. Integers and pointers only; a tensor or None is taken as the object.
struct Args {
    PyObject* const* a;
    Py_ssize_t n, at = 0;
    PyObject* object() { return a[at++]; }
    long integer() { return PyLong_AsLong(a[at++]); }
    void* pointer() { return a[at] == Py_None ? (++at, nullptr) : PyLong_AsVoidPtr(a[at++]); }
};
bool expect(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, got %zd", want, n);
    return false;
}
// the library call (no exceptions: a C interface), without the interpreter lock
template <class F>
bool launch(const char* what, F f) {
    PyThreadState* state = PyEval_SaveThread();
    const int e = f();
    PyEval_RestoreThread(state);
    if (e) PyErr_Format(PyExc_RuntimeError, "libstylemesh_hip: %s failed with HIP error code %d", what, e);
    return e == 0;
}

// a caller's tensor was written behind autograd's back: its version counter rises, as after any in-place operation
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();      // (inference tensors have no counter)
}

// room for a matrix of 8-bit codes: (codes, scales) for Python, the pointers for the library
PyObject* coded(int64_t rows, int64_t cols, int fmt, int tiles, int device, void** q, void** s) {
    const int64_t kb = (cols + BLOCK - 1) / BLOCK;
    at::Tensor codes = room({rows, kb * BLOCK}, FORMATS[fmt], device);
    at::Tensor scale = room({(kb + 3) / 4, tiles ? (rows + BLOCK - 1) / BLOCK : rows, 4}, at::kByte, device);
    *q = codes.data_ptr(), *s = scale.data_ptr();
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scale)));
}

// quantize(x, fmt, tiles, plain, transpose, device, stream) -> (rows, cols, parts or None, parts or None)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!expect(n, 7)) return nullptr;
    Args g{a, n};
    PyObject* x = g.object();
    const int fmt = (int)g.integer(), tiles = (int)g.integer(), plain = (int)g.integer(), transpose = (int)g.integer(), device = (int)g.integer();
    void* stream = g.pointer();
    if (PyErr_Occurred()) return nullptr;
    Matrix m;
    if (fmt < 0 || fmt > 1 || !m.take(x, device, false)) Py_RETURN_NONE;
    void *q = nullptr, *qs = nullptr, *qt = nullptr, *qts = nullptr;
    THPObjectPtr first(plain ? coded(m.rows, m.cols, fmt, tiles, device, &q, &qs) : Py_NewRef(Py_None));
    THPObjectPtr second(transpose ? coded(m.cols, m.rows, fmt, tiles, device, &qt, &qts) : Py_NewRef(Py_None));
    if (!first || !second) return nullptr;
    if (m.rows && m.cols && !launch("sm_fp8_quantize", [&] {
            return sm_fp8_quantize(m.p, m.type, (int)m.rows, (int)m.cols, (size_t)m.stride, fmt, tiles, q, qs, qt, qts, stream);
        }))
        return nullptr;
    return Py_BuildValue("LLNN", (long long)m.rows, (long long)m.cols, first.release(), second.release());
    END_HANDLE_TH_ERRORS
}

// fast: the sums may run on the 8-bit matrix instruction (bfloat16 results)
int result_type(int type, int fast) { return fast ? type | SM_FP8_FAST_SUM : type; }

// matmul(a, a_scale, a_fmt, a_pitch, b, b_scale, b_tiles, b_pitch, f32, M, N, K, out, out_type, accumulate, fast, device, stream) -> out;
// out: a tensor, or None for a new one of out_type
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!expect(n, 18)) return nullptr;
    Args g{a, n};
    PyObject *ac = g.object(), *as = g.object();
    const int a_fmt = (int)g.integer();
    const long a_pitch = g.integer();
    PyObject *bc = g.object(), *bs = g.object();
    const int b_tiles = (int)g.integer();
    const long b_pitch = g.integer();
    const int f32 = (int)g.integer();
    const long M = g.integer(), N = g.integer(), K = g.integer();
    PyObject* given = g.object();
    int type = (int)g.integer();
    const int accumulate = (int)g.integer(), fast = (int)g.integer(), device = (int)g.integer();
    void* stream = g.pointer();
    if (PyErr_Occurred()) return nullptr;
    if (M < 0 || N < 0 || K < 0 || M > MAX_DIM || N > MAX_DIM || K > MAX_DIM) Py_RETURN_NONE;
    Coded ca, cb;
    if (!ca.take(ac, as, M, a_pitch, 0, f32, device) || !cb.take(bc, bs, N, b_pitch, b_tiles, f32, device)) Py_RETURN_NONE;
    Matrix o;
    at::Tensor out;
    if (given != Py_None) {
        if (!o.take(given, device, true) || o.rows != M || o.cols != N) Py_RETURN_NONE;
        out = THPVariable_Unpack(given);
        type = o.type;
    } else {
        if (type < 0 || type > 2) Py_RETURN_NONE;
        out = room({M, N}, TYPES[type], device);
        o.stride = std::max(N, 1l);
    }
    if (M && N) {
        const size_t need = sm_fp8_matmul_ws_bytes((int)M, (int)N, (int)K);
        // scratch of this call's own: two captured graphs, or two streams, never share slabs
        at::Tensor ws = need ? room({(int64_t)need}, at::kByte, device) : at::Tensor();
        void *op = out.data_ptr(), *wp = need ? ws.data_ptr() : nullptr;
        if (!launch("sm_fp8_matmul", [&] {
                return sm_fp8_matmul(ca.codes, ca.scale, a_fmt, (size_t)a_pitch, cb.codes, cb.scale, b_tiles, (size_t)b_pitch, f32, (int)M, (int)N, (int)K, op,
                                     result_type(type, fast), (size_t)o.stride, accumulate, wp, need, stream);
            }))
            return nullptr;
    }
    if (given == Py_None) return THPVariable_Wrap(std::move(out));
    written(out);
    return Py_NewRef(given);
    END_HANDLE_TH_ERRORS
}

// linear(x, w, w_scale, w_tiles, w_pitch, N, K, out_type or -1: x's, fast, device, stream) -> y
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!expect(n, 11)) return nullptr;
    Args g{a, n};
    PyObject* x = g.object();
    PyObject *wc = g.object(), *ws = g.object();
    const int tiles = (int)g.integer();
    const long pitch = g.integer(), N = g.integer(), K = g.integer();
    int type = (int)g.integer();
    const int fast = (int)g.integer(), device = (int)g.integer();
    void* stream = g.pointer();
    if (PyErr_Occurred()) return nullptr;
    Matrix m;
    if (!m.take(x, device, true) || m.cols != K || N < 0 || N > MAX_DIM || type > 2) Py_RETURN_NONE;
    Coded w;
    if (!w.take(wc, ws, N, pitch, tiles, 0, device)) Py_RETURN_NONE;
    if (type < 0) type = m.type;
    at::Tensor y = room({m.rows, N}, TYPES[type], device);
    if (m.rows && N) {
        const size_t need = sm_fp8_linear_ws_bytes((int)m.rows, (int)N, (int)K);
        at::Tensor scratch = need ? room({(int64_t)need}, at::kByte, device) : at::Tensor();      // of this call's own, as matmul's
        void *yp = y.data_ptr(), *sp = need ? scratch.data_ptr() : nullptr;
        if (!launch("sm_fp8_linear", [&] {
                return sm_fp8_linear(m.p, m.type, (size_t)m.stride, w.codes, w.scale, tiles, (size_t)pitch, (int)m.rows, (int)N, (int)K, yp,
                                     result_type(type, fast), (size_t)N, sp, need, stream);
            }))
            return nullptr;
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// backward(dy, fmt, K, wt, wt_scale, wt_tiles, wt_pitch, xt, xt_scale, xt_tiles, xt_pitch, dx_type or -1: dy's, dw, accumulate, fast (dx),
// device, stream) -> (dx or None, dw or None), M, N, K > 0; wt / xt None: that gradient is not wanted; dw: a float32 matrix, or None for a new one
PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!expect(n, 17)) return nullptr;
    Args g{a, n};
    PyObject* dyo = g.object();
    const int fmt = (int)g.integer();
    const long K = g.integer();
    PyObject *wtc = g.object(), *wts = g.object();
    const int wt_tiles = (int)g.integer();
    const long wt_pitch = g.integer();
    PyObject *xtc = g.object(), *xts = g.object();
    const int xt_tiles = (int)g.integer();
    const long xt_pitch = g.integer();
    int type = (int)g.integer();
    PyObject* given = g.object();
    const int accumulate = (int)g.integer(), fast = (int)g.integer(), device = (int)g.integer();
    void* stream = g.pointer();
    if (PyErr_Occurred()) return nullptr;
    Matrix dy, w;
    if (!dy.take(dyo, device, true) || !dy.rows || !dy.cols || K <= 0 || K > MAX_DIM || fmt < 0 || fmt > 1 || type > 2) Py_RETURN_NONE;
    const bool wt = wtc != Py_None, xt = xtc != Py_None;      // the gradients wanted
    Coded cw, cx;
    if ((wt && !cw.take(wtc, wts, K, wt_pitch, wt_tiles, 0, device)) || (xt && !cx.take(xtc, xts, K, xt_pitch, xt_tiles, 0, device))) Py_RETURN_NONE;
    if (type < 0) type = dy.type;
    at::Tensor dx, dw;
    if (wt) dx = room({dy.rows, K}, TYPES[type], device);
    if (xt && given != Py_None) {
        if (!w.take(given, device, true) || w.type != 0 || w.rows != dy.cols || w.cols != K) Py_RETURN_NONE;
        dw = THPVariable_Unpack(given);
    } else if (xt) {
        dw = room({dy.cols, K}, at::kFloat, device);
        w.stride = K;
    }
    const size_t need = sm_fp8_linear_backward_ws_bytes((int)dy.rows, (int)dy.cols, (int)K, wt, xt);
    at::Tensor scratch = room({(int64_t)need}, at::kByte, device);
    void *dxp = wt ? dx.data_ptr() : nullptr, *dwp = xt ? dw.data_ptr() : nullptr, *sp = scratch.data_ptr();
    if (!launch("sm_fp8_linear_backward", [&] {
            return sm_fp8_linear_backward(dy.p, dy.type, (size_t)dy.stride, fmt, (int)dy.rows, (int)dy.cols, (int)K, cw.codes, cw.scale, wt_tiles, (size_t)wt_pitch,
                                          cx.codes, cx.scale, xt_tiles, (size_t)xt_pitch, dxp, result_type(type, fast), (size_t)K, (float*)dwp, (size_t)w.stride, accumulate, sp, need, stream);
        }))
        return nullptr;
    if (xt && given != Py_None) written(dw);
    return Py_BuildValue("NN", wt ? THPVariable_Wrap(std::move(dx)) : Py_NewRef(Py_None),
                         !xt ? Py_NewRef(Py_None) : given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(std::move(dw)));
    END_HANDLE_TH_ERRORS
}

PyMethodDef METHODS[] = {
    {"quantize", (PyCFunction)(void (*)())quantize, METH_FASTCALL, nullptr},
    {"matmul", (PyCFunction)(void (*)())matmul, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)())linear, METH_FASTCALL, nullptr},
    {"backward", (PyCFunction)(void (*)())backward, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_fp8_host", "Calls of the 8-bit operators", -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_host() { return PyModule_Create(&MODULE); }

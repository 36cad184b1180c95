// Host side of the gradient-list operators (runtime/gradclip.py): a list of tensors as the arrays sm_grad_norm / sm_grad_clip
// read, in one walk. A model's few hundred gradients are handed over anew every step, and an attribute of a tensor costs
// Python 70 ns: five of each of 161 gradients and their outputs were 95 of the call's 116 us, the kernels 34. Reads pointers, sizes
// and types only; nothing is kept between calls.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <vector>

namespace {

// An entry of a packed table: n pointers, n element counts (64 bits each), n types (int, SM_TYPE_*), one after the other.
constexpr Py_ssize_t ENTRY = 8 + 8 + 4;
constexpr long NO_DEVICE = -2, MIXED = -3;      // (-1: host)

struct Table {
    const uint64_t *ptr, *numel;
    const int32_t* type;
    Py_ssize_t n;
    uint64_t begin(Py_ssize_t i) const { return ptr[i]; }
    uint64_t end(Py_ssize_t i) const { return ptr[i] + numel[i] * (type[i] == 0 ? 4u : 2u); }
};

bool as_table(PyObject* o, Table& t) {
    if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) % ENTRY) {
        PyErr_SetString(PyExc_TypeError, "a packed table");
        return false;
    }
    t.n = PyBytes_GET_SIZE(o) / ENTRY;
    t.ptr = reinterpret_cast<const uint64_t*>(PyBytes_AS_STRING(o));
    t.numel = t.ptr + t.n;
    t.type = reinterpret_cast<const int32_t*>(t.numel + t.n);
    return true;
}

// pack(list) -> (table, its address, index of the first tensor of another type than fp32 / bf16 / fp16 (or that is no plain strided
// tensor) or -1, device of all, all contiguous?)
PyObject* pack(PyObject*, PyObject* arg) {
    if (!PyList_Check(arg)) {
        PyErr_SetString(PyExc_TypeError, "a list of tensors");
        return nullptr;
    }
    const Py_ssize_t n = PyList_GET_SIZE(arg);
    PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * ENTRY);
    if (!bytes) return nullptr;
    auto* ptr = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(bytes));
    uint64_t* numel = ptr + n;
    auto* type = reinterpret_cast<int32_t*>(numel + n);
    long device = NO_DEVICE;
    Py_ssize_t odd = -1;
    bool contiguous = true;
    try {
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(arg, i);
            if (!THPVariable_Check(o)) {
                Py_DECREF(bytes);
                PyErr_Format(PyExc_ValueError, "entry %zd is not a tensor", i);
                return nullptr;
            }
            const at::Tensor& t = THPVariable_Unpack(o);
            const auto s = t.scalar_type();
            const bool plain = t.layout() == at::kStrided && !t.is_neg();
            type[i] = !plain ? -1 : s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : s == at::kHalf ? 2 : -1;
            const long d = t.is_cuda() ? (long)t.get_device() : -1;
            device = device == NO_DEVICE || device == d ? d : MIXED;
            ptr[i] = numel[i] = 0;
            if (type[i] < 0 && odd < 0) odd = i;
            if (type[i] < 0 || d < 0) continue;
            ptr[i] = reinterpret_cast<uint64_t>(t.data_ptr());
            numel[i] = (uint64_t)t.numel();
            contiguous = contiguous && t.is_contiguous();
        }
    } catch (const std::exception& e) {      // (a tensor without storage, for one)
        Py_DECREF(bytes);
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    const auto address = (unsigned long long)reinterpret_cast<uint64_t>(PyBytes_AS_STRING(bytes));
    return Py_BuildValue("NKnlN", bytes, address, odd, device, PyBool_FromLong(contiguous));
}

// check_outputs(inputs, outputs) -> 0: every output may be written; 1: an output has not as many elements as its input; 2: an
// output that is its input has another type; 3: two outputs overlap; 4: an output overlaps an input that is not its own (its
// own: the same entry, starting at the same address)
PyObject* check_outputs(PyObject*, PyObject* args) {
    PyObject *a, *b;
    Table g, o;
    if (!PyArg_ParseTuple(args, "OO", &a, &b) || !as_table(a, g) || !as_table(b, o)) return nullptr;
    if (g.n != o.n) {
        PyErr_SetString(PyExc_ValueError, "tables of different lengths");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < g.n; ++i)
        if (g.numel[i] != o.numel[i]) return PyLong_FromLong(1);
    for (Py_ssize_t i = 0; i < g.n; ++i)
        if (g.numel[i] && g.ptr[i] == o.ptr[i] && g.type[i] != o.type[i]) return PyLong_FromLong(2);
    try {
        std::vector<Py_ssize_t> order;
        order.reserve(o.n);
        for (Py_ssize_t i = 0; i < o.n; ++i)
            if (o.numel[i]) order.push_back(i);
        std::sort(order.begin(), order.end(), [&](Py_ssize_t x, Py_ssize_t y) { return o.begin(x) < o.begin(y); });
        for (size_t k = 1; k < order.size(); ++k)
            if (o.end(order[k - 1]) > o.begin(order[k])) return PyLong_FromLong(3);
        if (a != b)
            for (Py_ssize_t i = 0; i < g.n; ++i) {
                if (!g.numel[i]) continue;
                // the outputs are disjoint and in order: the first that ends behind this input's begin, and whatever follows
                auto k = std::partition_point(order.begin(), order.end(), [&](Py_ssize_t x) { return o.end(x) <= g.begin(i); });
                for (; k != order.end() && o.begin(*k) < g.end(i); ++k)
                    if (*k != i || o.begin(i) != g.begin(i)) return PyLong_FromLong(4);
            }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    return PyLong_FromLong(0);
}

// written(list): the tensors have been written behind autograd's back; their version counters rise, as after any in-place operation
PyObject* written(PyObject*, PyObject* arg) {
    if (!PyList_Check(arg)) {
        PyErr_SetString(PyExc_TypeError, "a list of tensors");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(arg); ++i) {
        PyObject* o = PyList_GET_ITEM(arg, i);
        if (!THPVariable_Check(o)) {
            PyErr_Format(PyExc_ValueError, "entry %zd is not a tensor", i);
            return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();      // (inference tensors have no counter)
    }
    Py_RETURN_NONE;
}

PyMethodDef METHODS[] = {
    {"pack", pack, METH_O, "list of tensors -> (table, address, odd one, device, contiguous)"},
    {"check_outputs", check_outputs, METH_VARARGS, "(inputs, outputs) -> 0, or what is wrong with the outputs"},
    {"written", written, METH_O, "list of tensors: raises their version counters"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_tensor_list", "Tensor lists as the library's arrays", -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list() { return PyModule_Create(&MODULE); }

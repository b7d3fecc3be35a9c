// Python extension `_tensor_list`: what a list of torch tensors holds, read in one call.
//
// Operators over many small tensors (the gradients of every bias of a model) would otherwise spend
// some 0.4 us per tensor reading its pointer, size, type, device and layout through Python
// (256 tensors and their outputs: 112 us of a call whose kernels take 8 us).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>
#include <vector>

namespace {

// describe(list of tensors) -> (pointers, counts, total, type, device): the first two are bytes
// objects of 64-bit words, total is the number of elements; type is the common element type as a
// bccl::DataType (f32, bf16, f16), device the common CUDA device. None where the list is not that
// simple: mixed types or devices, host memory, other types, tensors that are not contiguous.
PyObject* Describe(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "describe: a list of tensors");
        return nullptr;
    }
    const Py_ssize_t n = PyList_GET_SIZE(list);
    PyObject* ptrs = PyBytes_FromStringAndSize(nullptr, n * static_cast<Py_ssize_t>(sizeof(uint64_t)));
    PyObject* counts = PyBytes_FromStringAndSize(nullptr, n * static_cast<Py_ssize_t>(sizeof(uint64_t)));
    if (ptrs == nullptr || counts == nullptr) {
        Py_XDECREF(ptrs);
        Py_XDECREF(counts);
        return nullptr;
    }
    auto* p = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(ptrs));
    auto* c = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(counts));
    int type = -1, device = -1;
    uint64_t total = 0;
    bool simple = n > 0;
    try {
        for (Py_ssize_t i = 0; i < n && simple; ++i) {
            PyObject* item = PyList_GET_ITEM(list, i);
            simple = THPVariable_CheckExact(item);
            if (!simple) break;
            const at::Tensor& t = THPVariable_Unpack(item);
            simple = t.defined() && t.layout() == at::kStrided && t.has_storage() && t.is_cuda() && t.is_contiguous();
            if (!simple) break;
            const auto s = t.scalar_type();
            const int k = s == at::kFloat ? 0 : s == at::kBFloat16 ? 4 : s == at::kHalf ? 5 : -1;
            const int d = static_cast<int>(t.get_device());
            if (i == 0) {
                type = k;
                device = d;
            }
            simple = k >= 0 && k == type && d == device;
            p[i] = reinterpret_cast<uint64_t>(t.data_ptr());
            c[i] = static_cast<uint64_t>(t.numel());
            total += c[i];
        }
    } catch (...) {  // tensors that hold no memory of their own
        simple = false;
    }
    if (!simple) {
        Py_DECREF(ptrs);
        Py_DECREF(counts);
        Py_RETURN_NONE;
    }
    return Py_BuildValue("(NNKii)", ptrs, counts, static_cast<unsigned long long>(total), type, device);
}

// apart(written, their counts, size, read, their counts, size) -> bool: no written tensor (counts[i] elements
// of `size` bytes) overlaps another one or any of the tensors read.
PyObject* Apart(PyObject*, PyObject* args) {
    Py_buffer b[4] = {};
    int size[2] = {};
    if (!PyArg_ParseTuple(args, "y*y*iy*y*i", &b[0], &b[1], &size[0], &b[2], &b[3], &size[1])) return nullptr;
    const bool lengths = b[0].len == b[1].len && b[2].len == b[3].len && b[0].len % 8 == 0 && b[2].len % 8 == 0;
    struct Range {
        uint64_t from, to;
        bool written;
    };
    bool apart = true, memory = true;
    if (lengths) try {
        std::vector<Range> ranges;
        ranges.reserve(static_cast<size_t>((b[0].len + b[2].len) / 8));
        for (int w = 0; w < 2; ++w) {
            for (Py_ssize_t i = 0; i < b[2 * w].len; i += 8) {
                uint64_t p, n;
                std::memcpy(&p, static_cast<const char*>(b[2 * w].buf) + i, 8);
                std::memcpy(&n, static_cast<const char*>(b[2 * w + 1].buf) + i, 8);
                if (n > 0) ranges.push_back({p, p + n * static_cast<uint64_t>(size[w]), w == 0});
            }
        }
        std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
        uint64_t any = 0, written = 0;  // ends of the ranges so far
        for (const Range& x : ranges) {
            if (x.from < (x.written ? any : written)) {
                apart = false;
                break;
            }
            any = std::max(any, x.to);
            if (x.written) written = std::max(written, x.to);
        }
    } catch (const std::bad_alloc&) {
        memory = false;
    }
    for (Py_buffer& x : b) PyBuffer_Release(&x);
    if (!memory) return PyErr_NoMemory();
    if (!lengths) {
        PyErr_SetString(PyExc_ValueError, "apart: lists of different lengths");
        return nullptr;
    }
    return PyBool_FromLong(apart ? 1 : 0);
}

PyMethodDef methods[] = {{"describe", Describe, METH_O, "(pointers, counts, total, type, device) of a list"},
                         {"apart", Apart, METH_VARARGS, "whether written tensors overlap nothing"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list() { return PyModule_Create(&module); }

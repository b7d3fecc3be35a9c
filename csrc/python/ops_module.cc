// Python extension `_ops`: the compute operators on torch tensors.
//
// Checks the operands, allocates outputs and workspaces from torch's allocator on the current
// stream and calls the C interface (bccl/ops.h). The smallest calls are bound by the host: a kernel of
// 2 us took 13 us behind Python checks, tensor allocations and ctypes, and reading 256 gradients
// and their outputs through Python 112 us. originccl_b200/ops documents the arguments.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "bccl/c_api.h"
#include "bccl/ops.h"

namespace {

using at::Tensor;
using Optional = std::optional<Tensor>;

// Raised as a Python exception of that type; a null type means that one is set already.
struct Refusal {
    PyObject* type;
    std::string what;
};
[[noreturn]] void type_error(const std::string& what) { throw Refusal{PyExc_TypeError, what}; }
[[noreturn]] void value_error(const std::string& what) { throw Refusal{PyExc_ValueError, what}; }

std::string shape_of(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}
std::string shape_of(const Tensor& t) { return shape_of(t.sizes()); }
std::string type_of(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    default: return at::toString(t);
    }
}

// ---------------------------------------------------------------- arguments
[[noreturn]] void no_storage(const char* op, const char* what) {
    // Wrappers (distributed tensors, say) have a shape, a type and a device but no storage of their own, and the
    // C interface reads a null pointer as "not given": a weight would be left out without a word.
    type_error(std::string(op) + ": " + what + " must have memory of its own, got a tensor without storage");
}
const Tensor& strided(const char* op, const char* what, PyObject* o) {
    if (!THPVariable_Check(o)) type_error(std::string(op) + ": " + what + " must be a tensor");
    const Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided) type_error(std::string(op) + ": " + what + " must be a strided tensor");
    if (t.is_neg()) type_error(std::string(op) + ": " + what + " must not be a view of negated values");
    return t;
}
const Tensor& tensor(const char* op, const char* what, PyObject* o) {
    const Tensor& t = strided(op, what, o);
    if (t.numel() != 0 && t.const_data_ptr() == nullptr) no_storage(op, what);
    return t;
}
Optional optional_tensor(const char* op, const char* what, PyObject* o) {
    if (o == Py_None) return std::nullopt;
    return tensor(op, what, o);
}
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refusal{nullptr, ""};
    return v != 0;
}

// ---------------------------------------------------------------- checks
int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 4 : t == at::kHalf ? 5 : -1; }
int size_of(int code) { return code == 0 ? 4 : 2; }

int float_code(const char* op, const char* what, const Tensor& t) {
    const int c = code_of(t.scalar_type());
    if (c < 0)
        type_error(std::string(op) + ": " + what + " must be float32, bfloat16 or float16, got " + type_of(t.scalar_type()));
    return c;
}
int int_code(const char* op, const char* what, const Tensor& t) {
    if (t.scalar_type() == at::kLong) return 3;
    if (t.scalar_type() != at::kInt)
        type_error(std::string(op) + ": " + what + " must be int32 or int64, got " + type_of(t.scalar_type()));
    return 2;
}
// A parameter next to operands of type `like`: the same type, or float32.
int like_or_f32(const char* op, const char* what, const Tensor& t, at::ScalarType like) {
    if (t.scalar_type() != like && t.scalar_type() != at::kFloat)
        type_error(std::string(op) + ": " + what + " must be " + type_of(like) + " or float32, got " +
                   type_of(t.scalar_type()));
    return code_of(t.scalar_type());
}
// All on the CUDA device of the first.
template <typename... Rest>
int one_device(const char* op, const Tensor& first, const Rest&... rest) {
    const auto bad = [&](const Tensor& t) {
        value_error(std::string(op) + ": operands must be CUDA tensors on one device, got " + first.device().str() +
                    " and " + t.device().str());
    };
    if (!first.is_cuda()) bad(first);
    const auto device = first.get_device();
    [[maybe_unused]] const auto check = [&](const auto& t) {
        if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Optional>) {
            if (t && (!t->is_cuda() || t->get_device() != device)) bad(*t);
        } else {
            if (!t.is_cuda() || t.get_device() != device) bad(t);
        }
    };
    (check(rest), ...);
    return static_cast<int>(device);
}

// A tensor as rows of its last dimension; copies only layouts whose rows are not evenly spaced
// with adjacent elements.
struct Rows {
    Tensor t;
    int64_t stride;
    Rows(const Tensor& from, int64_t h) : t(from), stride(h) {
        if (t.is_contiguous()) return;
        if (t.dim() == 2 && (h == 1 || t.stride(1) == 1)) {
            stride = t.stride(0);
            return;
        }
        t = t.contiguous();
    }
};
int64_t out_rows(const char* op, const Tensor& out, at::IntArrayRef shape, at::ScalarType type) {
    if (out.scalar_type() != type || out.sizes() != shape)
        value_error(std::string(op) + ": out must be a " + type_of(type) + " tensor of shape " + shape_of(shape) + ", got " +
                    type_of(out.scalar_type()) + " " + shape_of(out));
    const int64_t h = shape.back();
    if (out.is_contiguous()) return h;
    if (out.dim() == 2 && (h == 1 || out.stride(1) == 1) && out.stride(0) >= h) return out.stride(0);
    value_error(std::string(op) + ": out must have rows of adjacent elements, evenly spaced and apart");
}
// The bytes between a tensor's first and last element.
std::pair<uint64_t, uint64_t> extent(const Tensor& t) {
    if (t.numel() == 0) return {0, 0};
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    const auto from = reinterpret_cast<uint64_t>(t.data_ptr());
    return {from, from + static_cast<uint64_t>(last + 1) * t.element_size()};
}
// The bytes of a row and from row to row, where t is a matrix with rows of adjacent elements; else zeros.
std::pair<uint64_t, uint64_t> row_bytes(const Tensor& t) {
    if (t.dim() != 2 || (t.size(1) != 1 && t.stride(1) != 1)) return {0, 0};
    return {t.size(1) * t.element_size(), t.stride(0) * t.element_size()};
}
// An output must not lie in what is read while it is written. Columns of one array may lie beside each other.
void apart(const char* op, const Tensor& out, const Tensor& in) {
    const auto [a, b] = extent(out);
    const auto [c, d] = extent(in);
    if (a >= d || c >= b) return;
    const auto [out_row, pitch] = row_bytes(out);
    const auto [in_row, in_pitch] = row_bytes(in);
    if (pitch != 0 && pitch == in_pitch) {
        const uint64_t column = c >= a ? (c - a) % pitch : (pitch - (a - c) % pitch) % pitch;  // of in, counted from out's first
        if (column >= out_row && column + in_row <= pitch) return;
    }
    value_error(std::string(op) + ": out must not overlap an input");
}
void* data(const Tensor& t) { return t.numel() == 0 ? nullptr : t.data_ptr(); }
void* data(const Optional& t) { return t ? data(*t) : nullptr; }
// A tensor of the caller's that a kernel writes: autograd must see that it changed.
const Tensor& written(const Tensor& t) {
    t.unsafeGetTensorImpl()->bump_version();
    return t;
}
Tensor bytes(const Tensor& like, size_t n) {
    return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

// Calls f(stream) with the device current and without the interpreter's lock, and raises what the
// library says when it refuses.
template <typename F>
void launch(int device, F&& f) {
    int rc = 0;
    const auto call = [&] {
        void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
        Py_BEGIN_ALLOW_THREADS rc = f(stream);
        Py_END_ALLOW_THREADS
    };
    if (c10::cuda::current_device() == device) {
        call();
    } else {
        const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
        call();
    }
    if (rc != 0) throw Refusal{PyExc_RuntimeError, bcclGetLastError()};
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const Optional& t) { return t ? THPVariable_Wrap(*t) : Py_NewRef(Py_None); }
template <typename... T>
PyObject* wrap_all(const T&... t) {
    PyObject* r = PyTuple_New(sizeof...(T));
    if (r == nullptr) return nullptr;
    Py_ssize_t i = 0;
    bool ok = true;
    const auto put = [&](PyObject* o) {
        ok = ok && o != nullptr;
        PyTuple_SET_ITEM(r, i++, o);
    };
    (put(wrap(t)), ...);
    if (ok) return r;
    Py_DECREF(r);
    return nullptr;
}

// ---------------------------------------------------------------- norms
struct NormOperands {
    int code, wcode = 0;
    int64_t h, rows;
    Optional weight, bias;
    NormOperands(const char* op, const Tensor& x, const Optional& w, const Optional& b) : code(float_code(op, "input", x)) {
        h = x.dim() > 0 ? x.size(-1) : 0;
        if (h < 1)
            value_error(std::string(op) + ": input needs a last dimension of at least 1, got shape " + shape_of(x));
        rows = x.numel() / h;
        if (!w) {
            if (b) type_error(std::string(op) + ": bias needs a weight of its own type");
            return;
        }
        wcode = like_or_f32(op, "weight", *w, x.scalar_type());
        const auto vector = [&](const char* what, const Tensor& p) {
            if (p.dim() != 1 || p.size(0) != h)
                value_error(std::string(op) + ": " + what + " must have shape (" + std::to_string(h) + ",), got " + shape_of(p));
            return p.contiguous();
        };
        weight = vector("weight", *w);
        if (b) {
            if (b->scalar_type() != w->scalar_type()) type_error(std::string(op) + ": bias needs a weight of its own type");
            bias = vector("bias", *b);
        }
    }
};

// norm_forward(kind, x, weight, bias, eps, out) -> (y, mean, rstd), without the mean for RMS norm (kind 1)
PyObject* NormForward(PyObject* const* a) {
    const int kind = static_cast<int>(integer(a[0]));
    const char* op = kind == 0 ? "layer_norm" : "rms_norm";
    const Tensor& x = tensor(op, "input", a[1]);
    const NormOperands o(op, x, optional_tensor(op, "weight", a[2]), optional_tensor(op, "bias", a[3]));
    const double eps = number(a[4]);
    const Optional given = optional_tensor(op, "out", a[5]);
    if (!(eps >= 0.0)) value_error(std::string(op) + ": eps must not be negative or NaN");
    const int device = one_device(op, x, o.weight, o.bias, given);
    const Rows xr(x, o.h);
    // In place is fine: a row is read before it is written.
    if (given && !(given->data_ptr() == x.data_ptr() && given->strides() == x.strides())) apart(op, *given, x);
    if (given && o.weight) apart(op, *given, *o.weight);
    if (given && o.bias) apart(op, *given, *o.bias);
    const int64_t stride = given ? out_rows(op, *given, x.sizes(), x.scalar_type()) : o.h;
    const Tensor y = given ? written(*given) : at::empty(x.sizes(), x.options());
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const auto f32 = x.options().dtype(at::kFloat);
    const Optional mean = kind == 0 ? Optional(at::empty(lead, f32)) : std::nullopt;
    const Tensor rstd = at::empty(lead, f32);
    launch(device, [&](void* s) {
        return bcclNormForward(kind, data(xr.t), xr.stride, data(o.weight), data(o.bias), data(y), stride,
                               static_cast<float*>(data(mean)), static_cast<float*>(data(rstd)), o.rows, o.h,
                               static_cast<float>(eps), o.code, o.wcode, s);
    });
    return kind == 0 ? wrap_all(y, mean, rstd) : wrap_all(y, rstd);
}

// norm_backward(kind, dy, x, mean, rstd, weight, weight_grad, bias_grad) -> (dx, dweight, dbias), without
// the last for RMS norm
PyObject* NormBackward(PyObject* const* a) {
    const int kind = static_cast<int>(integer(a[0]));
    const char* op = kind == 0 ? "layer_norm_backward" : "rms_norm_backward";
    const Tensor &dy = tensor(op, "dy", a[1]), &x = tensor(op, "input", a[2]);
    const Optional mean = optional_tensor(op, "mean", a[3]);
    const Tensor& rstd = tensor(op, "rstd", a[4]);
    const NormOperands o(op, x, optional_tensor(op, "weight", a[5]), std::nullopt);
    const bool need_dw = o.weight && truth(a[6]), need_db = o.weight && truth(a[7]);
    if (dy.scalar_type() != x.scalar_type() || dy.sizes() != x.sizes())
        value_error(std::string(op) + ": dy must be " + type_of(x.scalar_type()) + " of shape " + shape_of(x) + ", got " +
                    type_of(dy.scalar_type()) + " " + shape_of(dy));
    const auto statistic = [&](const char* what, const Tensor& t) {
        if (t.scalar_type() != at::kFloat || t.sizes() != x.sizes().slice(0, x.dim() - 1) || !t.is_contiguous())
            value_error(std::string(op) + ": " + what + " must be the contiguous float32 tensor that the forward pass returned");
    };
    if (kind == 0 && !mean) value_error(std::string(op) + ": mean must be the tensor that the forward pass returned");
    if (mean) statistic("mean", *mean);
    statistic("rstd", rstd);
    const int device = one_device(op, x, dy, mean, rstd, o.weight);
    const Rows xr(x, o.h), dyr(dy, o.h);
    const Tensor dx = at::empty(x.sizes(), x.options());
    const Optional dw = need_dw ? Optional(at::empty({o.h}, o.weight->options())) : std::nullopt;
    const Optional db = need_db ? Optional(at::empty({o.h}, o.weight->options())) : std::nullopt;
    const size_t size = need_dw || need_db ? bcclNormBackwardWorkspace(kind, o.rows, o.h, o.code) : 0;
    const Optional ws = size > 0 ? Optional(bytes(x, size)) : std::nullopt;
    launch(device, [&](void* s) {
        return bcclNormBackward(kind, data(dyr.t), dyr.stride, data(xr.t), xr.stride, static_cast<const float*>(data(mean)),
                                static_cast<const float*>(data(rstd)), data(o.weight), data(dx), o.h, data(dw), data(db),
                                o.rows, o.h, o.code, o.wcode, data(ws), size, s);
    });
    return kind == 0 ? wrap_all(dx, dw, db) : wrap_all(dx, dw);
}

// ---------------------------------------------------------------- embedding
int64_t first_row(const char* op, PyObject* o) {
    const int64_t first = integer(o);
    if (first < 0) value_error(std::string(op) + ": first_row must not be negative, got " + std::to_string(first));
    return first;
}

// embedding_forward(ids, weight, scale, first_row, out) -> rows
PyObject* EmbeddingForward(PyObject* const* a) {
    const char* op = "embedding";
    const Tensor &ids = tensor(op, "ids", a[0]), &weight = tensor(op, "weight", a[1]);
    const int code = float_code(op, "weight", weight), icode = int_code(op, "ids", ids);
    const float scale = static_cast<float>(number(a[2]));
    const int64_t first = first_row(op, a[3]);
    const Optional given = optional_tensor(op, "out", a[4]);
    if (weight.dim() != 2 || weight.size(1) < 1)
        value_error(std::string(op) + ": weight must be 2-D, got shape " + shape_of(weight));
    const int device = one_device(op, weight, ids, given);
    const int64_t h = weight.size(1);
    at::DimVector shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(h);
    if (given) apart(op, *given, weight);
    if (given) apart(op, *given, ids);
    const int64_t stride = given ? out_rows(op, *given, shape, weight.scalar_type()) : h;
    const Tensor out = given ? written(*given) : at::empty(shape, weight.options()), i = ids.contiguous();
    const Rows w(weight, h);
    launch(device, [&](void* s) {
        return bcclEmbeddingForward(data(i), icode, i.numel(), data(w.t), w.stride, weight.size(0), h, first, scale, data(out),
                                    stride, code, s);
    });
    return wrap(out);
}

// embedding_backward(dy, ids, num_rows, scale, first_row, padding_idx, out, accumulate) -> the table's gradient
PyObject* EmbeddingBackward(PyObject* const* a) {
    const char* op = "embedding_backward";
    const Tensor &dy = tensor(op, "dy", a[0]), &ids = tensor(op, "ids", a[1]);
    const int code = float_code(op, "dy", dy), icode = int_code(op, "ids", ids);
    const int64_t rows = integer(a[2]);
    const float scale = static_cast<float>(number(a[3]));
    const int64_t first = first_row(op, a[4]);
    const bool has_skip = a[5] != Py_None;
    const int64_t skip = has_skip ? integer(a[5]) : 0;
    const Optional given = optional_tensor(op, "out", a[6]);
    const bool accumulate = truth(a[7]);
    if (dy.dim() < 1 || dy.size(-1) < 1 || dy.sizes().slice(0, dy.dim() - 1) != ids.sizes())
        value_error(std::string(op) + ": dy " + shape_of(dy) + " must be one row per id, ids " + shape_of(ids));
    if (rows < 0 || skip < 0) value_error(std::string(op) + ": num_rows and padding_idx must not be negative");
    if (accumulate && !given) value_error(std::string(op) + ": accumulate needs out");
    const int device = one_device(op, dy, ids, given);
    const int64_t h = dy.size(-1);
    if (given && (given->sizes() != at::IntArrayRef({rows, h}) || !given->is_contiguous()))
        value_error(std::string(op) + ": out must be a contiguous " + shape_of({rows, h}) + " tensor, got " + shape_of(*given));
    if (given) apart(op, *given, dy);
    if (given) apart(op, *given, ids);
    const int ocode = given ? like_or_f32(op, "out", *given, dy.scalar_type()) : code;
    const Tensor out = given ? written(*given) : at::empty({rows, h}, dy.options());
    const Tensor i = ids.contiguous();
    const Rows d(dy, h);
    const size_t size = bcclEmbeddingBackwardWorkspace(i.numel(), rows, h);
    const Optional ws = size > 0 ? Optional(bytes(dy, size)) : std::nullopt;
    launch(device, [&](void* s) {
        return bcclEmbeddingBackward(data(d.t), d.stride, data(i), icode, i.numel(), data(out), rows, h, first, scale, skip,
                                     has_skip, accumulate, code, ocode, data(ws), size, s);
    });
    return wrap(out);
}

// ---------------------------------------------------------------- experts
// expert_sort(ids, experts) -> (slots, sources, offsets)
PyObject* ExpertSort(PyObject* const* a) {
    const char* op = "sort_by_expert";
    const Tensor& ids = tensor(op, "expert_ids", a[0]);
    const int icode = int_code(op, "expert_ids", ids);
    const int64_t experts = integer(a[1]);
    if (ids.dim() != 1 && ids.dim() != 2)
        value_error(std::string(op) + ": expert_ids must be [tokens, top], got shape " + shape_of(ids));
    const int64_t tokens = ids.size(0), top = ids.dim() == 2 ? ids.size(1) : 1;
    if (top < 1 || top > BCCL_MAX_TOP)
        value_error(std::string(op) + ": 1 to " + std::to_string(BCCL_MAX_TOP) + " experts per token, got " + std::to_string(top));
    if (experts < 1 || experts > BCCL_MAX_EXPERTS)
        value_error(std::string(op) + ": 1 to " + std::to_string(BCCL_MAX_EXPERTS) + " experts, got " + std::to_string(experts));
    const int device = one_device(op, ids);
    const Tensor i = ids.contiguous();
    const auto i32 = ids.options().dtype(at::kInt);
    const Tensor slots = at::empty({tokens, top}, i32), sources = at::empty({tokens * top}, i32),
                 offsets = at::empty({experts + 1}, i32);
    const size_t size = bcclExpertSortWorkspace(tokens, static_cast<int>(top));
    const Optional ws = size > 0 ? Optional(bytes(ids, size)) : std::nullopt;
    launch(device, [&](void* s) {
        return bcclExpertSort(data(i), icode, tokens, static_cast<int>(top), static_cast<int>(experts),
                              static_cast<int32_t*>(data(slots)), static_cast<int32_t*>(data(sources)),
                              static_cast<int32_t*>(data(offsets)), data(ws), size, s);
    });
    return wrap_all(slots, sources, offsets);
}

// The tensors of an ExpertOrder, which its constructor has checked.
struct Order {
    const Tensor& slots;
    const Tensor& offsets;
    int64_t tokens, n;
    int top, experts;
    Order(const char* op, PyObject* s, PyObject* o)
        : slots(tensor(op, "order", s)), offsets(tensor(op, "order", o)), tokens(slots.size(0)), n(slots.numel()),
          top(static_cast<int>(slots.size(1))), experts(static_cast<int>(offsets.size(0) - 1)) {}
    const int32_t* slot() const { return static_cast<const int32_t*>(data(slots)); }
    const int32_t* offset() const { return static_cast<const int32_t*>(data(offsets)); }
};
int64_t width_of(const char* op, const char* what, const Tensor& t, int64_t n) {
    if (t.dim() != 2 || t.size(0) != n || t.size(1) < 1)
        value_error(std::string(op) + ": " + what + " must be [" + std::to_string(n) + ", h], got shape " + shape_of(t));
    return t.size(1);
}
struct Weights {
    Optional w;
    int code;
    Weights(const char* op, PyObject* o, const Order& order, const Tensor& rows, int rows_code)
        : w(optional_tensor(op, "weights", o)), code(rows_code) {
        if (!w) return;
        code = like_or_f32(op, "weights", *w, rows.scalar_type());
        if (w->sizes() != order.slots.sizes())
            value_error(std::string(op) + ": weights must be " + shape_of(order.slots) + ", got " + shape_of(*w));
        w = w->contiguous();
    }
};

// dispatch(x, slots, offsets, out) -> rows
PyObject* Dispatch(PyObject* const* a) {
    const char* op = "dispatch";
    const Tensor& x = tensor(op, "input", a[0]);
    const int code = float_code(op, "input", x);
    const Order o(op, a[1], a[2]);
    const Optional given = optional_tensor(op, "out", a[3]);
    const int64_t h = width_of(op, "input", x, o.tokens);
    const int device = one_device(op, x, o.slots, o.offsets, given);
    if (given && (given->scalar_type() != x.scalar_type() || given->sizes() != at::IntArrayRef({o.n, h}) ||
                  !given->is_contiguous()))
        value_error(std::string(op) + ": out must be a contiguous " + type_of(x.scalar_type()) + " tensor of shape " +
                    shape_of({o.n, h}) + ", got " + type_of(given->scalar_type()) + " " + shape_of(*given));
    if (given) apart(op, *given, x);
    const Tensor rows = given ? written(*given) : at::empty({o.n, h}, x.options());
    const Rows xr(x, h);
    launch(device, [&](void* s) {
        return bcclExpertDispatch(data(xr.t), xr.stride, o.slot(), o.offset(), o.tokens, o.top, o.experts, h, data(rows), code,
                                  s);
    });
    return wrap(rows);
}

// combine(rows, slots, offsets, weights) -> y
PyObject* Combine(PyObject* const* a) {
    const char* op = "combine";
    const Tensor& given = tensor(op, "rows", a[0]);
    const int code = float_code(op, "rows", given);
    const Order o(op, a[1], a[2]);
    const int64_t h = width_of(op, "rows", given, o.n);
    const Weights w(op, a[3], o, given, code);
    const int device = one_device(op, given, o.slots, o.offsets, w.w);
    const Tensor rows = given.contiguous(), y = at::empty({o.tokens, h}, given.options());
    launch(device, [&](void* s) {
        return bcclExpertCombine(data(rows), o.slot(), data(w.w), w.code, o.tokens, o.top, h, data(y), h, code, s);
    });
    return wrap(y);
}

// combine_backward(dy, rows, slots, offsets, weights, weight_grad) -> (drows, dweights)
PyObject* CombineBackward(PyObject* const* a) {
    const char* op = "combine_backward";
    const Tensor &dy = tensor(op, "dy", a[0]), &given = tensor(op, "rows", a[1]);
    const int code = float_code(op, "dy", dy);
    const Order o(op, a[2], a[3]);
    const int64_t h = width_of(op, "dy", dy, o.tokens);
    if (width_of(op, "rows", given, o.n) != h || given.scalar_type() != dy.scalar_type())
        value_error(std::string(op) + ": rows must be " + type_of(dy.scalar_type()) + " of width " + std::to_string(h) + ", got " +
                    type_of(given.scalar_type()) + " " + shape_of(given));
    const Weights w(op, a[4], o, dy, code);
    const int device = one_device(op, dy, given, o.slots, o.offsets, w.w);
    const Tensor rows = given.contiguous(), drows = at::empty({o.n, h}, dy.options());
    const Rows d(dy, h);
    const Optional dw = w.w && truth(a[5]) ? Optional(at::empty(w.w->sizes(), w.w->options())) : std::nullopt;
    launch(device, [&](void* s) {
        return bcclExpertCombineBackward(data(d.t), d.stride, data(rows), o.slot(), o.offset(), data(w.w), w.code, o.tokens,
                                         o.top, o.experts, h, data(drows), data(dw), code, s);
    });
    return wrap_all(drows, dw);
}

// ---------------------------------------------------------------- gradients
// Elements fill t's memory without gaps or overlaps, in some order of the dimensions.
bool dense(const Tensor& t) {
    if (t.is_contiguous()) return true;
    at::SmallVector<std::pair<int64_t, int64_t>, 8> dims;
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) != 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t n = 1;
    for (const auto& [stride, size] : dims) {
        if (stride != n) return false;
        n *= size;
    }
    return true;
}

struct Gradients {
    const char* op;
    int device = -1;
    Tensor like;
    // By type of gradient and output, and by whether other ranks hold the same: pointers and counts.
    struct Group {
        int code, out_code;
        bool replicated;
        uint64_t total = 0;
        std::vector<const void*> in;
        std::vector<void*> out;
        std::vector<size_t> count;
    };
    std::vector<Group> groups;
    double world;

    // replicated: None, or a list that says for each gradient whether all of `ranks` ranks hold the same.
    Gradients(const char* name, PyObject* grads, PyObject* outs, bool written, PyObject* replicated, int64_t ranks)
        : op(name), world(static_cast<double>(ranks)) {
        const Py_ssize_t n = PyList_Check(grads) ? PyList_GET_SIZE(grads) : 0;
        if (n == 0) value_error(std::string(op) + ": no gradients");
        const bool marked = replicated != Py_None;
        if (marked && (!PyList_Check(replicated) || PyList_GET_SIZE(replicated) != n || ranks < 1))
            value_error(std::string(op) + ": replicated must say yes or no for each gradient");
        const bool apart = outs != Py_None;
        if (apart && (!PyList_Check(outs) || PyList_GET_SIZE(outs) != n))
            value_error(std::string(op) + ": outs must be a tensor for each gradient");
        struct Range {
            uint64_t from, to;
            bool written;
        };
        std::vector<Range> ranges;
        if (written) ranges.reserve(static_cast<size_t>(apart ? 2 * n : n));
        const auto range = [&](const void* at, int64_t count, int code, bool w) {
            const auto p = reinterpret_cast<uint64_t>(at);
            ranges.push_back({p, p + static_cast<uint64_t>(count) * static_cast<uint64_t>(size_of(code)), w});
        };
        bool elsewhere = false;  // an output that is not its gradient
        for (Py_ssize_t i = 0; i < n; ++i) {
            const Tensor& t = strided(op, "each gradient", PyList_GET_ITEM(grads, i));
            const Tensor& o = apart ? strided(op, "each out", PyList_GET_ITEM(outs, i)) : t;
            const int code = float_code(op, "each gradient", t);
            if (i == 0) {
                device = one_device(op, t);
                like = t;
            }
            if (!t.is_cuda() || t.get_device() != device || !o.is_cuda() || o.get_device() != device)
                value_error(std::string(op) + ": gradients and outs must be CUDA tensors on one device");
            int out_code = code;
            if (!dense(t))
                value_error(std::string(op) + ": gradients must be dense in memory, got shape " + shape_of(t) + ", strides " +
                            shape_of(t.strides()));
            if (apart) {
                out_code = like_or_f32(op, "each out", o, t.scalar_type());
                if (o.sizes() != t.sizes() || (o.strides() != t.strides() && !(o.is_contiguous() && t.is_contiguous())))
                    value_error(std::string(op) + ": each out must have its gradient's shape and layout");
            }
            const int64_t count = t.numel();
            if (count == 0) continue;
            void* out = o.mutable_data_ptr();  // first: it may move a lazily copied gradient, in place
            const void* in = t.const_data_ptr();
            if (in == nullptr) no_storage(op, "each gradient");
            if (out == nullptr) no_storage(op, "each out");
            const bool same = marked && truth(PyList_GET_ITEM(replicated, i));
            const auto fits = [&](const Group& g) { return g.code == code && g.out_code == out_code && g.replicated == same; };
            if (groups.empty() || !fits(groups.back())) {
                const auto found = std::find_if(groups.begin(), groups.end(), fits);
                if (found == groups.end()) {
                    groups.push_back({code, out_code, same, 0, {}, {}, {}});
                    groups.back().in.reserve(static_cast<size_t>(n));
                    groups.back().out.reserve(static_cast<size_t>(n));
                    groups.back().count.reserve(static_cast<size_t>(n));
                } else {
                    std::iter_swap(found, groups.end() - 1);
                }
            }
            Group& g = groups.back();
            g.in.push_back(in);
            g.out.push_back(out);
            g.count.push_back(static_cast<size_t>(count));
            g.total += static_cast<uint64_t>(count);
            if (!written) continue;
            range(out, count, out_code, true);
            if (out != in || out_code != code) elsewhere = true;
            if (apart) range(in, count, code, false);
        }
        if (!written) return;
        check_apart(ranges, elsewhere);
        for (Py_ssize_t i = 0; i < n; ++i) ::written(THPVariable_Unpack(PyList_GET_ITEM(apart ? outs : grads, i)));
    }

    // No tensor written overlaps another one, nor (outputs in memory of their own) any that is read.
    template <typename R>
    void check_apart(std::vector<R>& ranges, bool elsewhere) const {
        if (!elsewhere)
            ranges.erase(std::remove_if(ranges.begin(), ranges.end(), [](const R& r) { return !r.written; }), ranges.end());
        std::sort(ranges.begin(), ranges.end(), [](const R& a, const R& b) { return a.from < b.from; });
        uint64_t any = 0, written = 0;  // ends of the ranges so far
        for (const R& x : ranges) {
            if (x.from < (x.written ? any : written))
                value_error(std::string(op) + ": tensors to be written overlap");
            any = std::max(any, x.to);
            if (x.written) written = std::max(written, x.to);
        }
    }

    // What this rank adds to the sum over all ranks: where all hold the same, its share of the squares.
    Tensor squares() const {
        const Tensor total = squares(false);
        if (std::any_of(groups.begin(), groups.end(), [](const Group& g) { return g.replicated; }))
            total.add_(squares(true), 1.0 / world);
        return total;
    }
    Tensor squares(bool replicated) const {
        const Tensor total = at::empty({1}, like.options().dtype(at::kDouble));
        std::vector<Tensor> keep;
        bool accumulate = false;
        const auto run = [&](const void* const* in, const size_t* count, int n, int code, uint64_t elements) {
            const size_t size = BCCL_GRAD_WORKSPACE(elements, n);
            keep.push_back(bytes(like, size));
            void* ws = keep.back().data_ptr();
            launch(device, [&](void* s) {
                return bcclGradSquares(in, count, n, code, accumulate, static_cast<double*>(total.data_ptr()), ws, size, s);
            });
            accumulate = true;
        };
        for (const Group& g : groups)
            if (g.replicated == replicated) run(g.in.data(), g.count.data(), static_cast<int>(g.in.size()), g.code, g.total);
        if (!accumulate) run(nullptr, nullptr, 0, 0, 0);
        return total;
    }

    Tensor clip(const Tensor& total, double max_norm, double eps) const {
        const Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
        float* to = static_cast<float*>(norm.data_ptr());
        const auto run = [&](const void* const* in, void* const* out, const size_t* count, int n, int code, int out_code) {
            launch(device, [&](void* s) {
                return bcclGradClip(in, out, count, n, code, out_code, static_cast<const double*>(total.data_ptr()),
                                    static_cast<float>(max_norm), static_cast<float>(eps), to, s);
            });
            to = nullptr;
        };
        for (const Group& g : groups)
            run(g.in.data(), g.out.data(), g.count.data(), static_cast<int>(g.in.size()), g.code, g.out_code);
        if (groups.empty()) run(nullptr, nullptr, nullptr, 0, 0, 0);
        return norm;
    }
};

// grad_squares(grads, replicated, ranks) -> this rank's part of the sum of squares, a float64 tensor of one element
PyObject* GradSquares(PyObject* const* a) {
    return wrap(Gradients("grad_norm", a[0], Py_None, false, a[1], integer(a[2])).squares());
}

// grad_norm_of(grads[0], total) -> the norm
PyObject* GradNormOf(PyObject* const* a) {
    const Tensor &like = tensor("grad_norm", "gradient", a[0]), &total = tensor("grad_norm", "total", a[1]);
    const int device = one_device("grad_norm", like, total);
    const Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
    launch(device, [&](void* s) {
        return bcclGradClip(nullptr, nullptr, nullptr, 0, 0, 0, static_cast<const double*>(total.data_ptr()), 0.0f, 0.0f,
                            static_cast<float*>(norm.data_ptr()), s);
    });
    return wrap(norm);
}

// grad_clip(grads, outs, max_norm, eps, replicated, ranks, reduce) -> the norm from before. reduce (None or a
// function) is called on this rank's part of the sum of squares between the two passes.
PyObject* GradClip(PyObject* const* a) {
    const double max_norm = number(a[2]), eps = number(a[3]);
    const Gradients g("clip_grad_norm", a[0], a[1], true, a[4], integer(a[5]));
    const Tensor total = g.squares();
    if (a[6] != Py_None) {
        PyObject* t = wrap(total);
        if (t == nullptr) return nullptr;
        PyObject* done = PyObject_CallOneArg(a[6], t);
        Py_DECREF(t);
        if (done == nullptr) return nullptr;
        Py_DECREF(done);
    }
    return wrap(g.clip(total, max_norm, eps));
}

// ---------------------------------------------------------------- captures
// leaf_stream(leaf) -> the CUDA stream on which its accumulation node was made, as an integer; None without a
// node that lives, or without a stream (host tensors)
PyObject* LeafStream(PyObject* const* a) {
    if (!THPVariable_Check(a[0])) type_error("leaf_stream: a tensor is needed");
    const auto node = torch::autograd::impl::try_get_grad_accumulator(THPVariable_Unpack(a[0]));
    const auto stream = node ? node->stream() : std::nullopt;
    if (!stream || stream->device_type() != c10::DeviceType::CUDA) return Py_NewRef(Py_None);
    return PyLong_FromUnsignedLongLong(reinterpret_cast<uintptr_t>(c10::cuda::CUDAStream(*stream).stream()));
}

// ---------------------------------------------------------------- the module
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        const at::AutoDispatchBelowADInplaceOrView below_autograd;  // outputs and copies record no graph
        return F(args);
    } catch (const Refusal& r) {
        if (r.type != nullptr) PyErr_SetString(r.type, r.what.c_str());
    } catch (...) {  // torch's own: an allocation that fails is a torch.OutOfMemoryError, as from torch's operators
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
constexpr PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<NormForward, 6>("norm_forward"),
                         method<NormBackward, 8>("norm_backward"),
                         method<EmbeddingForward, 5>("embedding_forward"),
                         method<EmbeddingBackward, 8>("embedding_backward"),
                         method<ExpertSort, 2>("expert_sort"),
                         method<Dispatch, 4>("dispatch"),
                         method<Combine, 4>("combine"),
                         method<CombineBackward, 6>("combine_backward"),
                         method<GradSquares, 3>("grad_squares"),
                         method<GradNormOf, 2>("grad_norm_of"),
                         method<GradClip, 7>("grad_clip"),
                         method<LeafStream, 1>("leaf_stream"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }

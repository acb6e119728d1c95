// Checks of arguments that the host calls of the serving operators share: what a
// plain GPU tensor is, whether views share memory, numbers and integers of a call,
// exceptions turned into Python's.  In an unnamed namespace of each source.
#pragma once

#include "host_calls.h"

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/clone.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cstdarg>
#include <string>

#include "serving_sizes.h"

namespace {

struct Refusal {
    PyObject* type;
    std::string message;
};

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    char text[320];
    va_list args;
    va_start(args, format);
    vsnprintf(text, sizeof(text), format, args);
    va_end(args);
    throw Refusal{type, text};
}

void check_status(int status) {
    if (status == W4G64_STATUS_OK) return;
    // (what these operators do not support is a matter of shapes and strides)
    PyObject* type = status == W4G64_STATUS_INVALID_DTYPE ? PyExc_TypeError
                     : status == W4G64_STATUS_INVALID_VALUE || status == W4G64_STATUS_WORKSPACE ||
                             status == W4G64_STATUS_UNSUPPORTED
                         ? PyExc_ValueError
                         : PyExc_RuntimeError;
    throw Refusal{type, w4g64_last_error()};
}

void check_count(const char* op, Py_ssize_t count, Py_ssize_t want) {
    if (count != want) refuse(PyExc_TypeError, "%s takes %zd arguments", op, want);
}

// The library is called directly: nothing that follows torch's operators sees it.
void check_state(const char* op) {
    if (c10::impl::TorchDispatchModeTLS::stack_len() || torch::jit::tracer::isTracing() ||
        c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        refuse(PyExc_RuntimeError, "%s cannot run under a dispatch mode, a trace or a function transform", op);
}

// A plain tensor (any device): torch.Tensor itself or a Parameter.
const at::Tensor& tensor(PyObject* obj, const char* op, const char* name, int64_t dims) {
    if (!THPVariable_CheckExact(obj)) refuse(PyExc_TypeError, "%s must be a torch.Tensor (no subclass)", name);
    const at::Tensor& t = THPVariable_Unpack(obj);
    if (!t.defined() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg() ||
        t.unsafeGetTensorImpl()->is_python_dispatch())
        refuse(PyExc_ValueError, "%s must be a plain strided tensor", name);
    if (t.dim() != dims) refuse(PyExc_ValueError, "%s must have %lld dimensions, got %lld", name, (long long)dims, (long long)t.dim());
    if ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined())
        refuse(PyExc_RuntimeError, "%s has no gradient, and %s requires one", op, name);
    return t;
}

void check_dtype(const at::Tensor& t, const char* name, at::ScalarType want, const char* said) {
    if (t.scalar_type() != want) refuse(PyExc_TypeError, "%s must have dtype %s", name, said);
}

void check_shape(const at::Tensor& t, const char* name, std::initializer_list<int64_t> want) {
    if (t.sizes() == at::IntArrayRef(want)) return;
    std::string text;
    for (int64_t n : want) text += (text.empty() ? "" : ", ") + std::to_string(n);
    refuse(PyExc_ValueError, "%s must have shape [%s]", name, text.c_str());
}

c10::Device device_of(std::initializer_list<std::pair<const at::Tensor*, const char*>> all) {
    const c10::Device device = all.begin()->first->device();
    for (const auto& [t, name] : all) {
        if (!t->is_cuda()) refuse(PyExc_ValueError, "%s must be a GPU tensor", name);
        if (t->device() != device) refuse(PyExc_ValueError, "%s must be on the same device as %s", name, all.begin()->second);
    }
    return device;
}

bool aligned(const at::Tensor& t) { return !(((uintptr_t)t.const_data_ptr()) & 15); }

// The stride of a dimension, 0 where it has one entry.
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// Whether rows of `t` (its last dimension) can be read 16 bytes at a time.
bool readable(const at::Tensor& t) {
    if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
    for (int64_t d = 0; d + 1 < t.dim(); ++d)
        if (step(t, d) % 8 || step(t, d) < 0) return false;
    return aligned(t);
}

at::Tensor usable(const at::Tensor& t) { return readable(t) ? t : at::clone(t, at::MemoryFormat::Contiguous); }
at::Tensor contiguous(const at::Tensor& t) { return t.is_contiguous() ? t : at::clone(t, at::MemoryFormat::Contiguous); }

// Whether no two entries share memory (enough: every stride covers the smaller ones).
bool distinct(const at::Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> dims;  // (stride, size)
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t covered = 1;
    for (const auto& [stride, size] : dims) {
        if (stride < covered) return false;
        covered = stride * (size - 1) + covered;
    }
    return true;
}

bool overlap(const at::Tensor& a, const at::Tensor& b) {
    if (!a.numel() || !b.numel()) return false;
    auto range = [](const at::Tensor& t) {
        int64_t span = 1;
        for (int64_t d = 0; d < t.dim(); ++d) span += (t.size(d) - 1) * t.stride(d);
        const char* at = (const char*)t.const_data_ptr();
        return std::make_pair(at, at + span * t.element_size());
    };
    const auto x = range(a), y = range(b);
    return x.first < y.second && y.first < x.second;
}

// Whether an entry of one view is one of the other: two addresses meet where the
// offset is a sum of strides, each as often as its dimension's indices can differ
// (a.size - 1 to -(b.size - 1)).  Dimensions go by falling strides; what is left
// after one has to lie within what the smaller ones span.
struct Dim {
    int64_t stride, up, down;
};
bool meets(const Dim* dim, int count, int64_t offset) {
    if (!count) return offset == 0;
    int64_t up = 0, down = 0;  // of the smaller strides
    for (int i = 1; i < count; ++i) up += dim[i].stride * dim[i].up, down += dim[i].stride * dim[i].down;
    const int64_t s = dim->stride;
    auto below = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };  // (rounded down)
    const int64_t from = std::max(-below(up - offset, s), -dim->down), to = std::min(below(offset + down, s), dim->up);
    if (to - from > 8) return true;  // (strides that do not nest: not told apart)
    for (int64_t n = from; n <= to; ++n)
        if (meets(dim + 1, count - 1, offset - n * s)) return true;
    return false;
}

// Whether two views may share memory: told exactly where they have the same strides
// (parts of one buffer), else by their ranges.
bool share(const at::Tensor& a, const at::Tensor& b) {
    if (!overlap(a, b)) return false;
    const int64_t bytes = (const char*)b.const_data_ptr() - (const char*)a.const_data_ptr();
    if (a.dim() != b.dim() || a.dim() > 5 || a.scalar_type() != b.scalar_type() || bytes % a.element_size()) return true;
    Dim dims[5];
    int count = 0;
    for (int64_t d = 0; d < a.dim(); ++d) {
        const int64_t x = step(a, d), y = step(b, d);
        if (a.size(d) > 1 && b.size(d) > 1 && x != y) return true;
        if (x + y) dims[count++] = Dim{std::max(x, y), a.size(d) - 1, b.size(d) - 1};
    }
    std::sort(dims, dims + count, [](const Dim& l, const Dim& r) { return l.stride > r.stride; });
    return meets(dims, count, bytes / a.element_size());
}

bool same_view(const at::Tensor& a, const at::Tensor& b) {
    return a.const_data_ptr() == b.const_data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// Whether two row tensors lie apart: told by share(), or, where their heads lie at
// other strides (parts of a fused projection), rows equally far from each other and
// within a row one behind the other.
bool apart(const at::Tensor& a, const at::Tensor& b) {
    if (!share(a, b)) return true;
    const at::Tensor& x = a.const_data_ptr() <= b.const_data_ptr() ? a : b;
    const at::Tensor& y = &x == &a ? b : a;
    const int64_t between = ((const char*)y.const_data_ptr() - (const char*)x.const_data_ptr()) / x.element_size();
    auto extent = [](const at::Tensor& t) { return (t.size(1) - 1) * step(t, 1) + t.size(2); };
    return x.size(0) > 1 && x.stride(0) == y.stride(0) && between >= extent(x) && between + extent(y) <= x.stride(0);
}

void check_output(const at::Tensor& out, const at::Tensor& q) {
    if (out.scalar_type() != q.scalar_type()) refuse(PyExc_TypeError, "out must have q's dtype");
    if (out.sizes() != q.sizes()) refuse(PyExc_ValueError, "out must have q's shape");
    if (out.numel() && (!readable(out) || !distinct(out)))
        refuse(PyExc_ValueError, "out must be 16-byte aligned with a contiguous last dimension, other strides multiples of 8");
}

void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

double number(PyObject* obj, const char* name) {
    if (THPVariable_Check(obj)) refuse(PyExc_TypeError, "%s must be a number, not a tensor", name);
    const double v = PyFloat_AsDouble(obj);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(PyExc_TypeError, "%s must be a number", name);
    }
    return v;
}

int64_t whole(PyObject* obj, const char* name) {
    if (!PyIndex_Check(obj) || PyBool_Check(obj) || THPVariable_Check(obj))  // (a tensor's would wait for the GPU)
        refuse(PyExc_TypeError, "%s must be an integer", name);
    PyObject* index = PyNumber_Index(obj);
    const long long v = index ? PyLong_AsLongLong(index) : -1;
    Py_XDECREF(index);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(PyExc_ValueError, "%s is out of range", name);
    }
    return v;
}

// Runs `call` with its exceptions turned into Python's.
template <class F>
PyObject* guarded(F call) {
    try {
        return call();
    } catch (const Refusal& r) {
        PyErr_SetString(r.type, r.message.c_str());
    } catch (...) {  // as torch's own bindings raise it (an allocation that failed)
        if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// The library's call without the interpreter's lock.
template <class F>
void released(F call) {
    PyThreadState* save = PyEval_SaveThread();
    const int status = call();
    PyEval_RestoreThread(save);
    check_status(status);
}

hipStream_t current_stream(c10::Device device) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream();
}

}  // namespace

// Host side of the paged serving operators (qwen_int4_hip.paged), in the module
// qwen_int4_hip._host: checks of the arguments, outputs and workspace, and the
// call into the C ABI.  There is no other route: what these refuse raises.
//
// Workspaces come from torch's allocator for each call and go back to it with
// the call's stream order, so that two captured graphs never share one.
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

#include "../../include/qwen2_decode.h"

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
    if (a.dim() != b.dim() || a.dim() > 4 || a.scalar_type() != b.scalar_type() || bytes % a.element_size()) return true;
    Dim dims[4];
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

// The cache arguments, checked but for their device; the index tensors made
// contiguous (and kept alive) here.
struct Cache {
    const at::Tensor &k, &v, &table_arg, &cu_arg, &lengths_arg;
    at::Tensor table, cu, lengths;
    qwen2_paged_cache c{};

    Cache(const char* op, PyObject* const* args)
        : k(tensor(args[0], op, "k_pages", 4)),
          v(tensor(args[1], op, "v_pages", 4)),
          table_arg(tensor(args[2], op, "page_table", 2)),
          cu_arg(tensor(args[3], op, "cu_rows", 1)),
          lengths_arg(tensor(args[4], op, "lengths", 1)) {
        if (k.scalar_type() != at::kBFloat16 && k.scalar_type() != at::kHalf)
            refuse(PyExc_TypeError, "k_pages must have dtype torch.bfloat16 or torch.float16");
        if (v.scalar_type() != k.scalar_type()) refuse(PyExc_TypeError, "v_pages must have the dtype of k_pages");
        if (v.sizes() != k.sizes()) refuse(PyExc_ValueError, "v_pages must have the shape of k_pages");
        if (!k.size(0) || !k.size(1)) refuse(PyExc_ValueError, "k_pages must hold at least one page and one head");
        check_dtype(table_arg, "page_table", at::kInt, "torch.int32");
        check_dtype(cu_arg, "cu_rows", at::kInt, "torch.int32");
        check_dtype(lengths_arg, "lengths", at::kInt, "torch.int32");
        check_shape(cu_arg, "cu_rows", {table_arg.size(0) + 1});
        check_shape(lengths_arg, "lengths", {table_arg.size(0)});
        if (!table_arg.size(1)) refuse(PyExc_ValueError, "page_table must have at least one column");
        for (const at::Tensor* t : {&k, &v})
            if (t->numel() && (!readable(*t) || !distinct(*t)))
                refuse(PyExc_ValueError, "%s must be 16-byte aligned with a contiguous last dimension, other strides "
                       "multiples of 8, and no two entries in one place", t == &k ? "k_pages" : "v_pages");
        if (share(k, v))
            refuse(PyExc_ValueError, "k_pages and v_pages must not share memory");
        c.num_pages = k.size(0), c.kv_heads = k.size(1), c.page_size = k.size(2), c.head_dim = k.size(3);
        c.k_page = step(k, 0), c.k_head = step(k, 1), c.k_position = step(k, 2);
        c.v_page = step(v, 0), c.v_head = step(v, 1), c.v_position = step(v, 2);
        c.table_width = table_arg.size(1);
        c.batch = table_arg.size(0);
        c.dtype = k.scalar_type() == at::kHalf ? W4G64_DTYPE_F16 : W4G64_DTYPE_BF16;
    }

    // (on the current device: copies what is not laid out as the library reads it)
    void bind() {
        table = table_arg.size(1) > 1 && table_arg.stride(1) != 1 ? at::clone(table_arg, at::MemoryFormat::Contiguous)
                                                                  : table_arg;
        cu = contiguous(cu_arg), lengths = contiguous(lengths_arg);
        c.k = k.mutable_data_ptr(), c.v = v.mutable_data_ptr();
        c.page_table = (const int32_t*)table.const_data_ptr();
        c.table_stride = table.stride(0);
        c.cu_rows = (const int32_t*)cu.const_data_ptr();
        c.lengths = (const int32_t*)lengths.const_data_ptr();
    }
};

qwen2_rows rows_of(const at::Tensor& t) { return qwen2_rows{const_cast<void*>(t.const_data_ptr()), step(t, 0), step(t, 1)}; }

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

// (q, k, v, k_pages, v_pages, page_table, cu_rows, lengths, inv_freq or None,
// interleaved, rotary_scale, out or None) -> the rotated queries
PyObject* host_paged_append(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "paged_append_hip";
        check_count(op, count, 12);
        check_state(op);
        const at::Tensor& q = tensor(args[0], op, "q", 3);
        const at::Tensor& k = tensor(args[1], op, "k", 3);
        const at::Tensor& v = tensor(args[2], op, "v", 3);
        Cache cache(op, args + 3);
        const at::Tensor* inv = args[8] == Py_None ? nullptr : &tensor(args[8], op, "inv_freq", 1);
        const at::Tensor* given = args[11] == Py_None ? nullptr : &tensor(args[11], op, "out", 3);
        const int interleaved = PyObject_IsTrue(args[9]);
        if (interleaved < 0) return nullptr;
        const double scale = number(args[10], "rotary_scale");
        const int64_t rows = q.size(0), heads = q.size(1);
        for (const auto& [t, name] : {std::make_pair(&q, "q"), std::make_pair(&k, "k"), std::make_pair(&v, "v")})
            if (t->scalar_type() != cache.k.scalar_type())
                refuse(PyExc_TypeError, "%s must have the dtype of k_pages", name);
        check_shape(q, "q", {rows, heads, cache.c.head_dim});
        check_shape(k, "k", {rows, cache.c.kv_heads, cache.c.head_dim});
        check_shape(v, "v", {rows, cache.c.kv_heads, cache.c.head_dim});
        if (inv) check_dtype(*inv, "inv_freq", at::kFloat, "torch.float32");
        if (given) check_output(*given, q);
        const c10::Device device = device_of({{&q, "q"}, {&k, "k"}, {&v, "v"}, {&cache.k, "k_pages"},
            {&cache.v, "v_pages"}, {&cache.table_arg, "page_table"}, {&cache.cu_arg, "cu_rows"},
            {&cache.lengths_arg, "lengths"}, {inv ? inv : &q, "inv_freq"}, {given ? given : &q, "out"}});
        for (const at::Tensor* t : {&cache.k, &cache.v}) {
            if (overlap(*t, q) || overlap(*t, k) || overlap(*t, v) || (given && overlap(*t, *given)))
                refuse(PyExc_ValueError, "the cache must not share memory with q, k, v or out");
        }
        if (given && same_view(*given, q)) {
            if (!apart(q, k) || !apart(q, v))
                refuse(PyExc_ValueError, "q must not share its rows with k and v where it is rotated in place");
        } else if (given && (!apart(*given, q) || !apart(*given, k) || !apart(*given, v))) {
            refuse(PyExc_ValueError, "out must be q itself or share no memory with q, k and v");
        }
        const c10::DeviceGuard guard(device);
        if (!cache.c.batch || !rows) return THPVariable_Wrap(given ? *given : at::zeros(q.sizes(), q.options().requires_grad(false)));
        cache.bind();
        // (q in place only where it is read as it stands)
        const at::Tensor qs = usable(q), ks = usable(k), vs = usable(v);
        const at::Tensor freq = inv ? contiguous(*inv) : at::Tensor();
        const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options().requires_grad(false));
        const qwen2_rows rq = rows_of(qs), rk = rows_of(ks), rv = rows_of(vs), ro = rows_of(out);
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_paged_append(&cache.c, &rq, &rk, &rv, &ro, inv ? (const float*)freq.const_data_ptr() : nullptr,
                                      inv ? 2 * freq.numel() : 0, interleaved, (float)scale, rows, heads, !given, stream);
        });
        written(cache.k), written(cache.v);
        if (given) written(*given);
        return THPVariable_Wrap(out);
    });
}

// (q, k_pages, v_pages, page_table, cu_rows, lengths, shared_pages, scale or
// None, out or None) -> the attended rows
PyObject* host_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "paged_attention_hip";
        check_count(op, count, 9);
        check_state(op);
        const at::Tensor& q = tensor(args[0], op, "q", 3);
        Cache cache(op, args + 1);
        const int64_t shared = whole(args[6], "shared_pages");
        const at::Tensor* given = args[8] == Py_None ? nullptr : &tensor(args[8], op, "out", 3);
        const int64_t rows = q.size(0), heads = q.size(1);
        if (q.scalar_type() != cache.k.scalar_type()) refuse(PyExc_TypeError, "q must have the dtype of k_pages");
        check_shape(q, "q", {rows, heads, cache.c.head_dim});
        const double scale = args[7] == Py_None ? 1.0 / std::sqrt((double)std::max<int64_t>(cache.c.head_dim, 1))
                                                : number(args[7], "scale");
        if (given) check_output(*given, q);
        const c10::Device device = device_of({{&q, "q"}, {&cache.k, "k_pages"}, {&cache.v, "v_pages"},
            {&cache.table_arg, "page_table"}, {&cache.cu_arg, "cu_rows"}, {&cache.lengths_arg, "lengths"},
            {given ? given : &q, "out"}});
        if (given && (!apart(*given, q) || overlap(*given, cache.k) || overlap(*given, cache.v)))
            refuse(PyExc_ValueError, "out must share no memory with q and the cache");
        const c10::DeviceGuard guard(device);
        if (!cache.c.batch || !rows) return THPVariable_Wrap(given ? *given : at::zeros(q.sizes(), q.options().requires_grad(false)));
        cache.bind();
        const at::Tensor qs = usable(q);
        const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options().requires_grad(false));
        const qwen2_rows rq = rows_of(qs), ro = rows_of(out);
        const int64_t need = qwen2_paged_attention_workspace_bytes(&cache.c, rows, heads, shared);
        at::Tensor workspace;
        if (need) workspace = at::empty({need}, q.options().dtype(at::kByte).requires_grad(false));
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_paged_attention(&cache.c, &rq, &ro, rows, heads, shared, (float)scale, !given,
                                         need ? workspace.mutable_data_ptr() : nullptr, need, stream);
        });
        if (given) written(*given);
        return THPVariable_Wrap(out);
    });
}

// (target_probs, draft_tokens, uniforms, draft_probs or None, draft_lengths or
// None) -> (tokens, accepted)
PyObject* host_verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "verify_drafts_hip";
        check_count(op, count, 5);
        check_state(op);
        const at::Tensor& target = tensor(args[0], op, "target_probs", 3);
        const at::Tensor& tokens = tensor(args[1], op, "draft_tokens", 2);
        const at::Tensor& uniforms = tensor(args[2], op, "uniforms", 2);
        const at::Tensor* draft = args[3] == Py_None ? nullptr : &tensor(args[3], op, "draft_probs", 3);
        const at::Tensor* lengths = args[4] == Py_None ? nullptr : &tensor(args[4], op, "draft_lengths", 1);
        const int code = target.scalar_type() == at::kFloat      ? W4G64_DTYPE_F32
                         : target.scalar_type() == at::kBFloat16 ? W4G64_DTYPE_BF16
                         : target.scalar_type() == at::kHalf     ? W4G64_DTYPE_F16
                                                                 : W4G64_DTYPE_NONE;
        if (code == W4G64_DTYPE_NONE)
            refuse(PyExc_TypeError, "target_probs must have dtype torch.float32, torch.bfloat16 or torch.float16");
        const int64_t batch = tokens.size(0), drafts = tokens.size(1), vocab = target.size(2);
        check_dtype(tokens, "draft_tokens", at::kLong, "torch.int64");
        check_dtype(uniforms, "uniforms", at::kFloat, "torch.float32");
        check_shape(target, "target_probs", {batch, drafts + 1, vocab});
        check_shape(uniforms, "uniforms", {batch, drafts + 1});
        if (!vocab) refuse(PyExc_ValueError, "target_probs must have at least one entry per row");
        if (draft) {
            if (draft->scalar_type() != target.scalar_type()) refuse(PyExc_TypeError, "draft_probs must have the dtype of target_probs");
            check_shape(*draft, "draft_probs", {batch, drafts, vocab});
        }
        if (lengths) {
            check_dtype(*lengths, "draft_lengths", at::kInt, "torch.int32");
            check_shape(*lengths, "draft_lengths", {batch});
        }
        const c10::Device device = device_of({{&target, "target_probs"}, {&tokens, "draft_tokens"}, {&uniforms, "uniforms"},
            {draft ? draft : &target, "draft_probs"}, {lengths ? lengths : &target, "draft_lengths"}});
        const c10::DeviceGuard guard(device);
        const auto options = tokens.options().requires_grad(false);
        const at::Tensor chosen = at::empty({batch, drafts + 1}, options);
        const at::Tensor accepted = at::empty({batch}, options.dtype(at::kInt));
        if (batch) {
            auto rows = [](const at::Tensor& t) {  // (vocabulary entries one after the other)
                return t.size(2) > 1 && t.stride(2) != 1 ? at::clone(t, at::MemoryFormat::Contiguous) : t;
            };
            const at::Tensor p = rows(target), q = draft ? rows(*draft) : at::Tensor();
            const at::Tensor x = contiguous(tokens), u = contiguous(uniforms);
            const at::Tensor n = lengths ? contiguous(*lengths) : at::Tensor();
            const int64_t need = qwen2_verify_drafts_workspace_bytes(batch, drafts, vocab);
            const at::Tensor workspace = at::empty({std::max<int64_t>(need, 1)}, options.dtype(at::kByte));
            const hipStream_t stream = current_stream(device);
            released([&] {
                return qwen2_verify_drafts(p.const_data_ptr(), p.stride(0), p.stride(1),
                                           draft && drafts ? q.const_data_ptr() : nullptr, draft ? q.stride(0) : 0,
                                           draft ? q.stride(1) : 0, code, (const int64_t*)x.const_data_ptr(),
                                           lengths ? (const int32_t*)n.const_data_ptr() : nullptr,
                                           (const float*)u.const_data_ptr(), (int64_t*)chosen.mutable_data_ptr(),
                                           (int32_t*)accepted.mutable_data_ptr(), batch, drafts, vocab,
                                           workspace.mutable_data_ptr(), need, stream);
            });
        }
        PyObject* first = THPVariable_Wrap(chosen);
        PyObject* second = first ? THPVariable_Wrap(accepted) : nullptr;
        PyObject* pair = second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return pair;
    });
}

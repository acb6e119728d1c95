// Host side of the page operators (qwen_int4_hip.pages), in the module
// qwen_int4_hip._host: checks of the arguments, outputs and workspace, and the call
// into the C ABI.  There is no other route: what these refuse raises.
//
// Index tensors are returned new; workspaces come from torch's allocator for each
// call, as in host_paged.cpp.
#include "host_checks.h"

namespace {

// An index tensor of a call (int32).
const at::Tensor& indices(PyObject* obj, const char* op, const char* name, int64_t dims) {
    const at::Tensor& t = tensor(obj, op, name, dims);
    check_dtype(t, name, at::kInt, "torch.int32");
    return t;
}

at::Tensor rows_contiguous(const at::Tensor& table) {
    return table.size(1) > 1 && table.stride(1) != 1 ? at::clone(table, at::MemoryFormat::Contiguous) : table;
}

// Pools of one layer [pages, kv_heads, page_size, head_dim], or of several, layers
// first.
struct Pools {
    const at::Tensor &k, &v;
    qwen2_page_pool c{};

    static const at::Tensor& pool(PyObject* obj, const char* op, const char* name) {
        const bool layers = THPVariable_CheckExact(obj) && THPVariable_Unpack(obj).dim() == 5;
        return tensor(obj, op, name, layers ? 5 : 4);
    }

    Pools(const char* op, PyObject* const* args) : k(pool(args[0], op, "k_pages")), v(pool(args[1], op, "v_pages")) {
        if (k.scalar_type() != at::kBFloat16 && k.scalar_type() != at::kHalf)
            refuse(PyExc_TypeError, "k_pages must have dtype torch.bfloat16 or torch.float16");
        if (v.scalar_type() != k.scalar_type()) refuse(PyExc_TypeError, "v_pages must have the dtype of k_pages");
        if (v.sizes() != k.sizes()) refuse(PyExc_ValueError, "v_pages must have the shape of k_pages");
        if (!k.numel()) refuse(PyExc_ValueError, "k_pages must hold at least one layer, page, head, position and dimension");
        for (const at::Tensor* t : {&k, &v})
            if (!readable(*t) || !distinct(*t))
                refuse(PyExc_ValueError, "%s must be 16-byte aligned with a contiguous last dimension, other strides "
                       "multiples of 8, and no two entries in one place", t == &k ? "k_pages" : "v_pages");
        if (share(k, v)) refuse(PyExc_ValueError, "k_pages and v_pages must not share memory");
        const int64_t first = k.dim() - 4;
        c.layers = first ? k.size(0) : 1;
        c.num_pages = k.size(first), c.kv_heads = k.size(first + 1), c.page_size = k.size(first + 2);
        c.head_dim = k.size(first + 3);
        c.k_layer = first ? step(k, 0) : 0, c.v_layer = first ? step(v, 0) : 0;
        c.k_page = step(k, first), c.k_head = step(k, first + 1), c.k_position = step(k, first + 2);
        c.v_page = step(v, first), c.v_head = step(v, first + 1), c.v_position = step(v, first + 2);
    }

    void bind() { c.k = k.mutable_data_ptr(), c.v = v.mutable_data_ptr(); }

    // (the kernels read indices while pages are written)
    void apart_from(std::initializer_list<std::pair<const at::Tensor*, const char*>> all) const {
        for (const auto& [t, name] : all)
            if (overlap(k, *t) || overlap(v, *t)) refuse(PyExc_ValueError, "the pools must not share memory with %s", name);
    }
};

int32_t* data(const at::Tensor& t) { return (int32_t*)t.const_data_ptr(); }

PyObject* tuple_of(std::initializer_list<at::Tensor> all) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)all.size());
    Py_ssize_t i = 0;
    for (const at::Tensor& t : all) {
        PyObject* wrapped = tuple ? THPVariable_Wrap(t) : nullptr;
        if (!wrapped) {
            Py_XDECREF(tuple);
            return nullptr;
        }
        PyTuple_SET_ITEM(tuple, i++, wrapped);
    }
    return tuple;
}

}  // namespace

// (page_table, lengths, page_users, page_size, cached or None) -> (table, users, missing)
PyObject* host_paged_resize(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "paged_resize_hip";
        check_count(op, count, 5);
        check_state(op);
        const at::Tensor& table = indices(args[0], op, "page_table", 2);
        const at::Tensor& lengths = indices(args[1], op, "lengths", 1);
        const at::Tensor& users = indices(args[2], op, "page_users", 1);
        const int64_t page_size = whole(args[3], "page_size");
        const at::Tensor* cached = args[4] == Py_None ? nullptr : &indices(args[4], op, "cached", 1);
        const int64_t batch = table.size(0), width = table.size(1), pages = users.size(0);
        check_shape(lengths, "lengths", {batch});
        if (cached) check_shape(*cached, "cached", {batch});
        if (!width) refuse(PyExc_ValueError, "page_table must have at least one column");
        if (!pages) refuse(PyExc_ValueError, "page_users must have at least one entry");
        const c10::Device device = device_of({{&table, "page_table"}, {&lengths, "lengths"}, {&users, "page_users"},
            {cached ? cached : &users, "cached"}});
        const c10::DeviceGuard guard(device);
        check_status(w4g64::paged_resize_sizes(batch, width, pages, page_size));  // (before anything is copied)
        const at::Tensor t = rows_contiguous(table), n = contiguous(lengths), u = contiguous(users);
        const at::Tensor held = cached ? contiguous(*cached) : at::Tensor();
        const auto options = users.options().requires_grad(false);
        const at::Tensor new_table = at::empty({batch, width}, options), new_users = at::empty({pages}, options);
        const at::Tensor missing = at::empty({batch}, options);
        const int64_t need = qwen2_paged_resize_workspace_bytes(batch, width, pages);
        at::Tensor workspace;
        if (need) workspace = at::empty({need}, options.dtype(at::kByte));
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_paged_resize_cached(data(t), t.stride(0), data(n), cached ? data(held) : nullptr, data(u),
                                             data(new_table), data(new_users), data(missing), batch, width, pages, page_size,
                                             need ? workspace.mutable_data_ptr() : nullptr, need, stream);
        });
        return tuple_of({new_table, new_users, missing});
    });
}

// (k_pages, v_pages, page_table, lengths, page_users, parents) -> (table, lengths, users, missing)
PyObject* host_paged_fork(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "paged_fork_hip";
        check_count(op, count, 6);
        check_state(op);
        Pools pools(op, args);
        const at::Tensor& table = indices(args[2], op, "page_table", 2);
        const at::Tensor& lengths = indices(args[3], op, "lengths", 1);
        const at::Tensor& users = indices(args[4], op, "page_users", 1);
        const at::Tensor& parents = indices(args[5], op, "parents", 1);
        const int64_t batch = table.size(0), width = table.size(1), children = parents.size(0);
        check_shape(lengths, "lengths", {batch});
        check_shape(users, "page_users", {pools.c.num_pages});
        if (!width) refuse(PyExc_ValueError, "page_table must have at least one column");
        const c10::Device device = device_of({{&pools.k, "k_pages"}, {&pools.v, "v_pages"}, {&table, "page_table"},
            {&lengths, "lengths"}, {&users, "page_users"}, {&parents, "parents"}});
        pools.apart_from({{&table, "page_table"}, {&lengths, "lengths"}, {&users, "page_users"}, {&parents, "parents"}});
        const c10::DeviceGuard guard(device);
        pools.bind();
        check_status(w4g64::paged_fork_sizes(&pools.c, batch, children, width));
        const at::Tensor t = rows_contiguous(table), n = contiguous(lengths), u = contiguous(users), p = contiguous(parents);
        const auto options = users.options().requires_grad(false);
        const at::Tensor new_table = at::empty({children, width}, options), new_lengths = at::empty({children}, options);
        const at::Tensor new_users = at::empty({pools.c.num_pages}, options), missing = at::empty({children}, options);
        const int64_t need = qwen2_paged_fork_workspace_bytes(batch, children, width, pools.c.num_pages);
        at::Tensor workspace;
        if (need) workspace = at::empty({need}, options.dtype(at::kByte));
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_paged_fork(&pools.c, data(t), t.stride(0), data(n), data(u), data(p), data(new_table),
                                    data(new_lengths), data(new_users), data(missing), batch, children, width,
                                    need ? workspace.mutable_data_ptr() : nullptr, need, stream);
        });
        written(pools.k), written(pools.v);
        return tuple_of({new_table, new_lengths, new_users, missing});
    });
}

// (k_pages, v_pages, page_table, page_users) -> (table, users, moved_to)
PyObject* host_paged_compact(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "paged_compact_hip";
        check_count(op, count, 4);
        check_state(op);
        Pools pools(op, args);
        const at::Tensor& table = indices(args[2], op, "page_table", 2);
        const at::Tensor& users = indices(args[3], op, "page_users", 1);
        const int64_t batch = table.size(0), width = table.size(1), pages = pools.c.num_pages;
        check_shape(users, "page_users", {pages});
        if (!width) refuse(PyExc_ValueError, "page_table must have at least one column");
        const c10::Device device = device_of({{&pools.k, "k_pages"}, {&pools.v, "v_pages"}, {&table, "page_table"},
            {&users, "page_users"}});
        pools.apart_from({{&table, "page_table"}, {&users, "page_users"}});
        const c10::DeviceGuard guard(device);
        pools.bind();
        check_status(w4g64::paged_compact_sizes(&pools.c, batch, width));
        const at::Tensor t = rows_contiguous(table), u = contiguous(users);
        const auto options = users.options().requires_grad(false);
        const at::Tensor new_table = at::empty({batch, width}, options);
        const at::Tensor new_users = at::empty({pages}, options), moved_to = at::empty({pages}, options);
        const int64_t need = qwen2_paged_compact_workspace_bytes(batch, width, pages);
        at::Tensor workspace;
        if (need) workspace = at::empty({need}, options.dtype(at::kByte));
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_paged_compact(&pools.c, data(t), t.stride(0), data(u), data(new_table), data(new_users),
                                       data(moved_to), batch, width, need ? workspace.mutable_data_ptr() : nullptr, need, stream);
        });
        written(pools.k), written(pools.v);
        return tuple_of({new_table, new_users, moved_to});
    });
}

// Host side of the packed prompt attention (qwen_int4_hip.packed), in the module
// qwen_int4_hip._host: checks of the arguments, the output, and the call into the C
// ABI.  There is no other route: what this refuses raises.
#include "host_checks.h"

// (q, k, v, cu_rows, scale or None, out or None) -> the attended rows
PyObject* host_packed_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const char* op = "packed_attention_hip";
        check_count(op, count, 6);
        check_state(op);
        const at::Tensor& q = tensor(args[0], op, "q", 3);
        const at::Tensor& k = tensor(args[1], op, "k", 3);
        const at::Tensor& v = tensor(args[2], op, "v", 3);
        const at::Tensor& cu = tensor(args[3], op, "cu_rows", 1);
        const at::Tensor* given = args[5] == Py_None ? nullptr : &tensor(args[5], op, "out", 3);
        const int64_t rows = q.size(0), heads = q.size(1), kv_heads = k.size(1), dim = q.size(2);
        if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf)
            refuse(PyExc_TypeError, "q must have dtype torch.bfloat16 or torch.float16");
        if (k.scalar_type() != q.scalar_type()) refuse(PyExc_TypeError, "k must have the dtype of q");
        if (v.scalar_type() != q.scalar_type()) refuse(PyExc_TypeError, "v must have the dtype of q");
        check_dtype(cu, "cu_rows", at::kInt, "torch.int32");
        check_shape(k, "k", {rows, kv_heads, dim});
        check_shape(v, "v", {rows, kv_heads, dim});
        if (!cu.size(0)) refuse(PyExc_ValueError, "cu_rows must have at least one entry");
        const double scale = args[4] == Py_None ? 1.0 / std::sqrt((double)std::max<int64_t>(dim, 1)) : number(args[4], "scale");
        if (given) check_output(*given, q);
        const c10::Device device = device_of({{&q, "q"}, {&k, "k"}, {&v, "v"}, {&cu, "cu_rows"}, {given ? given : &q, "out"}});
        if (given && (!apart(*given, q) || !apart(*given, k) || !apart(*given, v) || overlap(*given, cu)))
            refuse(PyExc_ValueError, "out must share no memory with q, k, v and cu_rows");
        const c10::DeviceGuard guard(device);
        const int64_t batch = cu.size(0) - 1;
        const int code = q.scalar_type() == at::kHalf ? W4G64_DTYPE_F16 : W4G64_DTYPE_BF16;
        const bool none = !batch || !rows;
        // (before anything is copied or filled; where nothing is, the library's call asks the same)
        if (none || !readable(q) || !readable(k) || !readable(v) || !cu.is_contiguous()) {
            auto row_step = [&](const at::Tensor& t) { return readable(t) ? step(t, 0) : kv_heads * dim; };
            check_status(w4g64::packed_attention_sizes(batch, rows, heads, kv_heads, dim, row_step(k), row_step(v), code, (float)scale));
        }
        const at::Tensor qs = usable(q), ks = usable(k), vs = usable(v), bounds = contiguous(cu);
        const at::Tensor out = given ? *given : none ? at::zeros(q.sizes(), q.options().requires_grad(false))
                                                     : at::empty(q.sizes(), q.options().requires_grad(false));
        auto rows_of = [](const at::Tensor& t) {
            return qwen2_rows{const_cast<void*>(t.const_data_ptr()), step(t, 0), step(t, 1)};
        };
        const qwen2_rows rq = rows_of(qs), rk = rows_of(ks), rv = rows_of(vs), ro = rows_of(out);
        const hipStream_t stream = current_stream(device);
        released([&] {
            return qwen2_packed_attention(&rq, &rk, &rv, &ro, (const int32_t*)bounds.const_data_ptr(), batch, rows, heads,
                                          kv_heads, dim, code, (float)scale, !given, stream);
        });
        if (given) written(*given);
        return THPVariable_Wrap(out);
    });
}

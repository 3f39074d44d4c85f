// The paged key-value cache's operators on tensors (camblas_hip.h says what each computes): argument
// checks, the output and workspace of a call, and the call. BF16, inference only.
#include "binding.hpp"

namespace py = pybind11;

namespace binding
{
namespace
{
camblas_cuda_paged_cache pages_of(const Tensor &k, const Tensor &v, const at::Device &device)
{
    bool alike = k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.dim() == 4 &&
                 k.sizes().equals(v.sizes()) && k.device() == device && v.device() == device;
    for (int axis = 0; alike && axis < 4; ++axis)
        alike = k.size(axis) < 2 || k.stride(axis) == v.stride(axis);
    require(alike,
            "a paged cache is two BF16 tensors [pages, page_size, kv_heads, dim] of one layout on the operands' device");
    require(!recording(k) && !recording(v), "the paged cache's operators support inference only");
    require(k.size(0) >= 1 && k.size(0) <= INT_MAX && k.size(1) <= INT_MAX && k.size(2) <= INT_MAX &&
                (k.size(3) == 64 || k.size(3) == 128) && k.stride(3) == 1,
            "paged heads must hold 64 or 128 contiguous values");
    camblas_cuda_paged_cache cache = {};
    cache.k = k.data_ptr();
    cache.v = v.data_ptr();
    // (the stride of an axis of one element says nothing)
    cache.page_stride = k.size(0) > 1 ? k.stride(0) : 0;
    cache.slot_stride = k.size(1) > 1 ? k.stride(1) : 0;
    cache.head_stride = k.size(2) > 1 ? k.stride(2) : 0;
    cache.pages = int(k.size(0));
    cache.page_size = int(k.size(1));
    cache.kv_heads = int(k.size(2));
    cache.dim = int(k.size(3));
    return cache;
}

// BF16 rows [tokens, heads, dim] whose heads lie next to each other; returns the stride between rows
int64_t row_stride(const char *role, const Tensor &rows, int64_t tokens, int64_t heads, int64_t dim, const at::Device &device)
{
    const bool fits = rows.scalar_type() == at::kBFloat16 && rows.dim() == 3 && rows.size(0) == tokens &&
                      rows.size(1) == heads && rows.size(2) == dim && rows.device() == device && rows.stride(2) == 1 &&
                      (heads == 1 || rows.stride(1) == dim) && tokens <= INT_MAX && heads <= INT_MAX;
    if (!fits)
        throw std::invalid_argument(std::string(role) + " must be BF16 [" + std::to_string(tokens) + ", " +
                                    std::to_string(heads) + ", " + std::to_string(dim) +
                                    "] with dense heads on the operands' GPU");
    require(!recording(rows), "the paged cache's operators support inference only");
    return tokens > 1 ? rows.stride(0) : heads * dim;
}

void check_integers(const char *role, const Tensor &values, at::ScalarType type, int64_t count, const at::Device &device)
{
    if (values.scalar_type() != type || values.dim() != 1 || values.size(0) != count || values.device() != device ||
        !values.is_contiguous())
        throw std::invalid_argument(std::string(role) + " must be contiguous " + (type == at::kInt ? "int32 [" : "int64 [") +
                                    std::to_string(count) + "] on the operands' GPU");
}

// out, or a new BF16 [tokens, heads, dim] tensor
Tensor output_rows(const std::optional<Tensor> &out, int64_t tokens, int64_t heads, int64_t dim, const Tensor &like)
{
    return out ? *out : at::empty({tokens, heads, dim}, like.options());
}

// After a call that wrote into `tensor`: a backward that kept it reports that it changed.
void changed(const Tensor &tensor)
{
    if (!tensor.is_inference())
        torch::autograd::impl::bump_version(tensor);
}

int as_int(const char *role, int64_t value)
{
    if (value < 0 || value > INT_MAX)
        throw std::invalid_argument(std::string(role) + " must lie in [0, 2^31)");
    return int(value);
}

Tensor append(const Tensor &qkv, const Tensor &positions, const Tensor &slots, const Tensor &k_cache, const Tensor &v_cache,
              int64_t q_heads, int64_t kv_heads, const std::optional<Tensor> &q_weight, const std::optional<Tensor> &k_weight,
              double epsilon, double theta, const std::optional<int64_t> &rotary_dim, const std::optional<Tensor> &out)
{
    require(qkv.is_cuda() && qkv.dim() == 3 && q_heads >= 1 && q_heads <= INT_MAX && kv_heads >= 1 && kv_heads <= INT_MAX,
            "qkv must be BF16 [tokens, q_heads + 2 kv_heads, dim] on a GPU");
    const at::Device device = qkv.device();
    const camblas_cuda_paged_cache cache = pages_of(k_cache, v_cache, device);
    const int64_t tokens = qkv.size(0), dim = qkv.size(2);
    require(cache.kv_heads == kv_heads && cache.dim == dim, "the cache's heads differ from the activation's");
    const int64_t stride = row_stride("qkv", qkv, tokens, q_heads + 2 * kv_heads, dim, device);
    check_integers("positions", positions, at::kInt, tokens, device);
    check_integers("slots", slots, at::kLong, tokens, device);
    require(q_weight.has_value() == k_weight.has_value(), "query and key norm weights come together");
    if (q_weight) {
        for (const Tensor *weight : {&*q_weight, &*k_weight})
            require((weight->scalar_type() == at::kFloat || weight->scalar_type() == at::kBFloat16) &&
                        weight->scalar_type() == q_weight->scalar_type() && weight->dim() == 1 && weight->size(0) == dim &&
                        weight->is_contiguous() && weight->device() == device && !recording(*weight),
                    "norm weights must be contiguous FP32 or BF16 [dim] on the operands' GPU, without gradients");
    }
    c10::DeviceGuard guard(device);
    Tensor queries = output_rows(out, tokens, q_heads, dim, qkv);
    const int64_t queries_stride = row_stride("out", queries, tokens, q_heads, dim, device);
    camblas_cuda_context *context = context_for(device.index(), current_default_algorithm());
    succeed(camblas_cuda_qk_norm_rope_append_wide_theta(
                context, int(tokens), int(q_heads), rotary_dim ? as_int("rotary_dim", *rotary_dim) : int(dim), theta,
                q_weight ? storage_code(*q_weight) : 0, float(epsilon), q_weight ? q_weight->const_data_ptr() : nullptr,
                k_weight ? k_weight->const_data_ptr() : nullptr, positions.const_data_ptr<int32_t>(),
                slots.const_data_ptr<int64_t>(), qkv.const_data_ptr(), stride, queries.mutable_data_ptr(), queries_stride,
                &cache),
            context);
    changed(k_cache);
    changed(v_cache);
    if (out)
        changed(queries);
    return queries;
}

// what the two attentions share
struct Attention {
    camblas_cuda_paged_cache cache;
    at::Device device;
    int batch, columns, tokens, q_heads, window, sinks;
    int64_t q_stride, output_stride, table_stride;
    float scale;
    Tensor output;

    Attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &lengths,
              const std::optional<double> &scale_in, int64_t window_in, int64_t sinks_in, const std::optional<Tensor> &out)
        : cache(pages_of(k_cache, v_cache, q.device())), device(q.device())
    {
        require(q.is_cuda() && q.dim() == 3, "q must be BF16 [tokens, heads, dim] on a GPU");
        require(page_table.scalar_type() == at::kInt && page_table.dim() == 2 && page_table.device() == device &&
                    page_table.size(0) <= INT_MAX && page_table.size(1) <= INT_MAX &&
                    (page_table.size(1) < 2 || page_table.stride(1) == 1),
                "page_table must be int32 [batch, columns] with dense rows on the operands' GPU");
        check_integers("lengths", lengths, at::kInt, page_table.size(0), device);
        q_stride = row_stride("q", q, q.size(0), q.size(1), cache.dim, device);
        batch = int(page_table.size(0));
        columns = int(page_table.size(1));
        table_stride = batch > 1 ? page_table.stride(0) : columns;
        tokens = int(q.size(0));
        q_heads = int(q.size(1));
        window = as_int("window", window_in);
        sinks = as_int("sinks", sinks_in);
        scale = scale_in ? float(*scale_in) : cache.dim == 64 ? 0.125f : 0.088388347648318447f;
        output = output_rows(out, q.size(0), q.size(1), q.size(2), q);
        output_stride = row_stride("out", output, q.size(0), q.size(1), q.size(2), device);
    }
};

Tensor decode(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &lengths,
              const std::optional<double> &scale, int64_t window, int64_t sinks, const std::optional<Tensor> &out)
{
    c10::OptionalDeviceGuard guard(q.device());
    Attention a(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out);
    require(a.batch == a.tokens, "one query, one table row and one length per sequence");
    camblas_cuda_context *context = context_for(a.device.index(), current_default_algorithm());
    const size_t bytes = camblas_cuda_paged_decode_workspace_size(context, a.batch, a.q_heads, &a.cache, a.columns, a.window, a.sinks);
    Tensor workspace;
    if (bytes)
        workspace = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
    succeed(camblas_cuda_paged_decode_attention(
                context, a.batch, a.q_heads, &a.cache, page_table.const_data_ptr<int32_t>(), a.table_stride, a.columns,
                lengths.const_data_ptr<int32_t>(), a.window, a.sinks, a.scale, q.const_data_ptr(), a.q_stride,
                bytes ? workspace.mutable_data_ptr() : nullptr, bytes, a.output.mutable_data_ptr(), a.output_stride),
            context);
    if (out)
        changed(a.output);
    return a.output;
}

Tensor prefill(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &page_table, const Tensor &lengths,
               const Tensor &query_starts, const std::optional<double> &scale, int64_t window, int64_t sinks,
               const std::optional<Tensor> &out)
{
    c10::OptionalDeviceGuard guard(q.device());
    Attention a(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out);
    check_integers("query_starts", query_starts, at::kInt, int64_t(a.batch) + 1, a.device);
    camblas_cuda_context *context = context_for(a.device.index(), current_default_algorithm());
    const size_t bytes =
        camblas_cuda_paged_prefill_workspace_size(context, a.batch, a.tokens, a.q_heads, &a.cache, a.columns, a.window, a.sinks);
    Tensor workspace;
    if (bytes)
        workspace = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
    succeed(camblas_cuda_paged_prefill_attention(
                context, a.batch, a.tokens, a.q_heads, &a.cache, page_table.const_data_ptr<int32_t>(), a.table_stride,
                a.columns, lengths.const_data_ptr<int32_t>(), query_starts.const_data_ptr<int32_t>(), a.window, a.sinks,
                a.scale, q.const_data_ptr(), a.q_stride, bytes ? workspace.mutable_data_ptr() : nullptr, bytes,
                a.output.mutable_data_ptr(), a.output_stride),
            context);
    if (out)
        changed(a.output);
    return a.output;
}
} // namespace

void register_paged(py::module_ &module)
{
    // (by position too: eight arguments found by their names are 1 of 5 us of a call)
    module.def("qk_norm_rope_append", &append, py::arg("qkv"), py::arg("positions"), py::arg("slots"), py::arg("k_cache"),
               py::arg("v_cache"), py::arg("q_heads"), py::arg("kv_heads"), py::arg("q_weight") = py::none(),
               py::arg("k_weight") = py::none(), py::arg("epsilon") = 1e-6, py::arg("theta") = 500000.,
               py::arg("rotary_dim") = py::none(), py::arg("out") = py::none(),
               "Normalise and rotate query and key heads, append keys and values to a paged cache; the queries.");
    module.def("paged_decode_attention", &decode, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("page_table"),
               py::arg("lengths"), py::arg("scale") = py::none(), py::arg("window") = 0, py::arg("sinks") = 0,
               py::arg("out") = py::none(), "Attention of one new token per sequence over a paged cache.");
    module.def("paged_prefill_attention", &prefill, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
               py::arg("page_table"), py::arg("lengths"), py::arg("query_starts"),
               py::arg("scale") = py::none(), py::arg("window") = 0, py::arg("sinks") = 0, py::arg("out") = py::none(),
               "Causal attention of the new tokens of ragged sequences over a paged cache.");
}
} // namespace binding

// KvCacheWrite, KvCacheRead, CacheAttention and PrefixAttention for Backend::HIP:
// descriptor rules, lowered onto nnops_hip_kv_cache_write / _read,
// nnops_hip_cache_attention and nnops_hip_prefix_attention.
#include "nnops/ops/kv_cache.hpp"
#include "nnops_amd.h"
#include "views.hpp"

namespace nnops {
namespace {

/// page_table, lengths [, row_starts], for a call of `rows` rows.
Status check_tables(std::span<const TensorDesc> t, int64_t rows)
{
    if (t[0].rank != 2 || t[1].rank != 1 || t[0].dims[0] != t[1].dims[0] || t[0].dtype != DataType::s32 ||
        t[1].dtype != DataType::s32) {
        return Status::invalid_argument;
    }
    if (t.size() > 2 && (t[2].rank != 1 || t[2].dims[0] != t[1].dims[0] + 1 || t[2].dtype != DataType::s32)) {
        return Status::invalid_argument;
    }
    // without starts, every sequence has as many rows
    const int64_t seqs = t[1].dims[0];
    if (rows > 0 && (seqs == 0 || (t.size() <= 2 && rows % seqs != 0))) {
        return Status::invalid_argument;
    }
    return Status::ok;
}

/// Rows of a type that the kernels take, heads * head_dim wide.
Status check_rows(const TensorDesc& r, int64_t heads, const TensorDesc& k_cache)
{
    if (r.rank != 2 || r.dims[1] != heads * k_cache.dims[3]) {
        return Status::invalid_argument;
    }
    return is_float(r.dtype) ? Status::ok : Status::unsupported;
}

NnopsKvPages pages_of(std::span<const TensorDesc> cache, std::span<const TensorDesc> tables)
{
    NnopsKvPages p{};
    p.pages = cache[0].dims[0];
    p.heads = cache[0].dims[1];
    p.page_tokens = cache[0].dims[2];
    p.head_dim = cache[0].dims[3];
    p.sequences = tables[0].dims[0];
    p.table_pages = tables[0].dims[1];
    p.ld_table = row_step(tables[0]);
    return p;
}

void set_data(NnopsKvPages& p, std::span<const TensorView> cache, std::span<const TensorView> tables)
{
    p.k = cache[0].ptr<int8_t>();
    p.v = cache[1].ptr<int8_t>();
    p.k_scale = cache[2].ptr<float>();
    p.v_scale = cache[3].ptr<float>();
    p.page_table = tables[0].ptr<const int32_t>();
    p.lengths = tables[1].ptr<const int32_t>();
    p.row_starts = tables.size() > 2 ? tables[2].ptr<const int32_t>() : nullptr;
}

/// The shared rules of write and read: rows k, v, the cache and the tables.
Status check_rw(std::span<const TensorDesc> rows, std::span<const TensorDesc> cache,
                std::span<const TensorDesc> tables)
{
    if (!all_plain(rows) || !all_plain(cache) || !all_plain(tables)) {
        return Status::invalid_argument;
    }
    if (Status s = check_cache(cache); !is_ok(s)) {
        return s;
    }
    if (rows[0].rank != 2 || !same_shape(rows[0], rows[1]) || rows[0].dtype != rows[1].dtype) {
        return Status::invalid_argument;
    }
    if (Status s = check_tables(tables, rows[0].dims[0]); !is_ok(s)) {
        return s;
    }
    return check_rows(rows[0], cache[0].dims[1], cache[0]);
}

NnopsKvRowsArgs rows_args(std::span<const TensorView> rows, std::span<const TensorDesc> rows_d,
                          std::span<const TensorView> cache, std::span<const TensorDesc> cache_d,
                          std::span<const TensorView> tables, std::span<const TensorDesc> tables_d)
{
    NnopsKvRowsArgs a{};
    a.cache = pages_of(cache_d, tables_d);
    set_data(a.cache, cache, tables);
    a.k_rows = rows[0].ptr<void>();
    a.v_rows = rows[1].ptr<void>();
    a.rows = rows_d[0].dims[0];
    a.ld_k = row_step(rows_d[0]);
    a.ld_v = row_step(rows_d[1]);
    a.f16 = rows_d[0].dtype == DataType::f16;
    return a;
}

}  // namespace

std::unique_ptr<KvCacheWrite> KvCacheWrite::create(Backend backend)
{
    return std::unique_ptr<KvCacheWrite>(new KvCacheWrite(backend));
}

std::vector<TensorDesc> KvCacheWrite::getOutputTensorDesc(std::span<const TensorDesc>) const { return {}; }

Status KvCacheWrite::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() < 4 || inputs.size() > 5 || outputs.size() != 4) {
        return Status::invalid_argument;
    }
    return check_rw(inputs.first(2), outputs, inputs.subspan(2));
}

Status KvCacheWrite::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                             const ComputeContext& ctx, void* workspace)
{
    (void)workspace;
    std::array<TensorDesc, 5> in;
    std::array<TensorDesc, 4> out;
    const std::span<const TensorView> cache(outputs);
    if (!descs_of(inputs, in) || !descs_of(cache, out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size()), od(out.data(), outputs.size());
    if (Status s = validate(id, od); !is_ok(s)) {
        return s;
    }
    const NnopsKvRowsArgs a = rows_args(inputs.first(2), id.first(2), cache, od, inputs.subspan(2), id.subspan(2));
    return from_abi(nnops_hip_kv_cache_write(&a, ctx.hip_stream));
}

std::unique_ptr<KvCacheRead> KvCacheRead::create(const KvCacheReadAttributes& attrs, Backend backend)
{
    return std::unique_ptr<KvCacheRead>(new KvCacheRead(attrs, backend));
}

std::vector<TensorDesc> KvCacheRead::getOutputTensorDesc(std::span<const TensorDesc>) const { return {}; }

Status KvCacheRead::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() < 6 || inputs.size() > 7 || outputs.size() != 2) {
        return Status::invalid_argument;
    }
    if (Status s = check_rw(outputs, inputs.first(4), inputs.subspan(4)); !is_ok(s)) {
        return s;
    }
    return outputs[0].dtype == attrs_.output_dtype ? Status::ok : Status::invalid_argument;
}

Status KvCacheRead::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                            const ComputeContext& ctx, void* workspace)
{
    (void)workspace;
    std::array<TensorDesc, 7> in;
    std::array<TensorDesc, 2> out;
    const std::span<const TensorView> rows(outputs);
    if (!descs_of(inputs, in) || !descs_of(rows, out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size()), od(out.data(), outputs.size());
    if (Status s = validate(id, od); !is_ok(s)) {
        return s;
    }
    const NnopsKvRowsArgs a =
        rows_args(rows, od, inputs.first(4), id.first(4), inputs.subspan(4), id.subspan(4));
    return from_abi(nnops_hip_kv_cache_read(&a, ctx.hip_stream));
}

namespace {

/// q, the cache and its tables, and the output of an attention.
Status check_attention(std::span<const TensorDesc> inputs, std::span<const TensorDesc> tables, const TensorDesc& out)
{
    if (Status s = check_cache(inputs.subspan(1, 4)); !is_ok(s)) {
        return s;
    }
    const TensorDesc& q = inputs[0];
    if (q.rank != 2) {
        return Status::invalid_argument;
    }
    if (Status s = check_tables(tables, q.dims[0]); !is_ok(s)) {
        return s;
    }
    const int64_t width = inputs[1].dims[1] * inputs[1].dims[3];
    if (width <= 0 || q.dims[1] <= 0 || q.dims[1] % width != 0 || !same_shape(q, out) || q.dtype != out.dtype) {
        return Status::invalid_argument;
    }
    return is_float(q.dtype) ? Status::ok : Status::unsupported;
}

NnopsCacheAttentionArgs attention_args(const CacheAttentionAttributes& attrs, std::span<const TensorDesc> in,
                                       const TensorDesc& out)
{
    NnopsCacheAttentionArgs a{};
    a.cache = pages_of(in.subspan(1, 4), in.subspan(5));
    a.rows = in[0].dims[0];
    a.q_heads = a.cache.head_dim > 0 ? in[0].dims[1] / a.cache.head_dim : 0;
    a.ld_q = row_step(in[0]);
    a.ld_out = row_step(out);
    a.f16 = in[0].dtype == DataType::f16;
    a.scale = attrs.scale;
    a.window = attrs.window;
    a.sinks = attrs.sinks;
    return a;
}

}  // namespace

std::unique_ptr<CacheAttention> CacheAttention::create(const CacheAttentionAttributes& attrs, Backend backend)
{
    return std::unique_ptr<CacheAttention>(new CacheAttention(attrs, backend));
}

std::vector<TensorDesc> CacheAttention::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.empty()) {
        return {};
    }
    TensorDesc y = inputs[0];
    y.row_stride_elems = 0;
    return {y};
}

Status CacheAttention::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() < 7 || inputs.size() > 8 || outputs.size() != 1 || !all_plain(inputs) || !all_plain(outputs) ||
        !(attrs_.scale >= 0.0f) || attrs_.window < 0 || attrs_.sinks < 0) {
        return Status::invalid_argument;
    }
    return check_attention(inputs, inputs.subspan(5), outputs[0]);
}

size_t CacheAttention::getWorkspaceSize(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (!is_ok(validate(inputs, outputs))) {
        return 0;
    }
    NnopsCacheAttentionArgs a = attention_args(attrs_, inputs, outputs[0]);
    // (whether there are row starts plays a part, not where they are)
    static const int32_t some = 0;
    a.cache.row_starts = inputs.size() > 7 ? &some : nullptr;
    return nnops_hip_cache_attention_workspace_size(&a);
}

Status CacheAttention::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                               const ComputeContext& ctx, void* workspace)
{
    std::array<TensorDesc, 8> in;
    std::array<TensorDesc, 1> out;
    if (!descs_of(inputs, in) || !descs_of(std::span<const TensorView>(outputs), out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size());
    if (Status s = validate(id, std::span<const TensorDesc>(out.data(), outputs.size())); !is_ok(s)) {
        return s;
    }
    NnopsCacheAttentionArgs a = attention_args(attrs_, id, out[0]);
    set_data(a.cache, inputs.subspan(1, 4), inputs.subspan(5));
    a.q = inputs[0].ptr<const void>();
    a.out = outputs[0].ptr<void>();
    // the workspace is the one that getWorkspaceSize asks for
    const size_t bytes = nnops_hip_cache_attention_workspace_size(&a);
    return from_abi(nnops_hip_cache_attention(&a, workspace, workspace != nullptr ? bytes : 0, ctx.hip_stream));
}

namespace {

/// page_table, lengths [, row_starts] of a PrefixAttention's inputs.
template <typename V>
struct Tables {
    std::array<V, 3> at;
    size_t n;
    explicit Tables(std::span<const V> inputs) : n(inputs.size() > 9 ? 3 : 2)
    {
        at[0] = inputs[5];
        at[1] = inputs[6];
        if (n > 2) {
            at[2] = inputs[9];
        }
    }
    std::span<const V> span() const { return {at.data(), n}; }
};

NnopsPrefixAttentionArgs prefix_args(const PrefixAttentionAttributes& attrs, std::span<const TensorDesc> in,
                                     const TensorDesc& out)
{
    NnopsPrefixAttentionArgs a{};
    a.cache = pages_of(in.subspan(1, 4), in.subspan(5, 2));
    a.rows = in[0].dims[0];
    a.q_heads = a.cache.head_dim > 0 ? in[0].dims[1] / a.cache.head_dim : 0;
    a.ld_q = row_step(in[0]);
    a.ld_out = row_step(out);
    a.f16 = in[0].dtype == DataType::f16;
    a.scale = attrs.scale;
    a.groups = in[8].dims[0];
    return a;
}

}  // namespace

std::unique_ptr<PrefixAttention> PrefixAttention::create(const PrefixAttentionAttributes& attrs, Backend backend)
{
    return std::unique_ptr<PrefixAttention>(new PrefixAttention(attrs, backend));
}

std::vector<TensorDesc> PrefixAttention::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.empty()) {
        return {};
    }
    TensorDesc y = inputs[0];
    y.row_stride_elems = 0;
    return {y};
}

Status PrefixAttention::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() < 9 || inputs.size() > 10 || outputs.size() != 1 || !all_plain(inputs) || !all_plain(outputs) ||
        !(attrs_.scale >= 0.0f)) {
        return Status::invalid_argument;
    }
    const TensorDesc &starts = inputs[7], &shared = inputs[8];
    if (starts.rank != 1 || shared.rank != 1 || starts.dtype != DataType::s32 || shared.dtype != DataType::s32 ||
        starts.dims[0] != shared.dims[0] + 1) {
        return Status::invalid_argument;
    }
    return check_attention(inputs, Tables<TensorDesc>(inputs).span(), outputs[0]);
}

size_t PrefixAttention::getWorkspaceSize(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (!is_ok(validate(inputs, outputs))) {
        return 0;
    }
    NnopsPrefixAttentionArgs a = prefix_args(attrs_, inputs, outputs[0]);
    // (whether there are row starts plays a part, not where they are)
    static const int32_t some = 0;
    a.cache.row_starts = inputs.size() > 9 ? &some : nullptr;
    return nnops_hip_prefix_attention_workspace_size(&a);
}

Status PrefixAttention::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                                const ComputeContext& ctx, void* workspace)
{
    std::array<TensorDesc, 10> in;
    std::array<TensorDesc, 1> out;
    if (!descs_of(inputs, in) || !descs_of(std::span<const TensorView>(outputs), out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size());
    if (Status s = validate(id, std::span<const TensorDesc>(out.data(), outputs.size())); !is_ok(s)) {
        return s;
    }
    NnopsPrefixAttentionArgs a = prefix_args(attrs_, id, out[0]);
    set_data(a.cache, inputs.subspan(1, 4), Tables<TensorView>(inputs).span());
    a.q = inputs[0].ptr<const void>();
    a.out = outputs[0].ptr<void>();
    a.group_starts = inputs[7].ptr<const int32_t>();
    a.shared = inputs[8].ptr<const int32_t>();
    const size_t bytes = nnops_hip_prefix_attention_workspace_size(&a);
    return from_abi(nnops_hip_prefix_attention(&a, workspace, workspace != nullptr ? bytes : 0, ctx.hip_stream));
}

}  // namespace nnops

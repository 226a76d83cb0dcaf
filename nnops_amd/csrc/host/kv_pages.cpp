// KvCacheFork, KvCacheCompact and KvCacheCopy for Backend::HIP: descriptor rules,
// lowered onto nnops_hip_kv_cache_fork / _compact / _copy.
#include "nnops/ops/kv_pages.hpp"
#include "nnops_amd.h"
#include "views.hpp"

namespace nnops {
namespace {

TensorDesc s32(std::initializer_list<int64_t> dims)
{
    TensorDesc d;
    d.dtype = DataType::s32;
    for (const int64_t n : dims) {
        d.dims[static_cast<size_t>(d.rank++)] = n;
    }
    return d;
}

bool all_s32(std::span<const TensorDesc> d)
{
    for (const TensorDesc& t : d) {
        if (!plain_dims(t) || t.dtype != DataType::s32) {
            return false;
        }
    }
    return true;
}

/// page_table, lengths, refs.
bool tables_fit(std::span<const TensorDesc> in)
{
    return in[0].rank == 2 && in[1].rank == 1 && in[2].rank == 1 && in[1].dims[0] == in[0].dims[0];
}

NnopsKvForkArgs fork_args(const KvCacheForkAttributes& attrs, std::span<const TensorDesc> in,
                          std::span<const TensorDesc> out)
{
    NnopsKvForkArgs a{};
    a.sequences = in[0].dims[0];
    a.table_pages = in[0].dims[1];
    a.ld_table = row_step(in[0]);
    a.pages = in[2].dims[0];
    a.page_tokens = attrs.page_tokens;
    a.children = in[3].dims[0];
    a.new_table_pages = out[0].dims[1];
    a.ld_new_table = row_step(out[0]);
    return a;
}

NnopsKvCompactArgs compact_args(const KvCacheCompactAttributes& attrs, std::span<const TensorDesc> in,
                                std::span<const TensorDesc> out)
{
    NnopsKvCompactArgs a{};
    a.sequences = in[0].dims[0];
    a.table_pages = in[0].dims[1];
    a.ld_table = row_step(in[0]);
    a.pages = in[2].dims[0];
    a.page_tokens = attrs.page_tokens;
    a.ld_new_table = row_step(out[0]);
    return a;
}

}  // namespace

std::unique_ptr<KvCacheFork> KvCacheFork::create(const KvCacheForkAttributes& attrs, Backend backend)
{
    return std::unique_ptr<KvCacheFork>(new KvCacheFork(attrs, backend));
}

std::vector<TensorDesc> KvCacheFork::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.size() != 5 || inputs[0].rank != 2 || inputs[2].rank != 1 || inputs[3].rank != 1) {
        return {};
    }
    const int64_t n = inputs[3].dims[0];
    return {s32({n, inputs[0].dims[1]}), s32({n}), s32({inputs[2].dims[0]}), s32({n, 2}), s32({2})};
}

Status KvCacheFork::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() != 5 || outputs.size() != 5 || !all_s32(inputs) || !all_s32(outputs) || !tables_fit(inputs) ||
        inputs[3].rank != 1 || !same_shape(inputs[3], inputs[4])) {
        return Status::invalid_argument;
    }
    const std::vector<TensorDesc> want = getOutputTensorDesc(inputs);
    if (outputs[0].rank != 2 || outputs[0].dims[0] != want[0].dims[0]) {
        return Status::invalid_argument;
    }
    for (size_t i = 1; i < 5; ++i) {
        if (!same_shape(outputs[i], want[i])) {
            return Status::invalid_argument;
        }
    }
    if (!dense(outputs[3])) {
        return Status::unsupported;
    }
    const int64_t t = attrs_.page_tokens;
    return t == 16 || t == 32 || t == 64 || t == 128 || t == 256 ? Status::ok : Status::unsupported;
}

size_t KvCacheFork::getWorkspaceSize(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (!is_ok(validate(inputs, outputs))) {
        return 0;
    }
    const NnopsKvForkArgs a = fork_args(attrs_, inputs, outputs);
    return nnops_hip_kv_cache_fork_workspace_size(&a);
}

Status KvCacheFork::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                            const ComputeContext& ctx, void* workspace)
{
    std::array<TensorDesc, 5> in, out;
    if (!descs_of(inputs, in) || !descs_of(std::span<const TensorView>(outputs), out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size()), od(out.data(), outputs.size());
    if (Status s = validate(id, od); !is_ok(s)) {
        return s;
    }
    NnopsKvForkArgs a = fork_args(attrs_, id, od);
    a.page_table = inputs[0].ptr<const int32_t>();
    a.lengths = inputs[1].ptr<const int32_t>();
    a.refs = inputs[2].ptr<const int32_t>();
    a.parents = inputs[3].ptr<const int32_t>();
    a.new_tokens = inputs[4].ptr<const int32_t>();
    a.new_table = outputs[0].ptr<int32_t>();
    a.new_lengths = outputs[1].ptr<int32_t>();
    a.new_refs = outputs[2].ptr<int32_t>();
    a.copies = outputs[3].ptr<int32_t>();
    a.counts = outputs[4].ptr<int32_t>();
    const size_t bytes = nnops_hip_kv_cache_fork_workspace_size(&a);
    return from_abi(nnops_hip_kv_cache_fork(&a, workspace, workspace != nullptr ? bytes : 0, ctx.hip_stream));
}

std::unique_ptr<KvCacheCompact> KvCacheCompact::create(const KvCacheCompactAttributes& attrs, Backend backend)
{
    return std::unique_ptr<KvCacheCompact>(new KvCacheCompact(attrs, backend));
}

std::vector<TensorDesc> KvCacheCompact::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.size() != 3 || inputs[0].rank != 2 || inputs[2].rank != 1) {
        return {};
    }
    const int64_t pages = inputs[2].dims[0];
    return {s32({inputs[0].dims[0], inputs[0].dims[1]}), s32({pages}), s32({pages / 2, 2}), s32({pages}), s32({2})};
}

Status KvCacheCompact::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() != 3 || outputs.size() != 5 || !all_s32(inputs) || !all_s32(outputs) || !tables_fit(inputs)) {
        return Status::invalid_argument;
    }
    const std::vector<TensorDesc> want = getOutputTensorDesc(inputs);
    for (size_t i = 0; i < 5; ++i) {
        if (!same_shape(outputs[i], want[i])) {
            return Status::invalid_argument;
        }
    }
    if (!dense(outputs[2])) {
        return Status::unsupported;
    }
    const int64_t t = attrs_.page_tokens;
    return t == 16 || t == 32 || t == 64 || t == 128 || t == 256 ? Status::ok : Status::unsupported;
}

size_t KvCacheCompact::getWorkspaceSize(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (!is_ok(validate(inputs, outputs))) {
        return 0;
    }
    const NnopsKvCompactArgs a = compact_args(attrs_, inputs, outputs);
    return nnops_hip_kv_cache_compact_workspace_size(&a);
}

Status KvCacheCompact::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                               const ComputeContext& ctx, void* workspace)
{
    std::array<TensorDesc, 3> in;
    std::array<TensorDesc, 5> out;
    if (!descs_of(inputs, in) || !descs_of(std::span<const TensorView>(outputs), out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    const std::span<const TensorDesc> id(in.data(), inputs.size()), od(out.data(), outputs.size());
    if (Status s = validate(id, od); !is_ok(s)) {
        return s;
    }
    NnopsKvCompactArgs a = compact_args(attrs_, id, od);
    a.page_table = inputs[0].ptr<const int32_t>();
    a.lengths = inputs[1].ptr<const int32_t>();
    a.refs = inputs[2].ptr<const int32_t>();
    a.new_table = outputs[0].ptr<int32_t>();
    a.new_refs = outputs[1].ptr<int32_t>();
    a.copies = outputs[2].ptr<int32_t>();
    a.moved = outputs[3].ptr<int32_t>();
    a.counts = outputs[4].ptr<int32_t>();
    const size_t bytes = nnops_hip_kv_cache_compact_workspace_size(&a);
    return from_abi(nnops_hip_kv_cache_compact(&a, workspace, workspace != nullptr ? bytes : 0, ctx.hip_stream));
}

std::unique_ptr<KvCacheCopy> KvCacheCopy::create(Backend backend)
{
    return std::unique_ptr<KvCacheCopy>(new KvCacheCopy(backend));
}

std::vector<TensorDesc> KvCacheCopy::getOutputTensorDesc(std::span<const TensorDesc>) const { return {}; }

Status KvCacheCopy::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() != 1 || outputs.size() != 4 || !all_s32(inputs) || inputs[0].rank != 2 ||
        inputs[0].dims[1] != 2 || !all_plain(outputs)) {
        return Status::invalid_argument;
    }
    if (Status s = check_cache(outputs); !is_ok(s)) {
        return s;
    }
    const int64_t t = outputs[0].dims[2], d = outputs[0].dims[3];
    const bool sizes = (t == 16 || t == 32 || t == 64 || t == 128 || t == 256) && d >= 16 && d <= 256 && d % 16 == 0;
    return sizes && dense(inputs[0]) ? Status::ok : Status::unsupported;
}

Status KvCacheCopy::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                            const ComputeContext& ctx, void* workspace)
{
    (void)workspace;
    std::array<TensorDesc, 1> in;
    std::array<TensorDesc, 4> out;
    if (!descs_of(inputs, in) || !descs_of(std::span<const TensorView>(outputs), out)) {
        return Status::invalid_argument;
    }
    if (backend_ != Backend::HIP) {
        return Status::unsupported;
    }
    if (Status s = validate(std::span<const TensorDesc>(in.data(), inputs.size()),
                            std::span<const TensorDesc>(out.data(), outputs.size()));
        !is_ok(s)) {
        return s;
    }
    NnopsKvCopyArgs a{};
    a.k = outputs[0].ptr<int8_t>();
    a.v = outputs[1].ptr<int8_t>();
    a.k_scale = outputs[2].ptr<float>();
    a.v_scale = outputs[3].ptr<float>();
    a.pages = out[0].dims[0];
    a.heads = out[0].dims[1];
    a.page_tokens = out[0].dims[2];
    a.head_dim = out[0].dims[3];
    a.copies = inputs[0].ptr<const int32_t>();
    a.count = in[0].dims[0];
    return from_abi(nnops_hip_kv_cache_copy(&a, ctx.hip_stream));
}

}  // namespace nnops

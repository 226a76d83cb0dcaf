// TokenLogProbs for Backend::HIP: descriptor rules, lowered onto
// nnops_hip_token_log_probs.
#include "nnops/ops/token_log_probs.hpp"
#include "nnops_amd.h"
#include "views.hpp"

namespace nnops {
namespace {

NnopsTokenLogProbsArgs args_of(const TokenLogProbsAttributes& attrs, std::span<const TensorDesc> in,
                               std::span<const TensorDesc> out)
{
    NnopsTokenLogProbsArgs a{};
    a.rows = in[0].dims[0];
    a.vocab = in[0].dims[1];
    a.ld_logits = row_step(in[0]);
    a.f16 = in[0].dtype == DataType::f16;
    a.top = static_cast<int32_t>(attrs.top);
    a.per_row = in[1].rank == 2 ? in[1].dims[1] : 1;
    a.ld_tokens = in[1].rank == 2 ? row_step(in[1]) : 1;
    a.ld_log_probs = out[0].rank == 2 ? row_step(out[0]) : 1;
    if (attrs.top > 0) {
        a.ld_top_tokens = row_step(out[2]);
        a.ld_top_log_probs = row_step(out[3]);
    }
    return a;
}

}  // namespace

std::unique_ptr<TokenLogProbs> TokenLogProbs::create(const TokenLogProbsAttributes& attrs, Backend backend)
{
    return std::unique_ptr<TokenLogProbs>(new TokenLogProbs(attrs, backend));
}

std::vector<TensorDesc> TokenLogProbs::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.size() != 2 || inputs[0].rank != 2) {
        return {};
    }
    TensorDesc lp = inputs[1];
    lp.dtype = DataType::f32;
    lp.row_stride_elems = 0;
    TensorDesc entropy;
    entropy.rank = 1;
    entropy.dims[0] = inputs[0].dims[0];
    std::vector<TensorDesc> out{lp, entropy};
    if (attrs_.top > 0) {
        TensorDesc top = entropy;
        top.rank = 2;
        top.dims[1] = attrs_.top;
        out.push_back(top);
        out[2].dtype = DataType::s32;
        out.push_back(top);
    }
    return out;
}

Status TokenLogProbs::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() != 2 || !all_plain(inputs) || !all_plain(outputs) || attrs_.top < 0 || inputs[0].rank != 2 ||
        (inputs[1].rank != 1 && inputs[1].rank != 2) || inputs[1].dims[0] != inputs[0].dims[0] ||
        inputs[1].dtype != DataType::s32 || attrs_.top > inputs[0].dims[1]) {
        return Status::invalid_argument;
    }
    const std::vector<TensorDesc> want = getOutputTensorDesc(inputs);
    if (outputs.size() != want.size()) {
        return Status::invalid_argument;
    }
    for (size_t i = 0; i < want.size(); ++i) {
        if (!same_shape(outputs[i], want[i]) || outputs[i].dtype != want[i].dtype) {
            return Status::invalid_argument;
        }
    }
    const int64_t rows = inputs[0].dims[0], vocab = inputs[0].dims[1];
    const bool sizes = attrs_.top <= 32 && vocab <= (1 << 21) && rows <= (1 << 22) &&
                       rows * ((vocab + 32767) / 32768) < (1 << 23);
    return is_float(inputs[0].dtype) && sizes ? Status::ok : Status::unsupported;
}

size_t TokenLogProbs::getWorkspaceSize(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (!is_ok(validate(inputs, outputs))) {
        return 0;
    }
    const NnopsTokenLogProbsArgs a = args_of(attrs_, inputs, outputs);
    return nnops_hip_token_log_probs_workspace_size(&a);
}

Status TokenLogProbs::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                              const ComputeContext& ctx, void* workspace)
{
    std::array<TensorDesc, 2> in;
    std::array<TensorDesc, 4> out;
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
    NnopsTokenLogProbsArgs a = args_of(attrs_, id, od);
    a.logits = inputs[0].ptr<const void>();
    a.tokens = inputs[1].ptr<const int32_t>();
    a.log_probs = outputs[0].ptr<float>();
    a.entropy = outputs[1].ptr<float>();
    if (attrs_.top > 0) {
        a.top_tokens = outputs[2].ptr<int32_t>();
        a.top_log_probs = outputs[3].ptr<float>();
    }
    const size_t bytes = nnops_hip_token_log_probs_workspace_size(&a);
    return from_abi(nnops_hip_token_log_probs(&a, workspace, workspace != nullptr ? bytes : 0, ctx.hip_stream));
}

}  // namespace nnops

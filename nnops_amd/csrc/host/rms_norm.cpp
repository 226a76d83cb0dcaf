// RmsNorm and Rotary for Backend::HIP: descriptor rules, lowered onto
// nnops_hip_rms_norm / nnops_hip_rotary.
#include "nnops/ops/rms_norm.hpp"
#include "nnops/ops/rotary.hpp"
#include "nnops_amd.h"
#include "views.hpp"

namespace nnops {

std::unique_ptr<RmsNorm> RmsNorm::create(const RmsNormAttributes& attrs, Backend backend)
{
    return std::unique_ptr<RmsNorm>(new RmsNorm(attrs, backend));
}

std::vector<TensorDesc> RmsNorm::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.size() < 2 || inputs.size() > 3 || inputs[0].rank < 1) {
        return {};
    }
    TensorDesc x = inputs[0];
    x.row_stride_elems = 0;
    TensorDesc y = x;
    y.dtype = attrs_.output_dtype;
    std::vector<TensorDesc> out{y};
    if (attrs_.output_dtype == DataType::s8) {
        TensorDesc s;
        s.rank = 1;
        s.dims[0] = x.rows();
        s.dtype = DataType::f32;
        out.push_back(s);
    }
    if (inputs.size() == 3) {
        out.push_back(x);
    }
    return out;
}

Status RmsNorm::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    if (inputs.size() < 2 || inputs.size() > 3 || !(attrs_.epsilon >= 0.0f)) {
        return Status::invalid_argument;
    }
    const bool s8 = attrs_.output_dtype == DataType::s8, res = inputs.size() == 3;
    if (outputs.size() != 1u + (s8 ? 1u : 0u) + (res ? 1u : 0u)) {
        return Status::invalid_argument;
    }
    for (const TensorDesc& d : inputs) {
        if (!plain_dims(d)) {
            return Status::invalid_argument;
        }
    }
    for (const TensorDesc& d : outputs) {
        if (!plain_dims(d)) {
            return Status::invalid_argument;
        }
    }
    const TensorDesc& x = inputs[0];
    if (x.rank < 1 || inputs[1].rank != 1 || inputs[1].dims[0] != x.cols()) {
        return Status::invalid_argument;
    }
    if (!is_float(x.dtype) || (!s8 && attrs_.output_dtype != x.dtype)) {
        return Status::unsupported;
    }
    if (inputs[1].dtype != x.dtype || (res && (inputs[2].dtype != x.dtype || !same_shape(inputs[2], x)))) {
        return Status::invalid_argument;
    }
    if (outputs[0].dtype != attrs_.output_dtype || !same_shape(outputs[0], x)) {
        return Status::invalid_argument;
    }
    if (s8 && (outputs[1].dtype != DataType::f32 || outputs[1].numel() != x.rows() || !dense(outputs[1]))) {
        return Status::invalid_argument;
    }
    if (res && (outputs.back().dtype != x.dtype || !same_shape(outputs.back(), x))) {
        return Status::invalid_argument;
    }
    return Status::ok;
}

Status RmsNorm::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                        const ComputeContext& ctx, void* workspace)
{
    (void)workspace;
    std::array<TensorDesc, 3> in, out;
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
    const bool s8 = attrs_.output_dtype == DataType::s8, res = inputs.size() == 3;
    NnopsRmsNormArgs a{};
    a.x = inputs[0].ptr<const void>();
    a.weight = inputs[1].ptr<const void>();
    a.rows = in[0].rows();
    a.cols = in[0].cols();
    a.ld_x = row_step(in[0]);
    a.y = outputs[0].ptr<void>();
    a.ld_y = row_step(out[0]);
    if (s8) {
        a.scale = outputs[1].ptr<float>();
    }
    if (res) {
        a.residual = inputs[2].ptr<const void>();
        a.ld_residual = row_step(in[2]);
        a.sum = outputs.back().ptr<void>();
        a.ld_sum = row_step(out[outputs.size() - 1]);
    }
    a.in_f16 = in[0].dtype == DataType::f16;
    a.out_kind = s8 ? NNOPS_OUT_S8 : a.in_f16 ? NNOPS_OUT_F16 : NNOPS_OUT_F32;
    a.epsilon = attrs_.epsilon;
    return from_abi(nnops_hip_rms_norm(&a, ctx.hip_stream));
}

std::unique_ptr<Rotary> Rotary::create(const RotaryAttributes& attrs, Backend backend)
{
    return std::unique_ptr<Rotary>(new Rotary(attrs, backend));
}

std::vector<TensorDesc> Rotary::getOutputTensorDesc(std::span<const TensorDesc> inputs) const
{
    if (inputs.empty()) {
        return {};
    }
    TensorDesc y = inputs[0];
    y.row_stride_elems = 0;
    return {y};
}

Status Rotary::validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const
{
    const int64_t d = attrs_.head_dim, rot = attrs_.rotary_dim == 0 ? d : attrs_.rotary_dim;
    if (inputs.size() != 3 || outputs.size() != 1 || d <= 0 || rot <= 0 || rot % 2 != 0 || rot > d) {
        return Status::invalid_argument;
    }
    const TensorDesc &x = inputs[0], &pos = inputs[1], &table = inputs[2], &y = outputs[0];
    if (!plain_dims(x) || !plain_dims(pos) || !plain_dims(table) || !plain_dims(y)) {
        return Status::invalid_argument;
    }
    if (x.rank != 2 || x.cols() % d != 0 || pos.rank != 1 || pos.dims[0] != x.dims[0] || table.rank != 2 ||
        table.dims[0] < 1 || table.dims[1] != rot) {
        return Status::invalid_argument;
    }
    if (!is_float(x.dtype)) {
        return Status::unsupported;
    }
    if (pos.dtype != DataType::s32 || table.dtype != DataType::f32 || y.dtype != x.dtype || !same_shape(x, y)) {
        return Status::invalid_argument;
    }
    return Status::ok;
}

Status Rotary::compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                       const ComputeContext& ctx, void* workspace)
{
    (void)workspace;
    std::array<TensorDesc, 3> in;
    std::array<TensorDesc, 1> out;
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
    NnopsRotaryArgs a{};
    a.x = inputs[0].ptr<const void>();
    a.y = outputs[0].ptr<void>();
    a.positions = inputs[1].ptr<const int32_t>();
    a.table = inputs[2].ptr<const float>();
    a.tokens = in[0].dims[0];
    a.heads = in[0].dims[1] / attrs_.head_dim;
    a.head_dim = attrs_.head_dim;
    a.rotary_dim = attrs_.rotary_dim == 0 ? attrs_.head_dim : attrs_.rotary_dim;
    a.max_pos = in[2].dims[0];
    a.ld_x = row_step(in[0]);
    a.ld_y = row_step(out[0]);
    a.ld_table = row_step(in[2]);
    a.in_f16 = in[0].dtype == DataType::f16;
    a.interleaved = attrs_.interleaved;
    return from_abi(nnops_hip_rotary(&a, ctx.hip_stream));
}

}  // namespace nnops

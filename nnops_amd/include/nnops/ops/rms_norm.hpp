#pragma once
/// @file rms_norm.hpp
/// @brief RmsNorm — root-mean-square norm with the residual's addition, on the
/// HIP backend (no counterpart in nnops).
///
/// inputs:  x [.., C] (f16 / f32), weight [C] (x's type) [, residual, x's shape
///          and type]
/// outputs: y (x's shape) [, scale f32 [rows], with an s8 y] [, sum = x +
///          residual, x's shape and type, with a residual]
///   h = x + residual;  y = h / sqrt(mean(h^2) + epsilon) * weight
/// in f32, rounded once. An s8 y holds codes of one scale per row, the
/// PerToken activation that Linear / MatMul take:
///   a = max |h weight|, code = rint(h weight (127 / a)),
///   scale = a / 127 / sqrt(mean(h^2) + epsilon).
/// sum may be x's or the residual's buffer, with its row pitch.

#include "nnops/core/op_base.hpp"

#include <memory>

namespace nnops {

struct RmsNormAttributes {
    float epsilon = 1e-6f;
    DataType output_dtype = DataType::f16;  ///< x's type, or s8
};

class RmsNorm : public OpBase {
public:
    static std::unique_ptr<RmsNorm> create(const RmsNormAttributes& attrs = {}, Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const RmsNormAttributes& attributes() const noexcept { return attrs_; }

private:
    RmsNorm(const RmsNormAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    RmsNormAttributes attrs_;
    Backend backend_;
};

}  // namespace nnops

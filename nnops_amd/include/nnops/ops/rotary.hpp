#pragma once
/// @file rotary.hpp
/// @brief Rotary — rotary positions over the heads of each row, on the HIP
/// backend (no counterpart in nnops).
///
/// inputs:  x [tokens, heads * head_dim] (f16 / f32, any row pitch: the q and k
///          columns of a fused projection in one call), positions s32 [tokens],
///          table f32 [max_pos, rotary_dim] (cosines, then sines;
///          nnops_hip_rotary_table fills one)
/// output:  y, x's shape and type; may be x itself
///   (y_a, y_b) = (x_a c - x_b s, x_b c + x_a s) over the first rotary_dim
///   values of each head, pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when
///   interleaved; the others are copied. A position outside the table gives NaN.

#include "nnops/core/op_base.hpp"

#include <memory>

namespace nnops {

struct RotaryAttributes {
    int64_t head_dim = 0;
    int64_t rotary_dim = 0;  ///< even, at most head_dim; 0: head_dim
    bool interleaved = false;
};

class Rotary : public OpBase {
public:
    static std::unique_ptr<Rotary> create(const RotaryAttributes& attrs, Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const RotaryAttributes& attributes() const noexcept { return attrs_; }

private:
    Rotary(const RotaryAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    RotaryAttributes attrs_;
    Backend backend_;
};

}  // namespace nnops

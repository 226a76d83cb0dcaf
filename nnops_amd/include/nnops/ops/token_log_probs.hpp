#pragma once
/// @file token_log_probs.hpp
/// @brief TokenLogProbs — log probabilities of given tokens, the entropy and the
/// most probable tokens of rows of logits, on the HIP backend (no counterpart in
/// nnops).

#include "nnops/core/op_base.hpp"

#include <memory>

namespace nnops {

struct TokenLogProbsAttributes {
    int64_t top = 0;            ///< alternatives, 0 to 32
};

/// inputs:  logits [T, V] (f16 / f32, V up to 2^21), tokens s32 [T, n] (or [T])
/// outputs: log_probs f32 of tokens' shape, entropy f32 [T] and, with top > 0,
///          top_tokens s32 [T, top], top_log_probs f32 [T, top]
class TokenLogProbs : public OpBase {
public:
    static std::unique_ptr<TokenLogProbs> create(const TokenLogProbsAttributes& attrs = {},
                                                 Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    size_t getWorkspaceSize(std::span<const TensorDesc> inputs,
                            std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const TokenLogProbsAttributes& attributes() const noexcept { return attrs_; }

private:
    TokenLogProbs(const TokenLogProbsAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    TokenLogProbsAttributes attrs_;
    Backend backend_;
};

}  // namespace nnops

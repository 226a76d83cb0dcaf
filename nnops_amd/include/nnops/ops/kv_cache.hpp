#pragma once
/// @file kv_cache.hpp
/// @brief KvCacheWrite, KvCacheRead, CacheAttention, PrefixAttention — a key / value
/// cache held in 8 bits, and attention over it, on the HIP backend (no counterpart
/// in nnops).
///
/// The cache's tensors (dense, 16-byte aligned codes):
///   k_cache s8 [pages, heads, page_tokens, head_dim]
///   v_cache s8 [pages, heads, head_dim, page_tokens]
///   k_scale, v_scale f32 [pages, heads]: value = code * scale
/// page_tokens: 16, 32, 64, 128 or 256; head_dim: a multiple of 16 up to 256.
/// The tables, device memory that the host does not read:
///   page_table s32 [sequences, table_pages]; lengths s32 [sequences], the
///   tokens that each sequence holds, this call's among them; row_starts s32
///   [sequences + 1], optional: sequence b has rows row_starts[b] up to
///   row_starts[b + 1] - 1 of the call (without it, as many each). A sequence's
///   rows are its last tokens.
/// A page table may be wider than any sequence: attention's launch, workspace and
/// choice of kernel go by the longest sequence that the table has room for, the
/// division of the work by the longest that there is.

#include "nnops/core/op_base.hpp"

#include <memory>

namespace nnops {

/// inputs:  k, v [rows, heads * head_dim] (f16 / f32), page_table, lengths
///          [, row_starts]
/// outputs: k_cache, v_cache, k_scale, v_scale, updated in place: per page and
///          head scale = max(old, max |new| / 127), codes rint(x / scale), the
///          page's older codes brought to a scale that grew.
class KvCacheWrite : public OpBase {
public:
    static std::unique_ptr<KvCacheWrite> create(Backend backend = Backend::HIP);

    /// Empty: the outputs are the caller's cache.
    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }

private:
    explicit KvCacheWrite(Backend backend) : backend_(backend) {}
    Backend backend_;
};

struct KvCacheReadAttributes {
    DataType output_dtype = DataType::f16;  ///< f16 / f32
};

/// inputs:  k_cache, v_cache, k_scale, v_scale, page_table, lengths
///          [, row_starts]
/// outputs: k, v [rows, heads * head_dim]: the last tokens of each sequence, as
///          many as it has rows
class KvCacheRead : public OpBase {
public:
    static std::unique_ptr<KvCacheRead> create(const KvCacheReadAttributes& attrs = {},
                                               Backend backend = Backend::HIP);

    /// Empty: the rows to read are the outputs'.
    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const KvCacheReadAttributes& attributes() const noexcept { return attrs_; }

private:
    KvCacheRead(const KvCacheReadAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    KvCacheReadAttributes attrs_;
    Backend backend_;
};

struct CacheAttentionAttributes {
    float scale = 0.0f;   ///< of the scores; 0: 1 / sqrt(head_dim)
    int64_t window = 0;   ///< last tokens that a query sees, itself among them; 0: all
    int64_t sinks = 0;    ///< first tokens of the sequence that stay visible
};

/// inputs:  q [rows, q_heads * head_dim] (f16 / f32; q_heads a multiple of the
///          cache's heads), k_cache, v_cache, k_scale, v_scale, page_table,
///          lengths [, row_starts]
/// output:  q's shape and type. Causal: a query sees the tokens up to its own,
///          which KvCacheWrite has put into the cache.
class CacheAttention : public OpBase {
public:
    static std::unique_ptr<CacheAttention> create(const CacheAttentionAttributes& attrs = {},
                                                  Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    size_t getWorkspaceSize(std::span<const TensorDesc> inputs,
                            std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const CacheAttentionAttributes& attributes() const noexcept { return attrs_; }

private:
    CacheAttention(const CacheAttentionAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    CacheAttentionAttributes attrs_;
    Backend backend_;
};

struct PrefixAttentionAttributes {
    float scale = 0.0f;   ///< of the scores; 0: 1 / sqrt(head_dim)
};

/// inputs:  q [rows, q_heads * head_dim] (f16 / f32; q_heads a multiple of the
///          cache's heads), k_cache, v_cache, k_scale, v_scale, page_table,
///          lengths, group_starts s32 [groups + 1], shared s32 [groups]
///          [, row_starts]
/// output:  q's shape and type: CacheAttention's (without a window) for groups of
///          sequences, group g those from group_starts[g] up to group_starts[g + 1]
///          - 1, whose first shared[g] tokens lie in the same pages (as far as they
///          fill whole pages): read once for the group.
class PrefixAttention : public OpBase {
public:
    static std::unique_ptr<PrefixAttention> create(const PrefixAttentionAttributes& attrs = {},
                                                   Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    size_t getWorkspaceSize(std::span<const TensorDesc> inputs,
                            std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const PrefixAttentionAttributes& attributes() const noexcept { return attrs_; }

private:
    PrefixAttention(const PrefixAttentionAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    PrefixAttentionAttributes attrs_;
    Backend backend_;
};

}  // namespace nnops

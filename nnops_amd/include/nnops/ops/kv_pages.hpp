#pragma once
/// @file kv_pages.hpp
/// @brief KvCacheFork, KvCacheCompact, KvCacheCopy — the page tables of a batch's
/// continuations over the paged cache of kv_cache.hpp, on the HIP backend (no
/// counterpart in nnops).
///
/// refs s32 [pages] counts the sequences that hold a page (and whoever else the
/// caller counts); 0: free. A sequence holds the pages of its first
/// ceil(length / page_tokens) cells of page_table. A table serves all layers: the
/// copies that fork and compact ask for are made in each layer's cache.
///
/// validate looks at shapes and types; how large they may be (16384 sequences and
/// children, a new table of 2^30 cells) the call says: Status::unsupported.

#include "nnops/core/op_base.hpp"

#include <memory>

namespace nnops {

struct KvCacheForkAttributes {
    int64_t page_tokens = 64;   ///< 16, 32, 64, 128 or 256
};

/// inputs:  page_table s32 [B, P], lengths s32 [B], refs s32 [pages], parents s32
///          [N] (-1: none), new_tokens s32 [N]
/// outputs: page_table s32 [N, any], lengths s32 [N], refs s32 [pages] (the
///          input's view if wanted), copies s32 [N, 2], counts s32 [2]
/// The B sequences are given up, N children of them take their place: they share
/// their parents' pages and get fresh ones for new_tokens more; a page that they
/// would write into and that others hold is replaced, and to be copied.
class KvCacheFork : public OpBase {
public:
    static std::unique_ptr<KvCacheFork> create(const KvCacheForkAttributes& attrs = {},
                                               Backend backend = Backend::HIP);

    /// (a table as wide as the input's)
    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    size_t getWorkspaceSize(std::span<const TensorDesc> inputs,
                            std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const KvCacheForkAttributes& attributes() const noexcept { return attrs_; }

private:
    KvCacheFork(const KvCacheForkAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    KvCacheForkAttributes attrs_;
    Backend backend_;
};

struct KvCacheCompactAttributes {
    int64_t page_tokens = 64;   ///< 16, 32, 64, 128 or 256
};

/// inputs:  page_table s32 [B, P], lengths s32 [B], refs s32 [pages]
/// outputs: page_table s32 [B, P] and refs s32 [pages] (the inputs' views if
///          wanted), copies s32 [pages / 2, 2], moved s32 [pages], counts s32 [2]
/// The pages in use are moved to the lowest numbers.
class KvCacheCompact : public OpBase {
public:
    static std::unique_ptr<KvCacheCompact> create(const KvCacheCompactAttributes& attrs = {},
                                                  Backend backend = Backend::HIP);

    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    size_t getWorkspaceSize(std::span<const TensorDesc> inputs,
                            std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }
    const KvCacheCompactAttributes& attributes() const noexcept { return attrs_; }

private:
    KvCacheCompact(const KvCacheCompactAttributes& attrs, Backend backend) : attrs_(attrs), backend_(backend) {}
    KvCacheCompactAttributes attrs_;
    Backend backend_;
};

/// inputs:  copies s32 [any, 2]: pages to copy from and to (a pair with a number
///          that is no page is skipped)
/// outputs: k_cache, v_cache, k_scale, v_scale, updated in place
class KvCacheCopy : public OpBase {
public:
    static std::unique_ptr<KvCacheCopy> create(Backend backend = Backend::HIP);

    /// Empty: the outputs are the caller's cache.
    std::vector<TensorDesc> getOutputTensorDesc(std::span<const TensorDesc> inputs) const override;
    Status validate(std::span<const TensorDesc> inputs, std::span<const TensorDesc> outputs) const override;
    using OpBase::compute;
    Status compute(std::span<TensorView> outputs, std::span<const TensorView> inputs,
                   const ComputeContext& ctx = {}, void* workspace = nullptr) override;
    Backend getBackend() const override { return backend_; }

private:
    explicit KvCacheCopy(Backend backend) : backend_(backend) {}
    Backend backend_;
};

}  // namespace nnops

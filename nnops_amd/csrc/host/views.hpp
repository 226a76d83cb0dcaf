// What the operators around the products share on the host: checks of views
// and descriptors, and the C ABI's status as a Status.
#pragma once

#include "nnops/core/status.hpp"
#include "nnops/core/tensor_view.hpp"
#include "nnops_amd.h"

#include <array>
#include <span>

namespace nnops {

inline Status from_abi(int code)
{
    switch (code) {
    case NNOPS_OK: return Status::ok;
    case NNOPS_INVALID_ARGUMENT: return Status::invalid_argument;
    case NNOPS_UNSUPPORTED: return Status::unsupported;
    case NNOPS_NOT_INITIALIZED: return Status::not_initialized;
    case NNOPS_OUT_OF_MEMORY: return Status::out_of_memory;
    default: return Status::internal;
    }
}

inline bool is_float(DataType dt) { return dt == DataType::f16 || dt == DataType::f32; }

inline bool same_shape(const TensorDesc& a, const TensorDesc& b)
{
    if (a.rank != b.rank) {
        return false;
    }
    for (int64_t i = 0; i < a.rank; ++i) {
        if (a.dims[static_cast<size_t>(i)] != b.dims[static_cast<size_t>(i)]) {
            return false;
        }
    }
    return true;
}

/// Elements between rows (a compact descriptor's are its columns).
inline int64_t row_step(const TensorDesc& d)
{
    return d.rank < 2 || d.row_stride_elems == 0 ? d.cols() : d.row_stride_elems;
}

inline bool dense(const TensorDesc& d) { return row_step(d) == d.cols(); }

inline bool plain_dims(const TensorDesc& d)
{
    for (int64_t i = 0; i < d.rank; ++i) {
        if (d.dims[static_cast<size_t>(i)] < 0) {
            return false;
        }
    }
    return d.layout == TensorLayout::Dense && row_step(d) >= d.cols();
}

/// A view that memory can be reached through: it has data where it has
/// elements, and whole elements between its rows.
inline bool reachable(const TensorView& v)
{
    const int64_t unit = static_cast<int64_t>(data_type_size(v.data_type()));
    return (!v.is_empty() || v.numel() == 0) && (v.rank() < 2 || (unit > 0 && v.pitch() % unit == 0));
}

/// The descriptors of a call's views; false where a view cannot be reached.
template <size_t N>
bool descs_of(std::span<const TensorView> views, std::array<TensorDesc, N>& d)
{
    if (views.size() > N) {
        return false;
    }
    for (size_t i = 0; i < views.size(); ++i) {
        if (!reachable(views[i])) {
            return false;
        }
        d[i] = views[i].desc();
    }
    return true;
}

inline bool all_plain(std::span<const TensorDesc> d)
{
    for (const TensorDesc& t : d) {
        if (!plain_dims(t)) {
            return false;
        }
    }
    return true;
}

/// The four tensors of a paged cache.
inline Status check_cache(std::span<const TensorDesc> c)
{
    const TensorDesc &k = c[0], &v = c[1], &ks = c[2], &vs = c[3];
    if (k.rank != 4 || v.rank != 4 || ks.rank != 2 || vs.rank != 2) {
        return Status::invalid_argument;
    }
    if (k.dtype != DataType::s8 || v.dtype != DataType::s8 || ks.dtype != DataType::f32 ||
        vs.dtype != DataType::f32) {
        return Status::invalid_argument;
    }
    if (v.dims[0] != k.dims[0] || v.dims[1] != k.dims[1] || v.dims[2] != k.dims[3] || v.dims[3] != k.dims[2] ||
        ks.dims[0] != k.dims[0] || ks.dims[1] != k.dims[1] || !same_shape(ks, vs)) {
        return Status::invalid_argument;
    }
    return dense(k) && dense(v) && dense(ks) && dense(vs) ? Status::ok : Status::unsupported;
}

}  // namespace nnops

// Shared by the row-wise operators: the last dimension of a tensor as its rows.
#pragma once

#include <cstddef>
#include <string>

#include <motifcl/core/error.hpp>
#include <motifcl/tensor/tensor.hpp>
#include <motifcl_amd.h>

namespace motifcl::rows {

inline int element_of(const Tensor& t, const std::string& what) {
    MCL_CHECK(t.dtype() == DType::F32 || t.dtype() == DType::F16, what + " supports f32 and f16 only");
    return t.dtype() == DType::F32 ? MCC_ELEMENT_F32 : MCC_ELEMENT_F16;
}
inline Shape leading(const Tensor& t, const std::string& what) {
    MCL_CHECK(t.ndim() >= 1, what + " requires at least one dimension");
    return Shape(std::vector<int64_t>(t.shape().dims.begin(), t.shape().dims.end() - 1));
}
inline std::size_t length(const Tensor& t) { return static_cast<std::size_t>(t.shape()[-1]); }
// numbers of one a row (or `more` a row) on the same backend
inline void check_numbers(const Tensor& t, const Tensor& like, DType dtype, const Shape& shape, const std::string& what) {
    MCL_CHECK(t.dtype() == dtype, what + " has the wrong type");
    MCL_CHECK(t.shape() == shape, what + " shape mismatch");
    MCL_CHECK(t.backend_ptr() == like.backend_ptr(), what + " is on another backend");
}
inline float* f32(const Tensor& t) { return static_cast<float*>(t.data()); }

}  // namespace motifcl::rows

// Helpers shared by the sources of flash_kmeans_cuda._C.
#pragma once

#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <stdexcept>
#include <string>

#include "fkc_capi.h"

namespace fkc_py {

inline void require(bool ok, const char* msg) {
  if (!ok) throw std::runtime_error(msg);
}

inline void check_status(int status, const char* what) {
  if (status != FKC_OK)
    throw std::runtime_error(std::string(what) + ": " + fkc_status_string(status) + ": " +
                             fkc_last_error());
}

inline int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return FKC_DTYPE_F16;
    case at::kBFloat16: return FKC_DTYPE_BF16;
    case at::kFloat: return FKC_DTYPE_F32;
    default:
      throw std::runtime_error(std::string("unsupported dtype ") +
                               c10::toString(t.scalar_type()) +
                               " (expected float16, bfloat16 or float32)");
  }
}

inline fkc_stream_t stream_of(const at::Tensor& t) {
  return reinterpret_cast<fkc_stream_t>(
      at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// Operators on clustered rows (py_clusters.cpp).
void bind_clusters(py::module_& m);

}  // namespace fkc_py

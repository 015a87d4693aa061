// What the operator shim's source files share: error and stream plumbing between ATen and the C ABI.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <string>

#include "../../../include/b2rt.h"

namespace {

inline std::string b2_error() {
  char buf[1024];
  b2rt_last_error(buf, sizeof(buf));
  return std::string(buf);
}

inline void b2_check(int rc, const char* what) { TORCH_CHECK(rc == 0, "b200 ", what, " failed: ", b2_error()); }

inline void count(const char* name) { b2rt_count_op(name); }
[[maybe_unused]] inline void count_fallback(const std::string& name) { b2rt_count_op(("fallback:" + name).c_str()); }

inline b2_stream_t cur_stream() { return (b2_stream_t)at::cuda::getCurrentCUDAStream().stream(); }

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B2_F32;
    case at::kBFloat16: return B2_BF16;
    case at::kHalf: return B2_F16;
    case at::kDouble: return B2_F64;
    default: return -1;
  }
}
inline bool is_row_dtype(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

}  // namespace

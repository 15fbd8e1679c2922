// Helpers shared by the compiled host layers of attention (host_ops.cpp) and of
// the training operators (train_ops.cpp).
#pragma once

#include <torch/extension.h>

#include <cstdint>
#include <sstream>
#include <string>
#include <utility>

#include "sageattn_mi355x.h"

namespace py = pybind11;

namespace sage_host {

// A negative status of the C ABI, raised in Python as the exception type the
// package registers (sageattention._capi.SageError: function, status, message).
struct SageStatus {
  const char* fn;
  int code;
  std::string msg;
};

inline void check(const char* fn, int rc) {
  if (rc != SAGE_OK) {
    const char* m = sage_last_error();
    throw SageStatus{fn, rc, m != nullptr ? m : ""};
  }
}

// (B, H, N, D) sizes and (b, h, n) strides in elements of a 4-D tensor;
// layout 1 = HND [B,H,N,D], 0 = NHD [B,N,H,D] (reference csrc/attn_gfx11.cu:32-33)
struct Dims {
  int64_t b, h, n, d;
  int64_t sb, sh, sn;
};

inline Dims bhnd(const at::Tensor& t, int64_t layout) {
  const auto s = t.sizes();
  const auto st = t.strides();
  if (layout == 1) return {s[0], s[1], s[2], s[3], st[0], st[1], st[2]};
  return {s[0], s[2], s[1], s[3], st[0], st[2], st[1]};
}

// t, or a copy that meets the 16-byte access contract (16-byte aligned base,
// batch/head/token strides multiples of 8 elements; a plain clone would keep
// the odd stride of a dimension of one element)
inline at::Tensor vector_ready(const at::Tensor& t) {
  const auto st = t.strides();
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

inline std::string shape_str(const at::Tensor& t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << ")";
  return s.str();
}

inline void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// sageattn's forward after its checks (host_ops.cpp); the LSE is undefined unless return_lse
std::pair<at::Tensor, at::Tensor> attn_fwd(at::Tensor q, at::Tensor k, at::Tensor v, int64_t layout, bool is_causal,
                                           double sm_scale, bool return_lse, bool smooth_k, bool direct,
                                           int64_t num_splits, void* stream);

// the training operators' functions (train_ops.cpp)
void bind_train(py::module_& m);

}  // namespace sage_host

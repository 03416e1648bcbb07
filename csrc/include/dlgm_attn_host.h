// Argument checks of the shared-key attention operators (shared_attn.hip, shared_decode.hip): everything a kernel
// assumes about its operands is checked here, on the host, before a launch.
#pragma once

#include <torch/all.h>
#include "dlgm_common.h"

namespace dlgm {

constexpr int kThreads = 256;  // of a workgroup, where a kernel does not say otherwise

inline void check_rows(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name, int dim) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on the device of q");
  TORCH_CHECK(DLGM_IS16(t) && t.scalar_type() == like.scalar_type(), op, ": ", name,
              " must be bf16 or fp16, one type for all tensors");
  TORCH_CHECK(t.dim() == dim && (t.numel() == 0 || t.stride(dim - 1) == 1), op, ": ", name, " must have ", dim,
              " dimensions, the last one with unit stride");
  for (int i = 0; i + 1 < dim; ++i)
    TORCH_CHECK(t.size(i) <= 1 || t.stride(i) % 8 == 0, op, ": ", name, " strides must keep 16-byte alignment");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, op, ": ", name, " must be 16-byte aligned");
  // a 128-row tile is addressed with 32-bit byte offsets from its own base
  const int rd = dim == 2 ? 0 : 1;
  TORCH_CHECK(t.size(rd) <= 1 || t.stride(rd) < (int64_t)1 << 23, op, ": ", name, " row stride is too large");
}

// The stride of dimension i as the kernels use it. Of a dimension of one it may be anything (1 for a permuted [B, H, D, 1]):
// rows a tile has beyond it are then placed a row's width apart, behind the end of the one that exists, where a descriptor
// gives zeros and every address stays aligned.
inline int64_t stride_of(const at::Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : t.size(t.dim() - 1); }

inline const int* check_lens(const c10::optional<at::Tensor>& lens, const at::Tensor& like, int64_t n, const char* op,
                             const char* name) {
  if (!lens.has_value() || !lens->defined()) return nullptr;
  TORCH_CHECK(lens->device() == like.device() && lens->scalar_type() == at::kInt && lens->is_contiguous() &&
                  lens->dim() == 1 && lens->numel() == n,
              op, ": ", name, " must be a contiguous int32 tensor of ", n, " lengths on the device of q");
  return lens->data_ptr<int>();
}

// the backward starts its scores from -lse / scale, in fp32
inline void check_scale(double s, const char* op) {
  TORCH_CHECK(s >= 1e-20 && s <= 1e20, op, ": softmax_scale must lie between 1e-20 and 1e20, got ", s);
}

// HIP needs gridDim.x * blockDim.x below 2^32
inline int64_t check_blocks(int64_t n, const char* op) {
  TORCH_CHECK(n <= (int64_t)(UINT32_MAX / kThreads), op, ": too many rows for one launch");
  return n;
}

template <typename E>
E* ptr(const at::Tensor& t) {
  return reinterpret_cast<E*>(t.data_ptr());
}

}  // namespace dlgm

// Helpers shared by the torch.ops.vlak translation units.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>

#include <initializer_list>

#include "vlak_b200.h"

namespace vlak_torch {

inline void check_status(int status, const char* op) {
  TORCH_CHECK(status == VLAK_OK, op, ": ", vlak_last_error_message(), " (",
              vlak_status_string(status), ")");
}

// Every op first reads the host-mapped error word (no device
// synchronization): a bounded wait that ran out in an attention kernel which
// has finished since is raised here, on the caller's next op, instead of
// going unnoticed. The word is cleared by the read, so the following call
// runs normally.
inline void raise_pending_device_error(const char* op) {
  int code = VLAK_OK;
  vlak_device_error_poll(&code);
  TORCH_CHECK(code == VLAK_OK, op, ": an earlier vlak kernel gave up a bounded device wait (",
              vlak_status_string(code), "); the output of that call is incomplete");
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return VLAK_F32;
    case at::kHalf: return VLAK_F16;
    case at::kBFloat16: return VLAK_BF16;
    case at::kDouble: return VLAK_F64;
    default: return -1;
  }
}

// A new contiguous tensor on the device of `like`. For implementations under the
// CUDA key only: it does not go through the dispatcher again, which cost a
// training call, with its seven or eight tensors, 3 of 80 us.
inline at::Tensor new_empty(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// The differentiable ops have no forward-mode derivative. Their autograd kernels
// go below autograd for inputs that need no gradient, where a tangent would be
// dropped in silence; so one on any input (they may be undefined) is refused.
inline void refuse_tangents(std::initializer_list<at::Tensor> inputs, const char* op) {
  for (const at::Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op,
                                " has no forward-mode derivative");
}

// Checks and arguments of the GQA attention ops (torch_ops.cpp).
vlak_attn_gqa_args gqa_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            double scale, int64_t prefix_len, int64_t dead_start,
                            int64_t dead_end, const char* op);

}  // namespace vlak_torch

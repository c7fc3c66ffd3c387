// polyrl_b200 — what the binding translation units share.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cstdint>
#include <string>
#include <vector>

namespace {

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "polyrl_b200 kernel '", what, "' failed with code ", rc);
}
#define CHECK_BF16(t) TORCH_CHECK((t).is_cuda() && (t).scalar_type() == at::kBFloat16, #t " must be a CUDA bf16 tensor")
#define CHECK_F32(t) TORCH_CHECK((t).is_cuda() && (t).scalar_type() == at::kFloat, #t " must be a CUDA fp32 tensor")
#define CHECK_LASTDIM(t) TORCH_CHECK((t).stride(-1) == 1, #t " must be contiguous in the last dim")

// scratch of a product whose last round of tiles is cut along the reduction (gemm2_sm100.cuh); nothing when it is not
inline at::Tensor split_scratch(int64_t floats, const at::Tensor& like) {
  return floats > 0 ? at::empty({floats}, like.options().dtype(at::kFloat)) : at::Tensor();
}
inline float* split_ptr(const at::Tensor& ws) { return ws.defined() ? ws.data_ptr<float>() : nullptr; }

// rows as the kernels read them: unit inner stride, pitch and base on 16 bytes (packed: and no gap between rows)
inline at::Tensor aligned_rows(const at::Tensor& t, bool packed = false) {
  const bool aligned = (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  if (t.dim() != 2 || (aligned && t.stride(1) == 1 && (packed ? t.stride(0) == t.size(1) : t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)))) return t;
  const at::Tensor c = t.contiguous(), d = (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
  return d.size(0) == 1 ? d.as_strided(d.sizes(), {d.size(1), 1}) : d;      // a single row counts as contiguous whatever its pitch is
}

}  // namespace

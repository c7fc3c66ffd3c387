// polyrl_b200 — bindings of what a request brings to a batch: its rules on the logits (logit_rules.cu) and its adapter (adapters.cu).
// Included by bindings_serve.cpp.
#pragma once
#include "adapters.hpp"
#include "bindings_common.hpp"
#include "logit_rules.hpp"

extern "C" {
int prl_adjust_logits(const prl::RuleParams*, int, cudaStream_t);
int prl_adapter_plan(const int32_t*, int, int, int, int, int32_t*, void*, int32_t*, cudaStream_t);
int prl_adapter_delta(const prl::DeltaParams*, int, int, int, cudaStream_t);
}

namespace {

using OptTensor = c10::optional<at::Tensor>;

// a vector of one value a row, on the device of `like`; null where absent
template <class T>
const T* row_vec(const OptTensor& t, const at::Tensor& like, int64_t rows, const char* what) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_VALUE(t->device() == like.device() && t->scalar_type() == c10::CppTypeToScalarType<T>::value && t->dim() == 1 && t->size(0) == rows &&
              (t->stride(0) == 1 || rows <= 1), what, ": one contiguous value a row on the device of the rows");
  return t->data_ptr<T>();
}
// rows of values with unit inner stride
template <class T>
const T* row_mat(const OptTensor& t, const at::Tensor& like, int64_t rows, int64_t* ld, const char* what) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_VALUE(t->device() == like.device() && t->scalar_type() == c10::CppTypeToScalarType<T>::value && t->dim() == 2 && (rows < 0 || t->size(0) == rows) &&
              (t->stride(1) == 1 || t->size(1) <= 1), what, ": rows of values with unit inner stride on the device of the rows");
  *ld = t->stride(0);
  return t->data_ptr<T>();
}

at::Tensor adjust_logits(const at::Tensor& z, OptTensor out, const OptTensor& tokens, const OptTensor& lens, const OptTensor& prompt_lens, const OptTensor& rep,
                         const OptTensor& pres, const OptTensor& freq, const OptTensor& bias_ids, const OptTensor& bias_values, const OptTensor& stop_ids,
                         const OptTensor& min_lens, const OptTensor& masks, const OptTensor& mask_rows) {
  TORCH_CHECK_VALUE(z.is_cuda() && z.dim() == 2 && (z.stride(1) == 1 || z.size(1) <= 1) && (z.scalar_type() == at::kFloat || z.scalar_type() == at::kBFloat16),
              "adjust_logits: bf16 or fp32 logits [rows, vocabulary] with unit inner stride");
  c10::cuda::CUDAGuard g(z.device());
  const int64_t rows = z.size(0), V = z.size(1);
  TORCH_CHECK_VALUE(rows <= 0x7fffffff && V < (1 << 30), "adjust_logits: too many rows or tokens");
  at::Tensor o = out.has_value() ? *out : at::empty({rows, V}, z.options());
  TORCH_CHECK_VALUE(o.device() == z.device() && o.scalar_type() == z.scalar_type() && o.sizes() == z.sizes() && (o.stride(1) == 1 || V <= 1) &&
              (o.stride(0) >= V || rows <= 1), "adjust_logits: out must be like the logits, its rows apart");
  if (rows == 0 || V == 0) return o;
  const int64_t e = z.element_size();
  const char *z0 = static_cast<const char*>(z.data_ptr()), *o0 = static_cast<const char*>(o.data_ptr());
  const int64_t zn = ((rows - 1) * z.stride(0) + V) * e, on = ((rows - 1) * o.stride(0) + V) * e;
  TORCH_CHECK_VALUE((z0 == o0 && (z.stride(0) == o.stride(0) || rows == 1)) || z0 + zn <= o0 || o0 + on <= z0,
              "adjust_logits: out must be the logits themselves or memory apart from them");
  prl::RuleParams p{};
  p.z = z0; p.out = const_cast<char*>(o0); p.ldz = z.stride(0); p.ldo = o.stride(0); p.rows = rows; p.V = V;
  p.tokens = row_mat<int32_t>(tokens, z, rows, &p.ld_tokens, "adjust_logits: tokens");
  p.max_tokens = tokens.has_value() ? tokens->size(1) : 0;
  TORCH_CHECK_VALUE(p.max_tokens < (1 << prl::kRuleCountBits), "adjust_logits: a history of less than 2^20 tokens");
  p.lens = row_vec<int32_t>(lens, z, rows, "adjust_logits: lens");
  p.prompt_lens = row_vec<int32_t>(prompt_lens, z, rows, "adjust_logits: prompt_lens");
  p.rep = row_vec<float>(rep, z, rows, "adjust_logits: repetition");
  p.pres = row_vec<float>(pres, z, rows, "adjust_logits: presence");
  p.freq = row_vec<float>(freq, z, rows, "adjust_logits: frequency");
  p.bias_ids = row_mat<int32_t>(bias_ids, z, rows, &p.ld_bias, "adjust_logits: bias_ids");
  int64_t ld = 0;
  p.bias_values = row_mat<float>(bias_values, z, rows, &ld, "adjust_logits: bias_values");
  TORCH_CHECK_VALUE(bias_ids.has_value() == bias_values.has_value() && (!bias_ids.has_value() || (bias_ids->size(1) == bias_values->size(1) && (ld == p.ld_bias || rows == 1))),
              "adjust_logits: bias_ids and bias_values belong together, laid out alike");
  TORCH_CHECK_VALUE(tokens.has_value() || !(p.rep || p.pres || p.freq), "adjust_logits: penalties need the rows' tokens");
  p.num_bias = p.bias_ids ? bias_ids->size(1) : 0;
  TORCH_CHECK_VALUE(p.num_bias <= prl::kRuleMaxBias, "adjust_logits: at most ", prl::kRuleMaxBias, " biased tokens a row");
  if (p.num_bias == 0) p.bias_ids = nullptr;
  p.stop_ids = row_mat<int32_t>(stop_ids, z, rows, &p.ld_stop, "adjust_logits: stop_ids");
  p.num_stop = p.stop_ids ? stop_ids->size(1) : 0;
  p.min_lens = row_vec<int32_t>(min_lens, z, rows, "adjust_logits: min_lens");
  TORCH_CHECK_VALUE(stop_ids.has_value() == min_lens.has_value() && (!stop_ids.has_value() || lens.has_value()), "adjust_logits: stop_ids, min_lens and lens belong together");
  TORCH_CHECK_VALUE(masks.has_value() || !mask_rows.has_value(), "adjust_logits: mask_rows without masks");
  p.masks = row_mat<int32_t>(masks, z, -1, &p.ld_masks, "adjust_logits: masks");
  p.mask_rows = row_vec<int32_t>(mask_rows, z, rows, "adjust_logits: mask_rows");
  if (p.masks) {
    p.num_masks = masks->size(0);
    TORCH_CHECK_VALUE(masks->size(1) >= (V + 31) / 32 && (p.mask_rows || p.num_masks == rows), "adjust_logits: masks [masks, ceil(vocabulary / 32)], one a row or mask_rows");
  }
  if (out.has_value() && !o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  check(prl_adjust_logits(&p, z.scalar_type() == at::kFloat, cur_stream()), "adjust_logits");
  return o;
}

// ids [T] int32 -> one int32 buffer: tiles in use (4 words), tiles [max_tiles][4], rows sorted by adapter [T]
at::Tensor adapter_plan(const at::Tensor& ids, int64_t adapters, int64_t tile_rows, int64_t max_tiles) {
  TORCH_CHECK_VALUE(ids.is_cuda() && ids.scalar_type() == at::kInt && ids.dim() == 1 && (ids.stride(0) == 1 || ids.size(0) <= 1), "adapter_plan: int32 vector of adapter ids");
  const int64_t T = ids.size(0), groups = std::min(adapters + 1, T);
  TORCH_CHECK_VALUE(adapters >= 1 && adapters <= prl::kPlanMaxAdapters, "adapter_plan: 1 to ", prl::kPlanMaxAdapters, " adapters");
  TORCH_CHECK_VALUE(tile_rows >= 1 && T <= 0x7fffffff / 4 && max_tiles >= (T ? (T - groups) / tile_rows + groups : 0), "adapter_plan: sizes");
  c10::cuda::CUDAGuard g(ids.device());
  at::Tensor buf = at::empty({4 + 4 * max_tiles + T}, ids.options());
  if (T == 0) return buf.zero_();
  int32_t* p = buf.data_ptr<int32_t>();
  check(prl_adapter_plan(ids.data_ptr<int32_t>(), T, adapters, tile_rows, max_tiles, p + 4 + 4 * max_tiles, p + 4, p, cur_stream()), "adapter_plan");
  return buf;
}

const void* delta_operand(const at::Tensor& t, const at::Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(t.device() == x.device() && t.scalar_type() == at::kBFloat16 && t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, what,
              ": bf16 on the rows' device, unit inner stride, 16-byte aligned");
  return t.data_ptr();
}

// what the adapters of the rows add to x W^T, with bias and residual, as bf16 [T, N] (adapters.cu)
at::Tensor adapter_delta(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& scales, const at::Tensor& plan, int64_t tile_rows,
                         int64_t max_tiles, const std::vector<int64_t>& widths, bool interleaved, const OptTensor& bias, const OptTensor& residual, const OptTensor& onto, int64_t ctas,
                         int64_t shares) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && a.dim() == 3 && b.dim() == 3, "adapter_delta: x [T, K], a [adapters, parts * rank, K], b [adapters, N, rank]");
  prl::DeltaParams p{};
  const int64_t T = x.size(0), K = x.size(1), L = a.size(0), N = b.size(1), rank = b.size(2), parts = widths.size();
  p.x = delta_operand(x, x, "adapter_delta: x"); p.a = delta_operand(a, x, "adapter_delta: a"); p.b = delta_operand(b, x, "adapter_delta: b");
  TORCH_CHECK_VALUE(a.is_contiguous() && b.is_contiguous() && b.size(0) == L && a.size(2) == K && a.size(1) == parts * rank, "adapter_delta: stacked adapters do not fit");
  TORCH_CHECK_VALUE(parts >= 1 && parts <= 3 && rank >= 16 && rank % 16 == 0 && parts * rank <= prl::kDeltaMaxLow && K > 0 && K % 32 == 0 && N > 0 && N % 32 == 0 &&
              K <= 0x7fffffff && N <= 0x7fffffff, "adapter_delta: sizes");
  int64_t end = 0;
  for (int64_t i = 0; i < parts; ++i) {
    TORCH_CHECK_VALUE(widths[i] > 0 && widths[i] % 32 == 0, "adapter_delta: parts of a multiple of 32 columns");
    p.ends[i] = end += widths[i];
  }
  TORCH_CHECK_VALUE(end == N && (!interleaved || (parts == 2 && widths[0] == widths[1] && N % 256 == 0)), "adapter_delta: parts do not make up the columns");
  TORCH_CHECK_VALUE(x.stride(0) % 8 == 0 || T <= 1, "adapter_delta: row pitch of a multiple of 8");
  TORCH_CHECK_VALUE(scales.device() == x.device() && scales.scalar_type() == at::kFloat && scales.is_contiguous() && scales.dim() == 1 && scales.size(0) == L,
              "adapter_delta: one fp32 scale an adapter");
  TORCH_CHECK_VALUE(plan.device() == x.device() && plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.numel() == 4 + 4 * max_tiles + T, "adapter_delta: plan of other rows");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, "adapter_delta: bias [N]");
    p.bias = delta_operand(*bias, x, "adapter_delta: bias");
  }
  if (residual.has_value()) {
    TORCH_CHECK_VALUE(residual->dim() == 2 && residual->size(0) == T && residual->size(1) == N && (residual->stride(0) % 8 == 0 || T <= 1), "adapter_delta: residual [T, N]");
    p.res = delta_operand(*residual, x, "adapter_delta: residual");
    p.ldr = residual->stride(0);
  }
  c10::cuda::CUDAGuard g(x.device());
  if (onto.has_value()) {
    TORCH_CHECK_VALUE(onto->dim() == 2 && onto->is_contiguous() && onto->size(0) == T && onto->size(1) == N, "adapter_delta: onto [T, N]");
    delta_operand(*onto, x, "adapter_delta: onto");
  }
  at::Tensor out = onto.has_value() ? *onto : at::empty({T, N}, x.options());
  if (T == 0) return out;
  p.onto = onto.has_value();
  const int32_t* pl = plan.data_ptr<int32_t>();
  p.scales = scales.data_ptr<float>(); p.out = out.data_ptr(); p.num_tiles = pl; p.tiles = reinterpret_cast<const prl::AdapterTile*>(pl + 4);
  p.order = pl + 4 + 4 * max_tiles; p.ldx = x.stride(0); p.ldo = N; p.K = K; p.N = N; p.rank = rank; p.parts = parts; p.max_tiles = max_tiles;
  p.interleaved = interleaved;
  check(prl_adapter_delta(&p, tile_rows, ctas, shares, cur_stream()), "adapter_delta");
  return out;
}

// x w^T (+ bias) by the library, as a decode step's plain products, and what the adapters add to it
at::Tensor adapter_linear(const at::Tensor& x_in, const at::Tensor& w, const at::Tensor& a, const at::Tensor& b, const at::Tensor& scales, const at::Tensor& plan,
                          int64_t adapters, int64_t tile_rows, int64_t max_tiles, const std::vector<int64_t>& widths, const OptTensor& bias, const OptTensor& residual) {
  TORCH_CHECK_VALUE(w.dim() == 2 && x_in.dim() == 2 && w.size(1) == x_in.size(1) && a.dim() == 3 && b.dim() == 3 && w.size(0) == b.size(1), "adapter_linear: the projection does not fit");
  TORCH_CHECK_VALUE(a.size(0) == adapters, "adapter_linear: a plan for ", adapters, " adapters, the stacks hold ", a.size(0));
  c10::cuda::CUDAGuard g(x_in.device());
  const at::AutoGradMode inference(false);
  const at::Tensor x = aligned_rows(x_in);
  return adapter_delta(x, a, b, scales, plan, tile_rows, max_tiles, widths, false, c10::nullopt, residual.has_value() ? OptTensor(aligned_rows(*residual)) : c10::nullopt,
                       at::linear(x, w, bias), 0, 0);
}

}  // namespace

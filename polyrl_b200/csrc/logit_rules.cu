// polyrl_b200 — a step's logits under the rules that each request brings: penalties for tokens it has used, biases, stop tokens that
// may not come yet, and a mask of allowed tokens.  For row b, token v, with c = times v is among the row's output tokens and "seen" =
// v is among its prompt or output tokens:
//
//   z1 = seen ? (z > 0 ? z / repetition : z * repetition) : z
//   z2 = z1 - frequency * c - (c > 0 ? presence : 0) + bias(v)
//   out = banned(v) ? -inf : z2            banned: not in the row's mask, or a stop token while the row is shorter than its least length
//
// All in fp32, rounded once to the logits' type; what no rule touches is copied bit for bit (in place: not touched at all).
//
// Split: a block takes `chunk` consecutive tokens of the vocabulary of one row.  Its table in shared memory has a 32-bit word per token of
// the chunk, addressed by the token itself, so nothing is hashed, sorted or kept between calls: the words are cleared, the row's biases and
// stop tokens marked, its whole history read (coalesced, out of L2 for all but a row's first block) and counted with shared-memory atomics,
// which are integers and therefore give the same words in any order.  Then the chunk is streamed once, 16 bytes a thread.
#include <type_traits>

#include "common.cuh"
#include "logit_rules.hpp"

namespace prl {

// word of the table: output count in the low 20 bits, "in the prompt", place in the bias list + 1
constexpr uint32_t kCountMask = (1u << kRuleCountBits) - 1, kPrompt = 1u << kRuleCountBits;
constexpr int kBiasShift = kRuleCountBits + 1;
constexpr uint32_t kBanned = (1u << (32 - kBiasShift)) - 1;
static_assert(kRuleMaxBias == kBanned - 1, "the last place means banned");

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }

struct RowRules {
  float rep, pres, freq;
  const float* bias;
  __device__ __forceinline__ float operator()(float z, uint32_t word) const {
    if (word & (kCountMask | kPrompt)) z = z > 0.f ? z / rep : z * rep;
    const uint32_t c = word & kCountMask, at = word >> kBiasShift;
    if (c) z = z - freq * static_cast<float>(c) - pres;
    if (at) z = at == kBanned ? -INFINITY : z + bias[at - 1];
    return z;
  }
};

template <class T, int VEC, bool INPLACE>
__global__ void __launch_bounds__(kRuleThreads) rules_kernel(RuleParams p, int chunks) {
  extern __shared__ uint32_t table[];
  const int row = blockIdx.x / chunks, base = (blockIdx.x % chunks) * p.chunk, size = min(p.chunk, p.V - base);
  grid_behind();
  const RowRules rr{p.rep ? p.rep[row] : 1.f, p.pres ? p.pres[row] : 0.f, p.freq ? p.freq[row] : 0.f,
                    p.bias_ids ? p.bias_values + row * p.ld_bias : nullptr};
  const int len = p.lens ? p.lens[row] : p.max_tokens;
  const bool counts = p.tokens && (rr.rep != 1.f || rr.pres != 0.f || rr.freq != 0.f);
  const bool early = p.stop_ids && len < p.min_lens[row];
  const int mask_row = p.masks ? p.mask_rows ? p.mask_rows[row] : row : -1;
  const uint32_t* mask = mask_row >= 0 && mask_row < p.num_masks ? reinterpret_cast<const uint32_t*>(p.masks) + mask_row * p.ld_masks + (base >> 5) : nullptr;
  const bool words = counts || early || p.bias_ids != nullptr;
  if (INPLACE && !words && !mask) return;

  if (words) {
    for (int i = threadIdx.x; i < p.chunk / 4; i += kRuleThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (p.bias_ids)                                    // of entries with the same token the last one counts
      for (int j = threadIdx.x; j < p.num_bias; j += kRuleThreads) {
        const uint32_t at = static_cast<uint32_t>(p.bias_ids[row * p.ld_bias + j] - base);
        if (at < static_cast<uint32_t>(size)) atomicMax(&table[at], static_cast<uint32_t>(j + 1) << kBiasShift);
      }
    if (early)
      for (int j = threadIdx.x; j < p.num_stop; j += kRuleThreads) {
        const uint32_t at = static_cast<uint32_t>(p.stop_ids[row * p.ld_stop + j] - base);
        if (at < static_cast<uint32_t>(size)) atomicMax(&table[at], kBanned << kBiasShift);
      }
    __syncthreads();                                   // marks first: counts are added below them
    if (counts) {
      const int n = min(max(len, 0), p.max_tokens), prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
      const int32_t* tok = p.tokens + row * p.ld_tokens;
      int i = threadIdx.x;
      for (; i + 3 * kRuleThreads < n; i += 4 * kRuleThreads) {
        uint32_t at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) at[u] = static_cast<uint32_t>(tok[i + u * kRuleThreads] - base);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (at[u] < static_cast<uint32_t>(size)) {
            if (i + u * kRuleThreads < prompt) atomicOr(&table[at[u]], kPrompt);
            else atomicAdd(&table[at[u]], 1u);
          }
      }
      for (; i < n; i += kRuleThreads) {
        const uint32_t at = static_cast<uint32_t>(tok[i] - base);
        if (at >= static_cast<uint32_t>(size)) continue;
        if (i < prompt) atomicOr(&table[at], kPrompt);
        else atomicAdd(&table[at], 1u);
      }
    }
    __syncthreads();
  }

  const T* z = static_cast<const T*>(p.z) + row * p.ldz + base;
  T* out = static_cast<T*>(p.out) + row * p.ldo + base;
  if constexpr (VEC > 1) {
    using Raw = int4;
    static_assert(sizeof(T) * VEC == sizeof(Raw));
#pragma unroll 4
    for (int i = threadIdx.x; i < size / VEC; i += kRuleThreads) {
      const int v = i * VEC;
      const uint32_t bits = mask ? mask[v >> 5] >> (v & 31) : ~0u;
      uint32_t w[VEC], any = 0;
#pragma unroll
      for (int q = 0; q < VEC; q += 4) {
        const uint4 t = words ? *reinterpret_cast<const uint4*>(table + v + q) : make_uint4(0, 0, 0, 0);
        w[q] = t.x; w[q + 1] = t.y; w[q + 2] = t.z; w[q + 3] = t.w;
        any |= t.x | t.y | t.z | t.w;
      }
      const bool all = (bits & ((1u << VEC) - 1)) == (1u << VEC) - 1;
      if (INPLACE && all && !any) continue;
      union { Raw raw; T e[VEC]; } x;
      x.raw = INPLACE ? ld_v4(z + v) : ld_nc_v4(z + v);
      if (any || !all) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          if (w[q]) from_f32(rr(to_f32(x.e[q]), w[q]), x.e[q]);
          if (!((bits >> q) & 1)) from_f32(-INFINITY, x.e[q]);
        }
      }
      st_v4(out + v, x.raw);
    }
  }
  // what is left of the row, or all of it where rows do not start on 16 bytes
#pragma unroll 4
  for (int v = (VEC > 1 ? size / VEC * VEC : 0) + threadIdx.x; v < size; v += kRuleThreads) {
    const uint32_t word = words ? table[v] : 0;
    const bool ok = !mask || ((mask[v >> 5] >> (v & 31)) & 1);
    if (INPLACE && ok && !word) continue;
    T e = z[v];
    if (word) from_f32(rr(to_f32(e), word), e);
    if (!ok) from_f32(-INFINITY, e);
    out[v] = e;
  }
}

template <class T>
static int run_rules(const RuleParams& p, cudaStream_t stream) {
  const int chunks = (p.V + p.chunk - 1) / p.chunk;
  const int64_t blocks = static_cast<int64_t>(p.rows) * chunks;
  if (blocks > 0x7fffffff) return -3;
  constexpr int VEC = 16 / sizeof(T);
  const bool inplace = p.z == p.out;
  const bool wide = ((reinterpret_cast<uintptr_t>(p.z) | reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 && p.ldz % VEC == 0 && p.ldo % VEC == 0;
  auto kern = wide ? inplace ? rules_kernel<T, VEC, true> : rules_kernel<T, VEC, false> : inplace ? rules_kernel<T, 1, true> : rules_kernel<T, 1, false>;
  const size_t smem = p.chunk * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRuleMaxChunk * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  PRL_CUDA_CHECK(launch_behind(kern, static_cast<unsigned>(blocks), kRuleThreads, smem, stream, p, chunks));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

}  // namespace prl

// p.chunk 0: chosen here.  A block reads the row's whole history, so long histories want wide chunks; few rows want many blocks.
extern "C" int prl_adjust_logits(const prl::RuleParams* q, int fp32, cudaStream_t stream) {
  prl::RuleParams p = *q;
  if (p.rows <= 0 || p.V <= 0) return 0;
  if (p.num_bias > prl::kRuleMaxBias || p.max_tokens >= (1 << prl::kRuleCountBits)) return -1;
  if (p.chunk <= 0) {
    p.chunk = 16384;
    while (p.chunk > 2048 && static_cast<int64_t>(p.rows) * ((p.V + p.chunk - 1) / p.chunk) < 2 * 148) p.chunk >>= 1;
  }
  if (p.chunk % 128 || p.chunk > prl::kRuleMaxChunk) return -2;
  return fp32 ? prl::run_rules<float>(p, stream) : prl::run_rules<__nv_bfloat16>(p, stream);
}

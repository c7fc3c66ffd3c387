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
// Split: a block takes a part of one row's vocabulary and has a word in shared memory for each of its tokens.  Half of its warps clear the words, read the
// row's whole history (out of L2 for all but the row's first block) and count the tokens of the part with shared-memory atomics, while the other half
// copy the part under the row's mask, 16 bytes a thread (and count with the rest afterwards, where histories are long).  Then all of them look through the words for touched tokens, pack them 32 to a warp, compute
// those logits from the input and write them over the copy.  In place only masked and touched tokens are written.  Nothing is hashed, sorted or kept
// between calls; counters are integers, so results do not depend on the order of the threads.
// Histories are sparse, so what bounds it is instructions before it is bytes.  A hashed table asked again for every token of the history ran its few hits
// a warp one lane at a time (256 rows of 128256 bf16 logits with histories of up to 1100: 52 us); a list that the counting threads append to saves the
// search but waits for every atomic's answer (24 rows with histories of 30011: 42 us).
// Now 39 us for the former (34 in place; a plain copy of these logits takes 22), 20 for the latter, 9 for 37 rows of 50257 fp32 logits, 4.5 for one row of
// 151936.
#include "common.cuh"
#include "logit_rules.hpp"

namespace prl {

// Word of a token: output count, then "in the prompt", "in the bias list", "may not come yet".  Adding to the count and setting bits commute.
// 16 bits a token where the count fits 13, two tokens to a 32-bit word of memory: half the memory, so more blocks on an SM, and half the words
// to clear and to look through.
template <int BITS>
struct RuleWord {
  static constexpr int kCountBits = BITS == 16 ? kRuleShortBits : kRuleCountBits;
  static constexpr uint32_t kCount = (1u << kCountBits) - 1, kPrompt = 1u << kCountBits, kBias = kPrompt << 1, kBanned = kPrompt << 2;
  static_assert(kCountBits + 3 <= BITS);
  static __device__ __forceinline__ void add(uint32_t* words, uint32_t at, uint32_t v) {
    if (BITS == 16) atomicAdd(words + (at >> 1), v << (16 * (at & 1)));
    else atomicAdd(words + at, v);
  }
  static __device__ __forceinline__ void mark(uint32_t* words, uint32_t at, uint32_t bit) {
    if (BITS == 16) atomicOr(words + (at >> 1), bit << (16 * (at & 1)));
    else atomicOr(words + at, bit);
  }
  // which of the words in 16 bytes are not clear, a bit each
  static __device__ __forceinline__ uint32_t set(const uint4& q) {
    if (BITS == 32) return (q.x != 0) | (q.y != 0) << 1 | (q.z != 0) << 2 | (q.w != 0) << 3;
    const uint32_t a = __vsetne2(q.x, 0), b = __vsetne2(q.y, 0), c = __vsetne2(q.z, 0), d = __vsetne2(q.w, 0);
    return ((a | a >> 15) & 3) | ((b | b >> 15) & 3) << 2 | ((c | c >> 15) & 3) << 4 | ((d | d >> 15) & 3) << 6;
  }
  static __device__ __forceinline__ uint32_t get(const uint32_t* words, int at) {
    return BITS == 16 ? reinterpret_cast<const uint16_t*>(words)[at] : words[at];
  }
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }

__device__ __forceinline__ const uint32_t* mask_of(const RuleParams& p, int64_t row) {
  if (!p.masks) return nullptr;
  const int64_t m = p.mask_rows ? p.mask_rows[row] : row;
  return m >= 0 && m < p.num_masks ? reinterpret_cast<const uint32_t*>(p.masks) + m * p.ld_masks : nullptr;
}

// Tokens [0, size) of a part from z to out under its mask, 16 bytes at a time between the first and the last 16-byte boundary inside (rows start
// anywhere; where z and out start differently, token by token).  In place nothing but masked tokens is touched.
template <class T, bool INPLACE>
__device__ __forceinline__ void copy_part(const T* z, T* out, int size, const uint32_t* mask, int tid, int threads) {
  constexpr int VEC = 16 / sizeof(T), kVecs = 4;
  constexpr uint32_t kAll = (1u << VEC) - 1;
  if (INPLACE && !mask) return;
  auto one = [&](int v) {
    const bool ok = !mask || ((__ldg(mask + (v >> 5)) >> (v & 31)) & 1);
    if (INPLACE && ok) return;
    T e = z[v];
    if (!ok) from_f32(-INFINITY, e);
    out[v] = e;
  };
  const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int head = alike ? min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) % 16 / sizeof(T)), size) : size;
  const int tail = head + (size - head) / VEC * VEC;
#pragma unroll 8
  for (int v = tid; v < head; v += threads) one(v);
  for (int v = tail + tid; v < size; v += threads) one(v);
  for (int v0 = head + tid * VEC; v0 < tail; v0 += kVecs * threads * VEC) {
    int4 x[kVecs];
    uint32_t bits[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int v = v0 + j * threads * VEC;
      if (v >= tail) continue;
      if constexpr (!INPLACE) x[j] = ld_nc_v4(z + v);
      bits[j] = mask ? __funnelshift_r(__ldg(mask + (v >> 5)), __ldg(mask + ((v + VEC - 1) >> 5)), v & 31) & kAll : kAll;
    }
    if constexpr (INPLACE) {                           // what is neither kept nor banned as a whole
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const int v = v0 + j * threads * VEC;
        if (v < tail && bits[j] != kAll && bits[j] != 0) x[j] = ld_v4(z + v);
      }
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int v = v0 + j * threads * VEC;
      if (v >= tail || (INPLACE && bits[j] == kAll)) continue;
      if (bits[j] != kAll) {
        int* w = reinterpret_cast<int*>(&x[j]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (VEC == 4) {
            if (!((bits[j] >> q) & 1)) w[q] = static_cast<int>(0xff800000u);
          } else {                                     // a pair of bf16: all ones over what stays, -inf over what does not
            const int lo = static_cast<int>(bits[j] << (31 - 2 * q)) >> 31, hi = static_cast<int>(bits[j] << (30 - 2 * q)) >> 31;
            const int keep = __byte_perm(lo, hi, 0x5410);
            w[q] = (w[q] & keep) | (static_cast<int>(0xff80ff80u) & ~keep);
          }
        }
      }
      st_v4(out + v, x[j]);
    }
  }
}

template <class T, bool INPLACE, int BITS>
__global__ void __launch_bounds__(kRuleThreads, BITS == 32 ? 2 : 3) rules_kernel(RuleParams p, int parts, int part) {
  constexpr int kAhead = 6, kVecsAhead = 4;            // tokens that a thread has in flight; 16-byte loads of long histories
  constexpr int kCounting = kRuleThreads / 2;
  // Histories so long that counting takes most of the time: the copying warps join once they are done, 16 bytes of tokens a load, with the registers of two
  // blocks an SM instead of three.  24 rows of 151936 with 30011 tokens 23 -> 20 us, 8 rows with 32000 15 (4-byte loads) -> 13, one row 12 -> 10.
  constexpr bool kLong = BITS == 32;
  constexpr int kStride = kLong ? kRuleThreads : kCounting;
  using Word = RuleWord<BITS>;
  constexpr int kEach = 128 / BITS, kStep = 32 * kEach;          // tokens a lane and a warp look at together
  extern __shared__ __align__(16) uint32_t words[];    // [part] words of BITS bits, the row's bias list
  __shared__ uint16_t packed[kRuleThreads / 32][32 + kStep];     // a warp packs touched tokens until it has 32
  int32_t* bias_ids = reinterpret_cast<int32_t*>(words + part * BITS / 32);
  const int64_t row = blockIdx.x / parts;
  const int tid = threadIdx.x, base = static_cast<int>(blockIdx.x % parts) * part, size = min(part, p.V - base);
  grid_behind();
  const T* z = static_cast<const T*>(p.z) + row * p.ldz + base;
  T* out = static_cast<T*>(p.out) + row * p.ldo + base;
  if (!INPLACE && tid == 0) {                          // on its way into L2 while the history is counted
    const uintptr_t from = (reinterpret_cast<uintptr_t>(z) + 15) & ~uintptr_t(15), to = reinterpret_cast<uintptr_t>(z + size) & ~uintptr_t(15);
    if (to > from) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(static_cast<uint32_t>(to - from)) : "memory");
  }
  // everything that has an address now is asked for now: a block is a few loads deep and little else
  const int32_t* tok = p.tokens + row * p.ld_tokens;
  int32_t token[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) token[u] = !kLong && tid < kCounting && tid + u * kStride < p.max_tokens ? __ldg(tok + tid + u * kStride) : -1;
  const int len = p.lens ? p.lens[row] : p.max_tokens, prompt = p.prompt_lens ? p.prompt_lens[row] : 0, least = p.num_stop > 0 ? p.min_lens[row] : 0;
  const float rep = p.rep ? p.rep[row] : 1.f, pres = p.pres ? p.pres[row] : 0.f, freq = p.freq ? p.freq[row] : 0.f;
  const uint32_t* mask = mask_of(p, row);
  if (mask) mask += base >> 5;
  const bool early = p.num_stop > 0 && len < least;
  const int n = rep != 1.f || pres != 0.f || freq != 0.f ? min(len, p.max_tokens) : 0;
  if (n <= 0 && !early && p.num_bias == 0) {
    copy_part<T, INPLACE>(z, out, size, mask, tid, kRuleThreads);
    return;
  }
  auto note = [&](int i, int32_t tkn) {               // the history's token i
    const uint32_t at = static_cast<uint32_t>(tkn) - static_cast<uint32_t>(base);
    if (at < static_cast<uint32_t>(size)) {
      if (i < prompt) Word::mark(words, at, Word::kPrompt);
      else Word::add(words, at, 1u);
    }
  };
  // this thread's share of the history; the first of its tokens are there already (long histories: 16 bytes at a time, nothing is there)
  auto count_tokens = [&]() {
    if constexpr (kLong) {
      const int head = min(static_cast<int>(-(reinterpret_cast<uintptr_t>(tok) >> 2) & 3), n), vecs = (n - head) / 4, tail = head + 4 * vecs;
      if (tid < head) note(tid, __ldg(tok + tid));
      if (tid < n - tail) note(tail + tid, __ldg(tok + tail + tid));
      for (int v0 = tid; v0 < vecs; v0 += kVecsAhead * kStride) {
        int4 q[kVecsAhead];
#pragma unroll
        for (int u = 0; u < kVecsAhead; ++u) q[u] = v0 + u * kStride < vecs ? __ldg(reinterpret_cast<const int4*>(tok + head) + v0 + u * kStride) : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int u = 0; u < kVecsAhead; ++u) {
          if (v0 + u * kStride >= vecs) continue;
          const int i = head + 4 * (v0 + u * kStride);
          note(i, q[u].x); note(i + 1, q[u].y); note(i + 2, q[u].z); note(i + 3, q[u].w);
        }
      }
    } else {
      for (int i0 = tid; i0 < n; i0 += kAhead * kStride) {
        if (i0 != tid) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u) token[u] = i0 + u * kStride < n ? __ldg(tok + i0 + u * kStride) : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i0 + u * kStride < n) note(i0 + u * kStride, token[u]);
      }
    }
  };
  if (tid < kCounting) {                               // half of the warps count while the other half copies: both are latencies more than work
    for (int j = tid; j < p.num_bias; j += kCounting) bias_ids[j] = p.bias_ids[row * p.ld_bias + j];
    for (int i = tid; i < part * BITS / 128; i += kCounting) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("bar.sync 1, %0;" ::"n"(kCounting) : "memory");
    if (kLong) asm volatile("bar.arrive 2, %0;" ::"n"(kRuleThreads) : "memory");
    count_tokens();
    for (int j = tid; j < p.num_bias; j += kCounting) {
      const uint32_t at = static_cast<uint32_t>(bias_ids[j]) - static_cast<uint32_t>(base);
      if (at < static_cast<uint32_t>(size)) Word::mark(words, at, Word::kBias);
    }
    if (early)
      for (int j = tid; j < p.num_stop; j += kCounting) {
        const uint32_t at = static_cast<uint32_t>(p.stop_ids[row * p.ld_stop + j]) - static_cast<uint32_t>(base);
        if (at < static_cast<uint32_t>(size)) Word::mark(words, at, Word::kBanned);
      }
  } else {
    copy_part<T, INPLACE>(z, out, size, mask, tid - kCounting, kRuleThreads - kCounting);
    if (kLong) {
      asm volatile("bar.sync 2, %0;" ::"n"(kRuleThreads) : "memory");        // the words are clear
      count_tokens();
    }
  }
  __syncthreads();                                     // the words are complete, the copy is written

  const int lane = tid & 31, warp = tid >> 5;
  uint16_t* mine = packed[warp];
  auto put = [&](int at) {                             // the token `at` of the part, a touched one
    const uint32_t w = Word::get(words, at), bits = mask ? __ldg(mask + (at >> 5)) : ~0u;
    float v = to_f32(z[at]);
    if (w & (Word::kCount | Word::kPrompt)) v = v > 0.f ? v / rep : v * rep;
    const uint32_t c = w & Word::kCount;
    if (c) v = v - freq * static_cast<float>(c) - pres;
    if (w & Word::kBias) {                             // of entries with the same token the last one counts
      int j = p.num_bias - 1;
      while (bias_ids[j] != base + at) --j;
      v += p.bias_values[row * p.ld_bias + j];
    }
    T o;
    from_f32((w & Word::kBanned) || !((bits >> (at & 31)) & 1) ? -INFINITY : v, o);
    out[at] = o;
  };
  int count = 0;                                       // tokens packed and not yet written, the same for the whole warp
  for (int i0 = warp * kStep; i0 < size; i0 += kRuleThreads * kEach) {            // (clear behind `size`)
    uint32_t set = Word::set(*reinterpret_cast<const uint4*>(words + (i0 + lane * kEach) * BITS / 32));
    if (!__any_sync(0xffffffffu, set)) continue;
    int upto = __popc(set);
    const int own = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    for (int to = count + upto - own; set; set &= set - 1) mine[to++] = static_cast<uint16_t>(i0 + lane * kEach + __ffs(set) - 1);
    count += __shfl_sync(0xffffffffu, upto, 31);
    __syncwarp();
    if (count < 32) continue;
    int from = 0;
    for (; count - from >= 32; from += 32) put(mine[from + lane]);
    const int rest = count - from;
    const uint16_t keep = lane < rest ? mine[from + lane] : 0;
    __syncwarp();
    if (lane < rest) mine[lane] = keep;
    __syncwarp();
    count = rest;
  }
  if (lane < count) put(mine[lane]);
}

template <class T, int BITS>
static int run_rules(const RuleParams& p, cudaStream_t stream) {
  // parts as wide as leave some blocks for every SM: each of them reads the row's history (a long one is worth a block less)
  int part = kRulePart;
  while (part > 2048 && static_cast<int64_t>(p.rows) * ((p.V + part - 1) / part) < (BITS == 32 ? 222 : 296)) part /= 2;
  const int parts = (p.V + part - 1) / part;
  const int64_t blocks = static_cast<int64_t>(p.rows) * parts;
  if (blocks > 0x7fffffff) return -3;
  auto kern = p.z == p.out ? rules_kernel<T, true, BITS> : rules_kernel<T, false, BITS>;
  const size_t smem = part * BITS / 8 + 4 * static_cast<size_t>(p.num_bias);
  PRL_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRulePart * BITS / 8 + 4 * kRuleMaxBias));
  PRL_CUDA_CHECK(launch_behind(kern, static_cast<unsigned>(blocks), kRuleThreads, smem, stream, p, parts, part));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

}  // namespace prl

extern "C" int prl_adjust_logits(const prl::RuleParams* q, int fp32, cudaStream_t stream) {
  prl::RuleParams p = *q;
  if (p.rows <= 0 || p.V <= 0) return 0;
  if (p.num_bias > prl::kRuleMaxBias || p.max_tokens >= (1 << prl::kRuleCountBits)) return -1;
  if (!(p.rep || p.pres || p.freq)) p.max_tokens = 0;            // nothing counts the tokens
  if (p.z == p.out && !p.masks && p.max_tokens + p.num_bias + p.num_stop == 0) return 0;
  if (p.max_tokens < (1 << prl::kRuleShortBits)) return fp32 ? prl::run_rules<float, 16>(p, stream) : prl::run_rules<__nv_bfloat16, 16>(p, stream);
  return fp32 ? prl::run_rules<float, 32>(p, stream) : prl::run_rules<__nv_bfloat16, 32>(p, stream);
}

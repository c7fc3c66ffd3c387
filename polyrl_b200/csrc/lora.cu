// polyrl_b200 — the thin products of a low-rank adapter that is trained beside a frozen projection y = x W^T:
//
//   t  = s x A^T     [T, R]      forward               dt = s dy B      [T, R]      backward, towards x and A
//   dA = dt^T x      [R, K]                            dB = dy^T t      [N, R]
//
// R is a few dozen (all parts of a fused projection side by side, B block-diagonal), the other two sides are thousands, so each product reads
// its one large operand (x or dy) once and is bound by that.  y += t B^T and dx += dt A are not here: t and dt are further k-blocks of the
// large products (gemm2_sm100.cuh, Gemm2Tail), so what the adapter adds is summed in fp32 with the rest, rounds nothing of its own and moves
// no [T, N] or [T, K] array.  There t and dt are bf16, as every operand of a product is (2^-8 at most of what the adapter adds).  The gradients dA and
// dB are all adapter, so for them t and dt come in two bf16 halves, the rounded value and what rounding left (2^-16): twice the columns of a product
// that is bound by its other operand.
//
// thin   D[m, r] = scale * sum_k A(m, k) B(r, k), 128 rows of D a tile: tcgen05.mma 128 x R x 16, both operands by TMA (K-major, or MN-major
//        where the sum runs over tokens: dA is computed as x^T dt and stored transposed).  A cluster of S CTAs shares a tile's reduction,
//        because R is narrow and 128-row tiles alone are too few to draw HBM bandwidth: 32 tiles for dA of a 4096-wide layer.  The CTAs
//        leave their fp32 sums in shared memory and each adds up its share of the tile over distributed shared memory, in the order of the
//        ranks: results do not depend on timing.  Bound by the stream of its large operand where its rows are contiguous (8191 rows, 48 columns: t from
//        4096 columns 11 us, 5.9 TB/s; dt from 6144 19 us, 5.3 TB/s), by pieces of 128 bytes a row out of it where the sum runs over its rows (dA 20 us, 3.4
//        TB/s; dB 25 us, 4.0 TB/s).  So dA and dB are one launch, whose CTAs fill the chip together: one after the other and together 53 and 40 us there,
//        35 and 22 for 4099 x 6144 / 2048, 64 columns, 11.2 and 6.4 for 387 x 896 / 1152.  One cluster size serves both: where one product is alone enough for the
//        chip and the other is not, that costs what the overlap gives, or more (2500 x 3584 / 37888, 32 columns: 50 and 54).
// pack   A parts one below the other, B parts block-diagonal in the order of the projection's columns, ranks padded to 8 with zeros; a bias
//        becomes one more column of B against a column of ones in t, which the forward product then adds for nothing.
#include "gemm_sm100.cuh"
#include "lora.hpp"

namespace prl {

constexpr int kThinThreads = 192;                    // warp 0 TMA, warp 1 MMA, warps 2..5 accumulators -> shared memory; all of them store
constexpr int kThinStageA = kBlockM * 128;
constexpr int kThinSmemMax = 201 * 1024;

// columns of the accumulator: NR, or twice that with the second half behind a whole number of 64-column boxes
__host__ __device__ constexpr int thin_lo(int NR) { return (NR + 63) / 64 * 64; }
template <bool MN>
__host__ __device__ constexpr int thin_b_bytes(int NR, bool halves) { return MN ? (halves ? 2 : 1) * ((NR + 63) / 64) * 8192 : NR * 128; }

struct ThinParams {
  __nv_bfloat16* out;
  int64_t ldo;
  int M, R, K, NR, stages;
  float scale;
  int pad;                                           // columns after the last one: the first is 1, the rest 0 (row-major output)
  int lo_out;                                        // > 0: column of the outputs' second halves (row-major output)
  int lo_in;                                         // > 0: the same of B (MN-major)
  // rows of a batch with adapters of their own (row-major output): `each` columns belong to an adapter; a row keeps those of ids[row], times
  // scales[ids[row]], and zeros elsewhere
  const int32_t* ids;
  const float* scales;
  int each;
  int trans;                                         // out is [R, M]
  int tiles;                                         // of 128 rows
};

struct alignas(64) ThinMaps {
  CUtensorMap A, B;
};

// grid (S, blocks of NR columns, tiles), so that the blocks that read the same rows of A run together; A_MN / B_MN: the reduction runs over the operand's rows
// in memory.  Tiles from the first product's last one on are a second product's, with the same reduction length and columns.
template <bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThinThreads) thin_kernel(const __grid_constant__ ThinMaps maps1, const __grid_constant__ ThinMaps maps2, const ThinParams p1, const ThinParams p2) {
  const bool second = static_cast<int>(blockIdx.z) >= p1.tiles;
  const CUtensorMap *tmA = second ? &maps2.A : &maps1.A, *tmB = second ? &maps2.B : &maps1.B;
  const ThinParams p = second ? p2 : p1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full_bar[8], empty_bar[8], done_bar;
  __shared__ uint32_t tmem_slot;
  const int b_bytes = thin_b_bytes<B_MN>(p.NR, p.lo_in > 0), stage_bytes = kThinStageA + b_bytes;
  const int cols_acc = B_MN && p.lo_in > 0 ? thin_lo(p.NR) + p.NR : p.NR, ld_acc = cols_acc + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t S;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(S));
  const uint32_t rank = cluster_ctarank();
  const int m0 = (static_cast<int>(blockIdx.z) - (second ? p1.tiles : 0)) * kBlockM, r0 = blockIdx.y * p.NR;
  const int num_kb = (p.K + 63) / 64, kb0 = num_kb * rank / S, kb1 = num_kb * (rank + 1) / S;
  const uint32_t tmem_cols = cols_acc <= 32 ? 32 : cols_acc <= 64 ? 64 : cols_acc <= 128 ? 128 : 256;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(tmA);
    tma_prefetch_desc(tmB);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    mbar_init(&done_bar, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_behind();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait(&empty_bar[stage], phase ^ 1);
        mbar_expect_tx(&full_bar[stage], stage_bytes);
        uint8_t* sa = smem + stage * stage_bytes;
        uint8_t* sb = sa + kThinStageA;
        if constexpr (A_MN) {
          tma_load_2d(tmA, &full_bar[stage], sa, m0, kb * 64);
          tma_load_2d(tmA, &full_bar[stage], sa + 8192, m0 + 64, kb * 64);
        } else {
          tma_load_2d(tmA, &full_bar[stage], sa, kb * 64, m0);
        }
        if constexpr (B_MN) {
          for (int c = 0; c < p.NR; c += 64) {
            tma_load_2d(tmB, &full_bar[stage], sb + c / 64 * 8192, r0 + c, kb * 64);
            if (p.lo_in > 0) tma_load_2d(tmB, &full_bar[stage], sb + (thin_lo(p.NR) + c) / 64 * 8192, p.lo_in + r0 + c, kb * 64);
          }
        } else {
          tma_load_2d(tmB, &full_bar[stage], sb, kb * 64, r0);
        }
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_major(kBlockM, cols_acc, 1, 1, A_MN ? 1 : 0, B_MN ? 1 : 0);
      constexpr uint32_t a_step = A_MN ? (16 * 128) >> 4 : 32 >> 4, b_step = B_MN ? (16 * 128) >> 4 : 32 >> 4;
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait(&full_bar[stage], phase);
        tc_fence_after();
        const uint8_t* sa = smem + stage * stage_bytes;
        const uint8_t* sb = sa + kThinStageA;
        const uint64_t da = A_MN ? umma_desc_sw128_mnmajor(sa, 8192) : umma_desc_sw128_kmajor(sa);
        const uint64_t db = B_MN ? umma_desc_sw128_mnmajor(sb, 8192) : umma_desc_sw128_kmajor(sb);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16_ss(tmem, da + k * a_step, db + k * b_step, idesc, kb != kb0 || k != 0);
        umma_commit(&empty_bar[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      umma_commit(&done_bar);
    }
  } else {
    // every load has landed and every product has read its stage: the pipeline's memory takes the sums, rows of cols_acc + 4 floats (an odd number
    // of 16-byte units, so that 8 lanes' rows start in different banks)
    mbar_wait(&done_bar, 0);
    tc_fence_after();
    const int quad = warp & 3, row = quad * 32 + lane;
    float* dst = reinterpret_cast<float*>(smem) + row * ld_acc;
    for (int c = 0; c < cols_acc; c += 16) {
      uint32_t r[16];
      __syncwarp();
      tmem_ld_32x16(tmem + c + (static_cast<uint32_t>(quad * 32) << 16), r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(dst + c + 4 * j) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
    }
    tc_fence_before();
  }
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }

  // four columns of a row, summed over the ranks
  const uint32_t base = smem_u32(smem);
  auto ranks = [&](int row, int c) {
    const uint32_t off = base + (row * ld_acc + c) * 4;
    float4 q[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k)
      if (k < S)
        asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}"
                     : "=f"(q[k].x), "=f"(q[k].y), "=f"(q[k].z), "=f"(q[k].w)
                     : "r"(off), "r"(k)
                     : "memory");
    float4 v = q[0];
#pragma unroll
    for (uint32_t k = 1; k < 8; ++k)
      if (k < S) { v.x += q[k].x; v.y += q[k].y; v.z += q[k].z; v.w += q[k].w; }
    return v;
  };
  auto sum = [&](int row, int c) {
    float4 v = ranks(row, c);
    if (B_MN && p.lo_in > 0) {
      const float4 l = ranks(row, thin_lo(p.NR) + c);
      v.x += l.x; v.y += l.y; v.z += l.z; v.w += l.w;
    }
    return make_float4(v.x * p.scale, v.y * p.scale, v.z * p.scale, v.w * p.scale);
  };
  const int cols = min(p.NR, p.R - r0);
  if (!p.trans) {                                    // a share of the rows, four columns a thread
    const int rows0 = kBlockM * rank / S, rows1 = kBlockM * (rank + 1) / S;
    const int last = blockIdx.y + 1 == gridDim.y ? p.pad : 0, quads = (cols + last) / 4;
    for (int e = threadIdx.x; e < (rows1 - rows0) * quads; e += kThinThreads) {
      const int row = rows0 + e / quads, c = e % quads * 4;
      if (m0 + row >= p.M) break;
      float4 v = c < cols ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(c == cols ? 1.f : 0.f, 0.f, 0.f, 0.f);
      const int owner = p.ids && c < cols ? (r0 + c) / p.each : -1;
      if (c < cols && (!p.ids || p.ids[m0 + row] == owner)) {
        v = sum(row, c);
        if (p.ids) {
          const float s = p.scales[owner];
          v.x *= s; v.y *= s; v.z *= s; v.w *= s;
        }
      }
      const uint2 hi = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      __nv_bfloat16* o = p.out + static_cast<int64_t>(m0 + row) * p.ldo + r0 + c;
      *reinterpret_cast<uint2*>(o) = hi;
      if (p.lo_out > 0 && c < cols) {
        const float2 a = unpack_bf16(hi.x), b = unpack_bf16(hi.y);
        *reinterpret_cast<uint2*>(o + p.lo_out) = make_uint2(pack_bf16(v.x - a.x, v.y - a.y), pack_bf16(v.z - b.x, v.w - b.y));
      }
    }
  } else {                                           // a share of the columns, lanes along the tile's rows
    const int quads = cols / 4, q0 = quads * rank / S, q1 = quads * (rank + 1) / S;
    for (int e = threadIdx.x; e < (q1 - q0) * kBlockM; e += kThinThreads) {
      const int c = (q0 + e / kBlockM) * 4, row = e % kBlockM;
      if (m0 + row >= p.M) continue;
      const float4 v = sum(row, c);
      __nv_bfloat16* o = p.out + static_cast<int64_t>(r0 + c) * p.ldo + m0 + row;
      o[0] = __float2bfloat16(v.x);
      o[p.ldo] = __float2bfloat16(v.y);
      o[2 * p.ldo] = __float2bfloat16(v.z);
      o[3 * p.ldo] = __float2bfloat16(v.w);
    }
  }
  cluster_sync_all();                                // a peer may still read this CTA's sums
}

// a product's operands, A and B with their pitches, and what is done with it
struct ThinProduct {
  const void *A, *B;
  int64_t lda, ldb;
  ThinParams p;
};

template <bool A_MN, bool B_MN>
static int run_thin(ThinProduct* q, int count, int split, cudaStream_t stream) {
  const ThinParams& f = q[0].p;
  const bool halves = B_MN && f.lo_in > 0;
  // blocks of up to 128 columns, as even as 16 allows: their CTAs share an SM with another's, whose loads run while these sum up.  Up to 256 columns a
  // block, K-major: 5003 x 2048, 320 columns 29 -> 15 us; 2900 x 3584, 768 columns 41 -> 22; 8191 x 4096, 192 columns 27 -> 21.
  const int even = (f.R + 127) / 128, NR = ((f.R + even - 1) / even + 15) / 16 * 16;
  const int cols = halves ? thin_lo(NR) + NR : NR;
  const int stage = kThinStageA + thin_b_bytes<B_MN>(NR, halves), sums = kBlockM * (cols + 4) * 4;
  const int budget = cols <= 128 ? 100 * 1024 : 200 * 1024;           // two CTAs an SM where two fit
  const int stages = budget / stage > 8 ? 8 : budget / stage;
  const int smem = (stages * stage > sums ? stages * stage : sums) + 1024;
  ThinMaps maps[2];
  int tiles = 0;
  for (int i = 0; i < count; ++i) {
    ThinParams& p = q[i].p;
    if (p.R != f.R || p.K != f.K || (p.lo_in > 0) != (f.lo_in > 0)) return -6;
    p.NR = NR;
    p.stages = stages;
    p.tiles = (p.M + kBlockM - 1) / kBlockM;
    tiles += p.tiles;
    if (A_MN ? make_tmap_kmajor(&maps[i].A, q[i].A, p.K, p.M, q[i].lda * 2, 64, 2) : make_tmap_kmajor(&maps[i].A, q[i].A, p.M, p.K, q[i].lda * 2, kBlockM, 2)) return -2;
    if (B_MN ? make_tmap_kmajor(&maps[i].B, q[i].B, p.K, halves ? p.lo_in + p.R : p.R, q[i].ldb * 2, 64, 2) : make_tmap_kmajor(&maps[i].B, q[i].B, p.R, p.K, q[i].ldb * 2, NR, 2))
      return -3;
  }
  if (count == 1) maps[1] = maps[0];
  const int blocks = (f.R + NR - 1) / NR, num_kb = (f.K + 63) / 64;
  int S = split;
  if (S <= 0) {
    // CTAs for every SM; clusters of eight only where four leave half of the chip idle (they are harder to place, and sum over more CTAs).
    // 64 tiles of 64 k-blocks, 48 columns, 1, 2, 4 and 8 CTAs: 26.7, 16.2, 12.1, 19.8 us; 32 tiles of 128 (dA): 49, 30, 24, 36; 224 tiles of 94: 57, 65,
    // 78, 97; 16 tiles of 65, 64 columns: 27.8, 17.1, 11.4, 10.3.
    const int64_t whole = static_cast<int64_t>(tiles) * blocks;
    S = 1;
    while (S < 4 && whole * S < 148 && num_kb >= 2 * S) S *= 2;
    if (S == 4 && whole * S < 74 && num_kb >= 32) S = 8;
  }
  if (S > 8 || S > num_kb || (S & (S - 1)) || tiles > 65535 || blocks > 65535) return -4;
  auto kern = thin_kernel<A_MN, B_MN>;
  PRL_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kThinSmemMax));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(S, blocks, tiles);
  cfg.blockDim = dim3(kThinThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  PRL_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], q[0].p, q[count - 1].p));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

// ------------------------------------------------------------------------------------------------------------ pack
__global__ void __launch_bounds__(256) lora_pack_kernel(const LoraPackParams p) {
  grid_behind();
  const int64_t na = static_cast<int64_t>(p.R) * p.K, nb = static_cast<int64_t>(p.N) * p.ldb;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e * 8 < na + nb; e += static_cast<int64_t>(gridDim.x) * 256) {
    union { int4 v; __nv_bfloat16 h[8]; } o;
    if (e * 8 < na) {                                // a row of A, or a row of padding
      const int r = static_cast<int>(e * 8 / p.K), k = static_cast<int>(e * 8 - static_cast<int64_t>(r) * p.K);
      int i = 0;
      while (i + 1 < p.parts && r >= p.off[i + 1]) ++i;
      const int own = r - p.off[i];
      o.v = own < p.rank[i] ? *reinterpret_cast<const int4*>(static_cast<const __nv_bfloat16*>(p.a[i]) + static_cast<int64_t>(own) * p.K + k) : make_int4(0, 0, 0, 0);
      reinterpret_cast<int4*>(p.a_out)[e] = o.v;
    } else {                                         // eight columns of a row of the block-diagonal B
      const int64_t f = e * 8 - na;
      const int n = static_cast<int>(f / p.ldb), c = static_cast<int>(f - static_cast<int64_t>(n) * p.ldb);
      int i = 0, row = n;
      if (p.interleaved) {
        i = (n >> 7) & 1;
        row = (n >> 8) * 128 + (n & 127);
      } else {
        while (i + 1 < p.parts && n >= p.ends[i]) ++i;
        row = n - (i ? p.ends[i - 1] : 0);
      }
      const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b[i]) + static_cast<int64_t>(row) * p.rank[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int own = c + j - p.off[i];
        o.h[j] = own >= 0 && own < p.rank[i] ? b[own] : __float2bfloat16(0.f);
      }
      if (p.bias && c == p.R) o.h[0] = static_cast<const __nv_bfloat16*>(p.bias)[n];
      reinterpret_cast<int4*>(p.b_out)[f / 8] = o.v;
    }
  }
}

}  // namespace prl

using namespace prl;

// layout 0: A [M, K], B [R, K]; 1: A [M, K], B [K, R]; 2: A [K, M], B [K, R]; 3: as 2, out [R, M].  Pitches in elements, multiples of 8.
// pad > 0 (layouts 0 to 2): so many more columns of out, ones in the first.  lo_out > 0 (0 to 2): out gets what rounding left in columns lo_out on;
// lo_in > 0 (1 to 3): B has such halves from column lo_in.
extern "C" int prl_lora_thin(const void* A, const void* B, void* out, int M, int R, int K, int64_t lda, int64_t ldb, int64_t ldo, float scale, int layout, int pad,
                             int lo_out, int lo_in, int split, cudaStream_t stream) {
  if (M <= 0 || R <= 0 || K <= 0) return 0;
  if (R % 8 || lda % 8 || ldb % 8 || pad % 8 || lo_out % 8 || lo_in % 8 || (layout != 3 && ldo % 4) || (layout == 3 && lo_out) || (layout == 0 && lo_in)) return -1;
  ThinProduct q{A, B, lda, ldb, ThinParams{static_cast<__nv_bfloat16*>(out), ldo, M, R, K, 0, 0, scale, pad, lo_out, lo_in, nullptr, nullptr, 1, layout == 3, 0}};
  switch (layout) {
    case 0: return run_thin<false, false>(&q, 1, split, stream);
    case 1: return run_thin<false, true>(&q, 1, split, stream);
    case 2:
    case 3: return run_thin<true, true>(&q, 1, split, stream);
  }
  return -5;
}

// Both gradients of an adapter in one launch, over the same K rows: da [R, M1] = dt^T x, x [K, M1], dt [K, ..] with its halves R and R + lo_dt on; db [M2, R] = dy^T t
extern "C" int prl_lora_grads(const void* x, const void* dt, void* da, const void* dy, const void* t, void* db, int M1, int M2, int R, int K, int64_t ldx, int64_t lddt,
                              int64_t lddy, int64_t ldt, int lo_dt, int lo_t, int split, cudaStream_t stream) {
  if (M1 <= 0 || M2 <= 0 || R <= 0 || K <= 0) return -1;
  if (R % 8 || ldx % 8 || lddt % 8 || lddy % 8 || ldt % 8 || lo_dt % 8 || lo_t % 8 || lo_dt <= 0 || lo_t <= 0) return -1;
  ThinProduct q[2] = {{dy, t, lddy, ldt, ThinParams{static_cast<__nv_bfloat16*>(db), R, M2, R, K, 0, 0, 1.f, 0, 0, lo_t, nullptr, nullptr, 1, 0, 0}},
                      {x, dt, ldx, lddt, ThinParams{static_cast<__nv_bfloat16*>(da), M1, M1, R, K, 0, 0, 1.f, 0, 0, lo_dt, nullptr, nullptr, 1, 1, 0}}};
  return run_thin<true, true>(q, 2, split, stream);
}

// layout 0 for rows whose adapters differ: B [adapters * each, K], out [M, adapters * each (+ pad)], see ThinParams
extern "C" int prl_adapter_thin(const void* A, const void* B, void* out, int M, int R, int K, int64_t lda, int64_t ldb, int64_t ldo, int pad, const int32_t* ids,
                                const float* scales, int each, cudaStream_t stream) {
  if (M <= 0 || R <= 0 || K <= 0) return 0;
  if (R % 8 || lda % 8 || ldb % 8 || pad % 8 || ldo % 4 || each < 4 || each % 4 || R % each) return -1;
  ThinProduct q{A, B, lda, ldb, ThinParams{static_cast<__nv_bfloat16*>(out), ldo, M, R, K, 0, 0, 1.f, pad, 0, 0, ids, scales, each, 0, 0}};
  return run_thin<false, false>(&q, 1, 0, stream);
}

namespace prl {
// b [adapters, N, rank] -> [N, adapters * parts * rank (+ 8)]: row n holds every adapter's row n in the columns of its part, a bias behind them
__global__ void __launch_bounds__(256) adapter_pack_kernel(const __nv_bfloat16* __restrict__ b, const __nv_bfloat16* __restrict__ bias, int4* __restrict__ out,
                                                           const LoraPackParams p, int adapters, int rank) {
  grid_behind();
  const int units = p.ldb / 8, each = p.parts * rank;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < static_cast<int64_t>(p.N) * units; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int n = static_cast<int>(e / units), c = static_cast<int>(e % units) * 8;
    union { int4 v; __nv_bfloat16 h[8]; } o;
    o.v = make_int4(0, 0, 0, 0);
    if (c < adapters * each) {
      const int part = p.interleaved ? (n >> 7) & 1 : (p.parts > 1 && n >= p.ends[0]) + (p.parts > 2 && n >= p.ends[1]);
      const int l = c / each, k = c % each - part * rank;
      if (k >= 0 && k < rank) o.v = __ldg(reinterpret_cast<const int4*>(b + (static_cast<int64_t>(l) * p.N + n) * rank + k));
    } else if (bias) {
      o.h[0] = bias[n];
    }
    out[e] = o.v;
  }
}
}  // namespace prl

extern "C" int prl_adapter_pack(const void* b, const void* bias, void* out, const prl::LoraPackParams* q, int adapters, int rank, cudaStream_t stream) {
  if (q->N <= 0 || adapters <= 0 || rank % 8 || q->ldb % 8) return -1;
  const int64_t blocks = (static_cast<int64_t>(q->N) * (q->ldb / 8) + 255) / 256;
  PRL_CUDA_CHECK(launch_behind(adapter_pack_kernel, static_cast<unsigned>(blocks < 16 * 148 ? blocks : 16 * 148), 256, 0, stream, static_cast<const __nv_bfloat16*>(b),
                               static_cast<const __nv_bfloat16*>(bias), static_cast<int4*>(out), *q, adapters, rank));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

extern "C" int prl_lora_pack(const prl::LoraPackParams* q, cudaStream_t stream) {
  const int64_t units = (static_cast<int64_t>(q->R) * q->K + static_cast<int64_t>(q->N) * q->ldb) / 8;
  if (q->K % 8 || q->ldb % 8 || q->R % 8) return -1;
  const int64_t blocks = (units + 255) / 256;
  PRL_CUDA_CHECK(launch_behind(lora_pack_kernel, static_cast<unsigned>(blocks < 8 * 148 ? blocks : 8 * 148), 256, 0, stream, *q));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

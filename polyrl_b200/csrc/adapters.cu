// polyrl_b200 — what the adapters of a batch's rows add to a shared projection:
//
//   out[i, n] = s_l * sum_r B_l[n, r] * t_i[p(n) * rank + r]  (+ bias[n]) (+ res[i, n]),     t_i = A_l x_i,   l = ids[i]
//
// p(n) is the part of the fused projection that column n belongs to (query / key / value, or gate / up in blocks of 128).  A row without
// an adapter gets bias and residual alone.  With few rows the shared product comes first and this is added to it (`onto`): a row without an adapter
// then is what it is in a batch that has none, and any other is rounded twice, as bf16 2^-8 of the value at most each time.  With many rows this
// comes first, and the shared product adds it to its fp32 sums before it rounds.  t is rounded to bf16, as an operand of the second product.
//
// plan   one block sorts the rows by adapter (stable, by counting) and cuts every adapter's rows into tiles.  One plan serves all
//        projections of a step.
// delta  a cluster of CTAs takes a tile.  Few rows: the adapter's weights are all there is to read, so each CTA takes a share of K in the
//        first product and a share of N in the second and reads every weight once, 16 (8) bytes a lane, straight into the fragments of
//        mma.m16n8k16; nothing goes through shared memory but t, which the CTAs sum in a fixed order over distributed shared memory.
//        The lanes' k-indices (and the columns of the second product) are permuted so that a lane's fragments are contiguous in memory:
//        both operands of a product use the same permutation, and sums do not mind.
//        Ranks are a few dozen, so the products are bound by their operands' bytes and mma.sync keeps up; tcgen05 would want 128 rows of
//        one adapter and a round trip through tensor memory, longer than the whole kernel at decode.  What bounds it is latency: loads, two
//        cluster barriers and loads again, in 5.1 us for one row (K 896, N 1152), 8.9 for 128 rows of 24 adapters (4096, 6144, rank 16; 17 MB; 10.0
//        added to the shared product), 13.4 for 45 rows of 9 (3584, 37888, rank 32; 30 MB), 50 for 5003 rows of 5 (2048, 2048, rank 64; 64 MB).
//        With cold caches the first product takes half of the time and the second one a quarter.  Rows of a and x copied into shared memory in bulk,
//        512 bytes a request, took 11.8 us for the 128 rows; the loads of the second product a step ahead of its products, tiles of 64 rows and
//        three CTAs an SM were slower, too.  Bringing the next product's first weights into L2 from here did not shorten that product.
#include "adapters.hpp"
#include "common.cuh"

namespace prl {

// ------------------------------------------------------------------------------------------------------------ plan
// Every warp has a run of rows: it counts them by adapter, sums over the warps and groups give each count its first place, and the warp goes through its
// rows again, 32 at a time ranked by match, to put them there.  Nothing waits for the block between 32 rows: 128 rows 2.7 us, 5003 of five adapters 4.4 (8.3
// where the block ranks 1024 rows at a time).
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* __restrict__ ids, int T, int L, int tile_rows, int max_tiles,
                                                            int32_t* __restrict__ order, AdapterTile* __restrict__ tiles, int32_t* __restrict__ num_tiles) {
  extern __shared__ int32_t sm[];
  constexpr int kAhead = 4;                          // ids a lane has in flight
  const int G = L + 1;                               // the last group: no adapter
  int32_t* rows_of = sm;                             // [G] rows of the group, then where its first one goes
  int32_t* tile_at = sm + G;                         // [G] its first tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* mine = sm + (2 + warp) * G;               // [warps][G] a warp's rows of each group, then how many are before its next one
  grid_behind();
  const int each = (T + kPlanThreads - 1) / kPlanThreads * 32, warps = (T + each - 1) / each, row0 = min(warp * each, T), row1 = min(row0 + each, T);
  for (int i = tid; i < warps * G; i += kPlanThreads) sm[2 * G + i] = 0;
  __syncthreads();
  // f(row, its group or -1), 32 rows of the warp at a time
  auto rows = [&](auto f) {
    for (int r0 = row0; r0 < row1; r0 += 32 * kAhead) {
      int g[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int row = r0 + 32 * u + lane, id = row < row1 ? __ldg(ids + row) : 0;
        g[u] = row >= row1 ? -1 : id >= 0 && id < L ? id : L;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (r0 + 32 * u >= row1) break;
        f(r0 + 32 * u + lane, g[u]);
      }
    }
  };
  rows([&](int, int g) {
    if (g >= 0) atomicAdd(mine + g, 1);
  });
  __syncthreads();
  for (int g = tid; g < G; g += kPlanThreads) {      // counts -> how many of the group's rows are before the warp's
    int n = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = sm[(2 + w) * G + g];
      sm[(2 + w) * G + g] = n;
      n += c;
    }
    rows_of[g] = n;
  }
  __syncthreads();
  if (warp == 0) {                                   // exclusive sums of rows and of tiles over the groups
    int rows0 = 0, tiles0 = 0;
    for (int g0 = 0; g0 < G; g0 += 32) {
      const int g = g0 + lane, n = g < G ? rows_of[g] : 0, nt = (n + tile_rows - 1) / tile_rows;
      int rs = n, ts = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int r = __shfl_up_sync(0xffffffffu, rs, o), t = __shfl_up_sync(0xffffffffu, ts, o);
        if (lane >= o) { rs += r; ts += t; }
      }
      if (g < G) {
        rows_of[g] = rows0 + rs - n;
        tile_at[g] = tiles0 + ts - nt;
      }
      rows0 += __shfl_sync(0xffffffffu, rs, 31);
      tiles0 += __shfl_sync(0xffffffffu, ts, 31);
    }
    if (lane == 0) *num_tiles = min(tiles0, max_tiles);
  }
  __syncthreads();
  for (int g = warp; g < G; g += 32) {
    const int first = rows_of[g], n = (g + 1 < G ? rows_of[g + 1] : T) - first, t0 = tile_at[g];
    for (int k = lane; k * tile_rows < n && t0 + k < max_tiles; k += 32) tiles[t0 + k] = AdapterTile{g < L ? g : -1, first + k * tile_rows, min(tile_rows, n - k * tile_rows), 0};
  }
  rows([&](int row, int g) {
    const unsigned same = __match_any_sync(0xffffffffu, g);
    const int before = g >= 0 ? mine[g] : 0;
    __syncwarp();
    if (g >= 0) {
      order[rows_of[g] + before + __popc(same & ((1u << lane) - 1))] = row;
      if (lane == __ffs(same) - 1) mine[g] = before + __popc(same);
    }
    __syncwarp();
  });
}

// ------------------------------------------------------------------------------------------------------------ delta
constexpr int kLowChunk = 64;                        // low-rank columns whose sums a warp holds at a time

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t map_shared(const void* p, uint32_t cta) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
  return a;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

// TM rows a tile.  Shared memory: partial sums [TM][R] fp32, those of the KW warps that split K [KW][TM][kLowChunk], t [TM][R + 8] bf16 (rows an odd
// number of 16-byte units apart)
template <int TM>
struct DeltaCfg {
  static constexpr int MT = TM / 16, WARPS = 8, THREADS = 32 * WARPS, KW = WARPS / MT;
  static int smem(int R) { return TM * R * 4 + KW * TM * kLowChunk * 4 + TM * (R + 8) * 2; }
};

// ADD: bias, res or onto are there
template <int TM, bool ADD>
__global__ void __launch_bounds__(DeltaCfg<TM>::THREADS, 2) delta_kernel(const DeltaParams p) {
  using Cfg = DeltaCfg<TM>;
  constexpr int MT = Cfg::MT, KW = Cfg::KW, kThreads = Cfg::THREADS;
  extern __shared__ __align__(16) uint8_t raw[];
  const int R = p.parts * p.rank, ldt = R + 8;
  float* part = reinterpret_cast<float*>(raw);
  float* red = part + TM * R;
  __nv_bfloat16* low = reinterpret_cast<__nv_bfloat16*>(red + KW * TM * kLowChunk);
  __shared__ int32_t rows_sm[TM];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, grp = lane >> 2;
  const uint32_t cs = cluster_size(), rank = cluster_ctarank();
  const int cluster = blockIdx.x / cs, t = cluster / p.shares, share = cluster % p.shares * cs + rank, shares = p.shares * cs;
  grid_behind();
  if (t >= *p.num_tiles) return;
  const AdapterTile tile = p.tiles[t];
  if (tid < TM) rows_sm[tid] = tid < tile.rows ? p.order[tile.first + tid] : -1;
  __syncthreads();

  // this CTA's columns, 32 at a time, and its first weights of the second product, which can come while the first one runs
  const int groups = p.N / 32, g0 = static_cast<int>(static_cast<int64_t>(groups) * share / shares),
            g1 = static_cast<int>(static_cast<int64_t>(groups) * (share + 1) / shares);
  // lane's place in the rows of b for 32 columns from `col`: a lane's columns of the four products are 8 consecutive ones
  auto b_row = [&](int col) {
    return static_cast<const __nv_bfloat16*>(p.b) + (static_cast<int64_t>(tile.adapter) * p.N + col + 8 * (grp >> 1) + (grp & 1)) * p.rank;
  };
  if (tile.adapter >= 0) {
    if (tid == 0 && g0 < g1)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const __nv_bfloat16*>(p.b) + (static_cast<int64_t>(tile.adapter) * p.N + g0 * 32) * p.rank),
                   "r"((g1 - g0) * 64 * p.rank)
                   : "memory");
    // ---- t = A x over this CTA's share of K
    const int mt = warp % MT, kw = warp / MT;
    const int steps = p.K / 32, s0 = steps * rank / cs, s1 = steps * (rank + 1) / cs;
    const int r0 = rows_sm[mt * 16 + grp], r1 = rows_sm[mt * 16 + grp + 8];
    const __nv_bfloat16* x0 = static_cast<const __nv_bfloat16*>(p.x) + static_cast<int64_t>(max(r0, 0)) * p.ldx + quad * 8;
    const __nv_bfloat16* x1 = static_cast<const __nv_bfloat16*>(p.x) + static_cast<int64_t>(max(r1, 0)) * p.ldx + quad * 8;
    const int4 zero = make_int4(0, 0, 0, 0);
    for (int c0 = 0; c0 < R; c0 += kLowChunk) {
      const int nt = min(kLowChunk, R - c0) / 8;
      const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + (static_cast<int64_t>(tile.adapter) * R + c0 + grp) * p.K + quad * 8;
      float acc[8][4] = {};
      if (mt * 16 < tile.rows) {
#pragma unroll 2
        for (int s = s0 + kw; s < s1; s += KW) {
          const int4 u = r0 >= 0 ? __ldg(reinterpret_cast<const int4*>(x0 + s * 32)) : zero;
          const int4 v = r1 >= 0 ? __ldg(reinterpret_cast<const int4*>(x1 + s * 32)) : zero;
          int4 w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < nt) w[j] = __ldg(reinterpret_cast<const int4*>(a + static_cast<int64_t>(j) * 8 * p.K + s * 32));
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < nt) {
              mma_bf16(acc[j], u.x, v.x, u.y, v.y, w[j].x, w[j].y);
              mma_bf16(acc[j], u.z, v.z, u.w, v.w, w[j].z, w[j].w);
            }
        }
      }
      float* dst = red + (kw * TM + mt * 16 + grp) * kLowChunk + quad * 2;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < nt) {
          *reinterpret_cast<float2*>(dst + j * 8) = make_float2(acc[j][0], acc[j][1]);
          *reinterpret_cast<float2*>(dst + 8 * kLowChunk + j * 8) = make_float2(acc[j][2], acc[j][3]);
        }
      __syncthreads();
      for (int e = tid; e < tile.rows * nt * 4; e += kThreads) {
        const int m = e / (nt * 4), c = e % (nt * 4) * 2;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          const float2 q = *reinterpret_cast<const float2*>(red + (k * TM + m) * kLowChunk + c);
          v.x += q.x; v.y += q.y;
        }
        *reinterpret_cast<float2*>(part + m * R + c0 + c) = v;
      }
      __syncthreads();
    }
    // ---- the CTAs' sums, each for its share of the values, in the order of the ranks; scaled, rounded and given to all
    const float scale = p.scales[tile.adapter];
    if (cs > 1) cluster_sync_all();
    const int pairs = tile.rows * (R / 2), e1 = pairs * (rank + 1) / cs;
    for (int e = pairs * rank / cs + tid; e < e1; e += kThreads) {
      const int m = e / (R / 2), c = e % (R / 2) * 2;
      float2 v = make_float2(0.f, 0.f);
      if (cs == 1) {
        v = *reinterpret_cast<float2*>(part + m * R + c);
      } else {
        float2 q[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
          if (k < cs) q[k] = ld_cluster_f2(map_shared(part + m * R + c, k));
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
          if (k < cs) { v.x += q[k].x; v.y += q[k].y; }
      }
      const uint32_t packed = pack_bf16(scale * v.x, scale * v.y);
      if (cs == 1) {
        *reinterpret_cast<uint32_t*>(low + m * ldt + c) = packed;
      } else {
        for (uint32_t k = 0; k < cs; ++k) st_cluster_u32(map_shared(low + m * ldt + c, k), packed);
      }
    }
    if (cs > 1) cluster_sync_all();                  // after this nobody touches another CTA's shared memory
    else __syncthreads();
  }

  // ---- out = t B^T (+ bias) (+ res) (+ base) over this CTA's share of the columns
  for (int g = g0 + warp; g < g1; g += Cfg::WARPS) {
    const int col = g * 32;
    const int pt = p.interleaved ? (col >> 7) & 1 : (p.parts > 1 && col >= p.ends[0]) + (p.parts > 2 && col >= p.ends[1]);
    const int4 none = make_int4(0, 0, 0, 0);
    int4 extra = none, add[MT][2], own[MT][2];
    if constexpr (ADD) {
      if (p.bias) extra = __ldg(reinterpret_cast<const int4*>(static_cast<const __nv_bfloat16*>(p.bias) + col + quad * 8));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = rows_sm[m * 16 + grp + 8 * h];
          add[m][h] = p.res && row >= 0 ? ld_nc_v4(static_cast<const __nv_bfloat16*>(p.res) + static_cast<int64_t>(row) * p.ldr + col + quad * 8) : none;
          own[m][h] = p.onto && row >= 0 ? ld_v4(static_cast<const __nv_bfloat16*>(p.out) + static_cast<int64_t>(row) * p.ldo + col + quad * 8) : none;
        }
    }
    float acc[MT][4][4] = {};
    if (tile.adapter >= 0) {
      const __nv_bfloat16* b = b_row(col);
      const __nv_bfloat16* tl = low + pt * p.rank;
      int k = 0;
#pragma unroll 2
      for (; k + 32 <= p.rank; k += 32) {            // 16 bytes a lane: two steps of 16
        int4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const int4*>(b + 2 * j * p.rank + k + quad * 8));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int4 u = *reinterpret_cast<const int4*>(tl + (m * 16 + grp) * ldt + k + quad * 8);
          const int4 v = *reinterpret_cast<const int4*>(tl + (m * 16 + grp + 8) * ldt + k + quad * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_bf16(acc[m][j], u.x, v.x, u.y, v.y, w[j].x, w[j].y);
            mma_bf16(acc[m][j], u.z, v.z, u.w, v.w, w[j].z, w[j].w);
          }
        }
      }
      if (k < p.rank) {
        uint2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint2*>(b + 2 * j * p.rank + k + quad * 4));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint2 u = *reinterpret_cast<const uint2*>(tl + (m * 16 + grp) * ldt + k + quad * 4);
          const uint2 v = *reinterpret_cast<const uint2*>(tl + (m * 16 + grp + 8) * ldt + k + quad * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_bf16(acc[m][j], u.x, v.x, u.y, v.y, w[j].x, w[j].y);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = rows_sm[m * 16 + grp + 8 * h];
        if (row < 0) continue;
        int4 o;
        int* ow = reinterpret_cast<int*>(&o);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 v = make_float2(acc[m][j][2 * h], acc[m][j][2 * h + 1]);
          if constexpr (ADD) {
            const float2 e = unpack_bf16(reinterpret_cast<const uint32_t*>(&extra)[j]), r = unpack_bf16(reinterpret_cast<const uint32_t*>(&add[m][h])[j]),
                         y = unpack_bf16(reinterpret_cast<const uint32_t*>(&own[m][h])[j]);
            v.x += e.x + r.x + y.x;
            v.y += e.y + r.y + y.y;
          }
          ow[j] = static_cast<int>(pack_bf16(v.x, v.y));
        }
        st_v4(static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(row) * p.ldo + col + quad * 8, o);
      }
  }
}

template <int TM>
static int run_delta(const DeltaParams& p, int ctas, cudaStream_t stream) {
  const int smem = DeltaCfg<TM>::smem(p.parts * p.rank);
  auto kern = p.bias || p.res || p.onto ? delta_kernel<TM, true> : delta_kernel<TM, false>;
  PRL_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DeltaCfg<TM>::smem(kDeltaMaxLow)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.max_tiles) * p.shares * ctas);
  cfg.blockDim = dim3(DeltaCfg<TM>::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  PRL_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

}  // namespace prl

extern "C" int prl_adapter_plan(const int32_t* ids, int T, int L, int tile_rows, int max_tiles, int32_t* order, void* tiles, int32_t* num_tiles, cudaStream_t stream) {
  if (T <= 0 || L < 1 || L > prl::kPlanMaxAdapters || tile_rows < 1) return -1;
  const int smem = 34 * (L + 1) * 4;
  PRL_CUDA_CHECK(cudaFuncSetAttribute(prl::plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 34 * (prl::kPlanMaxAdapters + 1) * 4));
  PRL_CUDA_CHECK(launch_behind(prl::plan_kernel, 1, prl::kPlanThreads, smem, stream, ids, T, L, tile_rows, max_tiles, order,
                               static_cast<prl::AdapterTile*>(tiles), num_tiles));
  PRL_CUDA_CHECK(cudaGetLastError());
  return 0;
}

// tile_rows 16 or 32, as the plan was made; ctas: of a cluster, shares: clusters that take a tile's columns between them, each with the whole first
// product; 0 = as many CTAs (8 at most) as leave about four for every SM, and where that leaves fewer than one, more shares of at least 512 columns a CTA
extern "C" int prl_adapter_delta(const prl::DeltaParams* q, int tile_rows, int ctas, int shares, cudaStream_t stream) {
  prl::DeltaParams p = *q;
  if (p.max_tiles <= 0) return 0;
  if (p.K <= 0 || p.K % 32 || p.N <= 0 || p.N % 32 || p.rank < 16 || p.rank % 16 || p.parts < 1 || p.parts > 3 || p.parts * p.rank > prl::kDeltaMaxLow) return -1;
  if (ctas <= 0) {
    ctas = 8;
    while (ctas > 1 && static_cast<int64_t>(p.max_tiles) * ctas > 4 * 148) ctas >>= 1;
  }
  if (shares <= 0) {
    shares = 1;
    while (static_cast<int64_t>(p.max_tiles) * ctas * shares < 148 && p.N / (2 * shares * ctas) >= 512) shares *= 2;
  }
  if (ctas != 1 && ctas != 2 && ctas != 4 && ctas != 8) return -2;
  p.shares = shares;
  if (static_cast<int64_t>(p.max_tiles) * ctas * shares > 0x7fffffff) return -3;
  if (tile_rows == 16) return prl::run_delta<16>(p, ctas, stream);
  if (tile_rows == 32) return prl::run_delta<32>(p, ctas, stream);
  return -4;
}

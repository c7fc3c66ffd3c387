// polyrl_b200 — operands of the adapter kernels (adapters.cu), shared with the bindings.
#pragma once
#include <cstdint>

namespace prl {

constexpr int kPlanMaxAdapters = 1024;
constexpr int kDeltaMaxLow = 384;                   // low-rank columns: parts times rank

// A tile of rows that share an adapter: rows order[first .. first + rows), adapter -1 for rows without one.
struct AdapterTile {
  int32_t adapter, first, rows, pad;
};

struct DeltaParams {
  const void* x;                   // [T, K] bf16
  const void* a;                   // [adapters, parts * rank, K] bf16
  const void* b;                   // [adapters, N, rank] bf16
  const float* scales;             // [adapters]
  const void* bias;                // [N] bf16 or null
  const void* res;                 // [T, N] bf16 or null
  void* out;                       // [T, N] bf16
  const int32_t* order;
  const AdapterTile* tiles;
  const int32_t* num_tiles;
  int64_t ldx, ldr, ldo;
  int K, N, rank, parts, max_tiles;
  int ends[3];                     // column where each part ends; interleaved: parts alternate in blocks of 128 columns
  int interleaved;
  int onto;                        // out holds the shared product: added to
  int shares;                      // clusters a tile
};

}  // namespace prl

// polyrl_b200 — operands of the adapter packing kernel (lora.cu), shared with the bindings.
#pragma once
#include <cstdint>

namespace prl {

// Contiguous bf16 parts a[i] [rank[i], K] and b[i] [columns of the part, rank[i]]; rank 0: a part without an adapter (null pointers).
struct LoraPackParams {
  const void *a[3], *b[3];
  const void* bias;                // [N] or null: goes to column R of b_out
  void* a_out;                     // [R, K]
  void* b_out;                     // [N, ldb]
  int rank[3], off[3], ends[3];    // off: the part's first row of a_out and column of b_out
  int parts, interleaved, R, K, N, ldb;
};

}  // namespace prl

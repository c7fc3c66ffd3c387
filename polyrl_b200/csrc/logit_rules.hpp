// polyrl_b200 — operands of the logit rules kernel (logit_rules.cu), shared with the bindings.
#pragma once
#include <cstdint>

namespace prl {

constexpr int kRuleThreads = 512;
constexpr int kRuleCountBits = 20;                  // a history is shorter than 2^20 tokens
constexpr int kRuleShortBits = 13;                  // shorter than 2^13: 16 bits a token
constexpr int kRuleMaxBias = 2046;                  // entries of a row's bias list
constexpr int kRulePart = 16384;                    // most tokens of the vocabulary a block takes: their places are packed into 16 bits

// Strides in elements.  A pointer that is null leaves its rule out.
struct RuleParams {
  const void* z;
  void* out;                       // may be z
  int64_t ldz, ldo;
  int rows, V;
  const int32_t* tokens;           // [rows, max_tokens]: prompt tokens, then output tokens; ids outside the vocabulary count for nothing
  int64_t ld_tokens;
  int max_tokens;
  const int32_t *lens, *prompt_lens;
  const float *rep, *pres, *freq;  // [rows]
  const int32_t* bias_ids;         // [rows, num_bias]; ids outside the vocabulary: no entry
  const float* bias_values;
  int64_t ld_bias;
  int num_bias;
  const int32_t* stop_ids;         // [rows, num_stop], with min_lens: may not come while lens < min_lens
  int64_t ld_stop;
  int num_stop;
  const int32_t* min_lens;
  const int32_t* masks;            // [num_masks, words]: bit v % 32 of word v / 32 says whether token v may come
  int64_t ld_masks;
  int num_masks;
  const int32_t* mask_rows;        // [rows]: the row's mask, negative for none; null: mask b belongs to row b
};

}  // namespace prl

// Host-side description of a scored attention launch over prompts.
#pragma once

#include "prefill_launch.hpp"
#include "score.hpp"

namespace sia {

// scored_rows: any head_dim of 16 ... 256, f16 or bf16, one wave per query row.
struct ScoredRowsArgs {
  const char* q; int64_t q_sb, q_sh, q_sm;     // byte strides; head_dim contiguous
  const char* k; int64_t k_sb, k_sh, k_sn;
  const char* v; int64_t v_sb, v_sh, v_sn;
  char* out; int64_t o_sb, o_sh, o_sm;
  int32_t B, Hq, G, Tq, Tk;
  int64_t rows;                                // B Hq Tq
  float qk_scale;                              // sm_scale log2(e)
  ScoreArgs s;
};
int launch_scored_rows(const ScoredRowsArgs& a, int D, int dtype, hipStream_t stream);

// Checks a call's score options (NULL: none) and fills the kernels' arguments; prompt: the fields for prompts are allowed.
int fill_score(const sia_score_options* o, bool prompt, int64_t B, int64_t Hq, float sm_scale, int causal, ScoreArgs& s);

}  // namespace sia

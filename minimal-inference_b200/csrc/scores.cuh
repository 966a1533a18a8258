// Accumulated attention weights (scores.cu, scores_tc.cu): shared arguments.
#pragma once

#include "mi_common.cuh"

namespace mi {

struct ScoreParams {
  const void *q;
  int64_t qsn, qsh;
  const int32_t *qo_indptr;  // null: one query per request, row = request
  int total_q;
  const void *kv;
  int64_t num_pages;
  int ps, hkv, d;
  const int32_t *indptr, *indices, *last;
  int batch, hq, group;
  int causal, window;  // window <= 0: all queries
  float scale;
  const float *lse;  // [total_q][hq], natural log
  float *scores;     // [num_pages][hkv][ps]
  int32_t *status;
};

// Tensor-core prompt scores (scores_tc.cu). ctr: two work-item counters, zero
// between calls, or null (fixed round robin). Returns -1 (nothing launched)
// when the shape or layout is outside its coverage.
int launch_scores_tc(const ScoreParams &p, int dtype, unsigned *ctr, cudaStream_t s);

}  // namespace mi

// Stream-K TMA decode kernel (decode_sk.cu): arguments and entry points used
// by the mi_paged_decode dispatcher in decode.cu.
#pragma once

#include "mi_common.cuh"

namespace mi {

struct SkArgs {
  const void *q;
  int64_t qsb, qsh;
  const void *kv;
  int64_t num_pages;
  int ps, hkv, d, dtype;
  const int32_t *indptr, *indices, *last;
  int batch, hq;
  float sm_scale;
  void *out;
  float *lse;
  void *ws;
  size_t ws_bytes;
  int32_t *status;
  cudaStream_t stream;
  // fused append (mi_paged_decode_append); k_new == nullptr: plain decode
  const void *k_new = nullptr, *v_new = nullptr;
  int64_t ksb = 0, ksh = 0, vsb = 0, vsh = 0;
  const void *rope_cos = nullptr, *rope_sin = nullptr;
  int rope_max = 0;
  // score form (mi_paged_decode_scores): scaled logits [hq][logit_stride] and
  // log2-sum-exp [batch][hq] also come out; null: not wanted
  float *logits = nullptr, *lse2 = nullptr;
  int64_t logit_stride = 0;
  const int32_t *rope_pos = nullptr;  // RoPE position per request (null: its last slot)
};

// Shapes and alignments the workspace kernels (stream-K, then the ticket
// kernel) serve; every other call runs the generic kernel, which needs no
// workspace.
bool decode_fast_shape(const void *q, int64_t qsb, int64_t qsh, const void *kv, const void *out,
                       int head_dim, int dtype, int group, int batch);
// Workspace bytes the stream-K kernel needs for this shape.
size_t decode_sk_workspace_bytes(int batch, int hq, int hkv, int d);
// Launches the stream-K kernel; returns -1 (nothing launched) when the
// shape, alignment or workspace is outside its coverage.
int launch_decode_sk(const SkArgs &a);

}  // namespace mi

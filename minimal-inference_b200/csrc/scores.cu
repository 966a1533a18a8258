// Accumulated attention weights of cached tokens, per KV head:
//   scores[page][h][slot] += sum over queries i and the group's heads g of
//                            exp(q_ig . k_slot * sm_scale - lse_ig),
// what an eviction by accumulated weight (evict.cu) ranks the cache by. The
// reference keeps every token (its cache only grows); no counterpart there.
//
// Two forms:
//   * Decode (one query per request): the stream-K decode kernel already has
//     every logit, so its score form stores them (fp32, log2 units; written and
//     read back 8 bytes a token and query head, 1/16 of the bytes of K and V at
//     4 heads of 128 per KV head, from L2 while a batch's fit it) and
//     weights_kernel turns them into weights once the row sums are known:
//     no second pass over K. fp32 and odd head sizes do the same in three
//     plain kernels (logits by 16-token pieces, softmax and P V by row); other
//     shapes run the generic prompt form after the decode.
//   * A prompt's last `window` queries, whose log-sum-exp the prefill
//     attention returned (scores_tc.cu for 16-bit types; the generic kernel
//     here for any type and head_dim).
// Sums are fp32 and per token in a fixed order; the addition into `scores` is
// one fp32 reduction per token and KV head (red.add), so a page listed once
// gets the same bits every time, and one listed twice gets both sums.
#include <algorithm>

#include "decode_sk.cuh"
#include "mi_common.cuh"
#include "scores.cuh"

namespace mi {
namespace {

__device__ __forceinline__ void red_add(float *p, float v) {
  asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory");
}

// Request that holds page position `pos` (counted from indptr[0]).
__device__ __forceinline__ int request_of(const int32_t *indptr, int batch, int pos) {
  const int base = indptr[0];
  int l = 0, h = batch - 1;
  while (l < h) {
    const int mid = (l + h + 1) >> 1;
    if (indptr[mid] - base <= pos) l = mid; else h = mid - 1;
  }
  return l;
}

// ---- generic ---------------------------------------------------------------
// Work item: 16 tokens of a page under one KV head. K rows in shared memory
// as fp32 (row stride d + 1: the 16 tokens of a half-warp in different banks);
// thread = (token, part): every 8th (query, group head) row, dot products in
// fp32 over the whole head, the parts added in order at the end.
constexpr int kGTok = 16, kGParts = 8;

template <typename T>
__global__ void __launch_bounds__(kGTok *kGParts) scores_generic_kernel(const ScoreParams p) {
  extern __shared__ float s_k[];  // [16][d + 1]
  __shared__ float s_part[kGParts][kGTok];
  const int total = p.indptr[p.batch] - p.indptr[0];
  const int chunks = (p.ps + kGTok - 1) / kGTok;
  const int64_t items = static_cast<int64_t>(total) * chunks * p.hkv;
  const int tok = threadIdx.x % kGTok, part = threadIdx.x / kGTok;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int h = static_cast<int>(it % p.hkv);
    const int chunk = static_cast<int>(it / p.hkv % chunks);
    const int pos = static_cast<int>(it / p.hkv / chunks);
    const int b = request_of(p.indptr, p.batch, pos);
    const int first = p.indptr[b] - p.indptr[0];
    const int kvlen = kv_len_of(p.indptr, p.last, b, p.ps);
    const int slot0 = chunk * kGTok;
    const int j0 = (pos - first) * p.ps + slot0;  // the chunk's first token
    const int nt = min(min(kGTok, p.ps - slot0), kvlen - j0);
    if (nt <= 0) continue;
    const int64_t page = p.indices[p.indptr[0] + pos];
    if (page < 0 || page >= p.num_pages) {
      if (threadIdx.x == 0) flag(p.status, MI_STATUS_BAD_PAGE);
      continue;
    }
    // the request's queries: rows [q0, q0 + nq), the last `window` of them
    int q0 = b, nq = 1;
    if (p.qo_indptr) {
      q0 = p.qo_indptr[b];
      nq = p.qo_indptr[b + 1] - q0;
      if (q0 < 0 || nq <= 0 || q0 + nq > p.total_q) {
        if (nq != 0 && threadIdx.x == 0) flag(p.status, MI_STATUS_BAD_POSITION);
        continue;
      }
    }
    const int i0 = p.window > 0 ? max(0, nq - p.window) : 0;
    __syncthreads();  // the previous item's readers are done
    const T *kp = static_cast<const T *>(p.kv) +
                  ((page * 2) * p.ps + slot0) * (static_cast<int64_t>(p.hkv) * p.d) +
                  static_cast<int64_t>(h) * p.d;
    for (int e = threadIdx.x; e < nt * p.d; e += blockDim.x) {
      const int r = e / p.d, c = e % p.d;
      s_k[r * (p.d + 1) + c] = Elt<T>::to(kp[static_cast<int64_t>(r) * p.hkv * p.d + c]);
    }
    __syncthreads();
    float sum = 0.f;
    if (tok < nt) {
      const int j = j0 + tok;
      const float *kr = s_k + tok * (p.d + 1);
      // causal: query i sees tokens j <= kvlen - nq + i
      const int lo = p.causal ? max(i0, j - (kvlen - nq)) : i0;
      const int rows = max(0, nq - lo) * p.group;
      for (int r = part; r < rows; r += kGParts) {
        const int i = q0 + lo + r / p.group, hq = h * p.group + r % p.group;
        const float l = p.lse[static_cast<int64_t>(i) * p.hq + hq];
        if (l == -INFINITY) continue;  // a row that saw nothing
        const T *qr = static_cast<const T *>(p.q) + i * p.qsn + hq * p.qsh;
        float s = 0.f;
        for (int c = 0; c < p.d; ++c) s = fmaf(Elt<T>::to(qr[c]), kr[c], s);
        sum += expf(fmaf(s, p.scale, -l));
      }
    }
    s_part[part][tok] = sum;
    __syncthreads();
    if (threadIdx.x < nt) {
      float t = 0.f;
      for (int i = 0; i < kGParts; ++i) t += s_part[i][threadIdx.x];
      red_add(p.scores + (page * p.hkv + h) * p.ps + slot0 + threadIdx.x, t);
    }
  }
}

template <typename T>
int launch_generic_t(const ScoreParams &p, cudaStream_t s) {
  const int smem = kGTok * (p.d + 1) * 4;
  scores_generic_kernel<T><<<num_sms() * 8, kGTok * kGParts, smem, s>>>(p);
  return check_launch("scores_generic_kernel");
}

int launch_generic(const ScoreParams &p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case MI_DTYPE_F32: return launch_generic_t<float>(p, s);
    case MI_DTYPE_F16: return launch_generic_t<__half>(p, s);
    default: return launch_generic_t<__nv_bfloat16>(p, s);
  }
}

// ---- generic decode ---------------------------------------------------------
// Logits of every token: the same work items and dot products as above, each
// (token, query head) stored in log2 units at [hq][stride].
template <typename T>
__global__ void __launch_bounds__(kGTok *kGParts) logits_generic_kernel(
    const ScoreParams p, float *logits, int64_t stride) {
  extern __shared__ float s_k[];  // [16][d + 1]
  const int total = p.indptr[p.batch] - p.indptr[0];
  const int chunks = (p.ps + kGTok - 1) / kGTok;
  const int64_t items = static_cast<int64_t>(total) * chunks * p.hkv;
  const int tok = threadIdx.x % kGTok, part = threadIdx.x / kGTok;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int h = static_cast<int>(it % p.hkv);
    const int chunk = static_cast<int>(it / p.hkv % chunks);
    const int pos = static_cast<int>(it / p.hkv / chunks);
    const int b = request_of(p.indptr, p.batch, pos);
    const int slot0 = chunk * kGTok;
    const int64_t at = static_cast<int64_t>(pos) * p.ps + slot0;  // in a row of logits
    const int j0 = (pos - (p.indptr[b] - p.indptr[0])) * p.ps + slot0;
    const int nt = min(min(kGTok, p.ps - slot0), kv_len_of(p.indptr, p.last, b, p.ps) - j0);
    if (nt <= 0 || at + nt > stride) continue;
    const int64_t page = p.indices[p.indptr[0] + pos];
    const bool bad = page < 0 || page >= p.num_pages;
    if (bad && threadIdx.x == 0) flag(p.status, MI_STATUS_BAD_PAGE);
    __syncthreads();  // the previous item's readers are done
    if (!bad) {
      const T *kp = static_cast<const T *>(p.kv) +
                    ((page * 2) * p.ps + slot0) * (static_cast<int64_t>(p.hkv) * p.d) +
                    static_cast<int64_t>(h) * p.d;
      for (int e = threadIdx.x; e < nt * p.d; e += blockDim.x) {
        const int r = e / p.d, c = e % p.d;
        s_k[r * (p.d + 1) + c] = Elt<T>::to(kp[static_cast<int64_t>(r) * p.hkv * p.d + c]);
      }
    }
    __syncthreads();
    if (tok < nt) {
      const float *kr = s_k + tok * (p.d + 1);
      for (int r = part; r < p.group; r += kGParts) {
        const int hq = h * p.group + r;
        float s = -INFINITY;  // a bad page's tokens are left out
        if (!bad) {
          const T *qr = static_cast<const T *>(p.q) + b * p.qsn + hq * p.qsh;
          s = 0.f;
          for (int c = 0; c < p.d; ++c) s = fmaf(Elt<T>::to(qr[c]), kr[c], s);
          s *= p.scale * kLog2e;
        }
        logits[hq * stride + at + tok] = s;
      }
    }
  }
}

// One CTA per (request, query head): maximum and sum of its logits, then P V
// with a thread per element of head_dim and as many token streams as fit, 8
// rows of V in flight each; the streams' sums are added in order.
// The three generic kernels together are a chain of latencies: 4 requests of
// 37-500 tokens, fp32, 14/2 heads of 64, take 32.8 us for 1.1 MB.
constexpr int kRowThreads = 1024;  // (with 256 a row of 500 tokens takes 20 us longer)

template <typename T>
__global__ void __launch_bounds__(kRowThreads) row_generic_kernel(
    const ScoreParams p, const float *logits, int64_t stride, T *out, float *lse, float *lse2) {
  __shared__ float s_red[kRowThreads];
  const int b = blockIdx.x, hq = blockIdx.y, h = hq / p.group;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = p.indptr[b] - p.indptr[0];
  const int64_t base = static_cast<int64_t>(first) * p.ps;
  const int n = static_cast<int>(
      max(int64_t(0), min(int64_t(kv_len_of(p.indptr, p.last, b, p.ps)), stride - base)));
  const float *x = logits + hq * stride + base;
  float m = -INFINITY;
  for (int t = tid; t < n; t += kRowThreads) m = fmaxf(m, x[t]);
  m = warp_max(m);
  if (lane == 0) s_red[warp] = m;
  __syncthreads();
  for (int i = 0; i < kRowThreads / 32; ++i) m = fmaxf(m, s_red[i]);
  __syncthreads();
  float l = 0.f;
  if (m > -INFINITY)
    for (int t = tid; t < n; t += kRowThreads) l += exp2f(x[t] - m);
  l = warp_sum(l);
  if (lane == 0) s_red[warp] = l;
  __syncthreads();
  l = 0.f;
  for (int i = 0; i < kRowThreads / 32; ++i) l += s_red[i];
  __syncthreads();
  const float all = m + log2f(l);
  if (tid == 0) {
    lse2[b * p.hq + hq] = l > 0.f ? all : INFINITY;  // (+inf: every weight is 0)
    if (lse) lse[b * p.hq + hq] = l > 0.f ? all * kLn2 : -INFINITY;
  }
  const int streams = max(1, kRowThreads / p.d);  // head_dim <= 256
  const int c = tid % p.d, st = tid / p.d;
  const int64_t row = static_cast<int64_t>(p.hkv) * p.d;
  float acc = 0.f;
  if (st < streams && l > 0.f) {
    const T *v = static_cast<const T *>(p.kv) + p.ps * row + static_cast<int64_t>(h) * p.d + c;
    const int32_t *table = p.indices + p.indptr[b];
    constexpr int kAhead = 8;
    for (int t0 = st; t0 < n; t0 += streams * kAhead) {
      float w[kAhead], vv[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int t = t0 + i * streams;
        w[i] = t < n ? x[t] : -INFINITY;
        const int64_t page = t < n ? table[t / p.ps] : -1;
        vv[i] = page >= 0 && page < p.num_pages
                    ? Elt<T>::to(v[(page * 2 * p.ps + t % p.ps) * row]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) acc = fmaf(exp2f(w[i] - m), vv[i], acc);
    }
  }
  s_red[tid] = acc;
  __syncthreads();
  if (st == 0) {
    for (int i = 1; i < streams; ++i) acc += s_red[i * p.d + c];
    out[(static_cast<int64_t>(b) * p.hq + hq) * p.d + c] =
        Elt<T>::from(l > 0.f ? acc / l : 0.f);
  }
}

template <typename T>
int launch_generic_decode_t(const ScoreParams &p, float *logits, int64_t stride, void *out,
                            float *lse, float *lse2, cudaStream_t s) {
  const int64_t items = stride / p.ps * ((p.ps + kGTok - 1) / kGTok) * p.hkv;
  const int blocks = static_cast<int>(std::min<int64_t>(items, num_sms() * 8));
  logits_generic_kernel<T><<<blocks, kGTok * kGParts, kGTok * (p.d + 1) * 4, s>>>(p, logits,
                                                                                  stride);
  int rc = check_launch("logits_generic_kernel");
  if (rc) return rc;
  row_generic_kernel<T><<<dim3(p.batch, p.hq), kRowThreads, 0, s>>>(
      p, logits, stride, static_cast<T *>(out), lse, lse2);
  return check_launch("row_generic_kernel");
}

int launch_generic_decode(const ScoreParams &p, int dtype, float *logits, int64_t stride,
                          void *out, float *lse, float *lse2, cudaStream_t s) {
  switch (dtype) {
    case MI_DTYPE_F32: return launch_generic_decode_t<float>(p, logits, stride, out, lse, lse2, s);
    case MI_DTYPE_F16: return launch_generic_decode_t<__half>(p, logits, stride, out, lse, lse2, s);
    default:
      return launch_generic_decode_t<__nv_bfloat16>(p, logits, stride, out, lse, lse2, s);
  }
}

// ---- decode: stored logits to weights ----------------------------------------
// One thread per (token, KV head): grid y = KV head, x strides over the page
// positions' slots. Reads of a head's logits and the score additions are both
// contiguous over the tokens of a page. The decode with scores, this kernel
// included (bf16, CUDA graph): 61.8 us for 32 requests of 256-4096 tokens and
// 32/8 heads of 128 (0.72 of the copy rate over the bytes of both), of which
// 54 are the decode kernel's, bound by HBM; 33.1 us for one of 32000 tokens
// and 28/4 heads (0.31), where the start, the merge of 148 partial rows and
// this kernel's latency weigh as much as the bytes.
__global__ void __launch_bounds__(256) weights_kernel(
    const float *__restrict__ logits, int64_t stride, const float *__restrict__ lse2,
    const int32_t *indptr, const int32_t *indices, const int32_t *last, int batch, int group,
    int hq, int ps, int hkv, int64_t num_pages, float *scores) {
  pdl_trigger();  // dependents wait for this grid themselves; it writes only scores
  const int h = blockIdx.y;
  const int base = indptr[0];
  const int64_t n = min(static_cast<int64_t>(indptr[batch] - base) * ps, stride);
  bool waited = false;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    // the token's request and page, under the decode's last kernel
    const int pos = static_cast<int>(i / ps), slot = static_cast<int>(i % ps);
    const int b = request_of(indptr, batch, pos);
    const int first = indptr[b] - base;
    const bool real =
        static_cast<int64_t>(pos - first) * ps + slot < kv_len_of(indptr, last, b, ps);
    const int64_t page = indices[base + pos];
    if (!waited) pdl_wait();
    waited = true;
    if (!real || page < 0 || page >= num_pages) continue;  // (a bad page: flagged by the decode)
    const float *lg = logits + static_cast<int64_t>(h) * group * stride + i;
    const float *l2 = lse2 + b * hq + h * group;
    float w = 0.f;
#pragma unroll 8
    for (int g = 0; g < group; ++g) w += exp2f(lg[g * stride] - l2[g]);
    red_add(scores + (page * hkv + h) * ps + slot, w);
  }
  if (!waited) pdl_wait();  // this grid ends after the decode's, whoever waits for it
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace
}  // namespace mi

extern "C" size_t mi_paged_decode_scores_scratch_size(int32_t batch_size, int32_t num_qo_heads,
                                                      int32_t page_size, int64_t max_pages) {
  if (batch_size <= 0 || num_qo_heads <= 0 || page_size <= 0 || max_pages <= 0) return 0;
  return mi::up256(size_t(batch_size) * num_qo_heads * 4) +
         size_t(max_pages) * page_size * num_qo_heads * 4;
}

extern "C" int mi_paged_decode_scores(
    const void *q, int64_t q_stride_b, int64_t q_stride_h,
    const void *k_new, int64_t k_stride_b, int64_t k_stride_h,
    const void *v_new, int64_t v_stride_b, int64_t v_stride_h,
    const void *rope_cos, const void *rope_sin, int32_t rope_max_pos,
    const int32_t *rope_positions,
    void *kv_data, int64_t num_pages, int32_t page_size, int32_t num_kv_heads,
    int32_t head_dim, int32_t dtype,
    const int32_t *kv_indptr, const int32_t *kv_indices, int64_t max_pages,
    const int32_t *kv_last_page_len, int32_t batch_size, int32_t num_qo_heads, float sm_scale,
    void *out, float *lse, float *scores, void *scratch, size_t scratch_bytes,
    void *workspace, size_t workspace_bytes, int32_t *status, mi_stream_t stream) {
  using namespace mi;
  MI_REQUIRE(batch_size >= 0, "decode_scores: negative batch_size");
  if (batch_size == 0) return MI_OK;
  MI_REQUIRE(q && kv_data && kv_indptr && kv_indices && kv_last_page_len && out && scores &&
                 scratch && workspace,
             "decode_scores: null pointer argument");
  MI_REQUIRE(page_size > 0 && num_kv_heads > 0 && head_dim > 0 && head_dim <= 256 &&
                 num_pages > 0 && max_pages > 0,
             "decode_scores: bad pool geometry");
  MI_REQUIRE(num_qo_heads <= 65535, "decode_scores: too many heads");
  MI_REQUIRE(num_qo_heads >= num_kv_heads && num_qo_heads % num_kv_heads == 0,
             "decode_scores: num_qo_heads %d is not a multiple of num_kv_heads %d", num_qo_heads,
             num_kv_heads);
  MI_REQUIRE(dtype == MI_DTYPE_F32 || dtype == MI_DTYPE_F16 || dtype == MI_DTYPE_BF16,
             "decode_scores: bad dtype %d", dtype);
  MI_REQUIRE(!k_new || (v_new && rope_cos && rope_sin && rope_max_pos > 0),
             "decode_scores: k_new needs v_new and the RoPE tables");
  MI_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0 &&
                 reinterpret_cast<uintptr_t>(scratch) % 256 == 0,
             "decode_scores: workspace and scratch must be 256-byte aligned");
  const size_t need = mi_paged_decode_scores_scratch_size(batch_size, num_qo_heads, page_size,
                                                          max_pages);
  if (scratch_bytes < need)
    return fail(MI_ERR_WORKSPACE, "decode_scores: scratch of %zu bytes, %zu needed",
                scratch_bytes, need);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int group = num_qo_heads / num_kv_heads;
  float *row_lse = static_cast<float *>(scratch);  // [batch][hq]
  float *logits = reinterpret_cast<float *>(static_cast<unsigned char *>(scratch) +
                                            up256(size_t(batch_size) * num_qo_heads * 4));
  const int64_t stride = max_pages * page_size;
  auto launch_weights = [&]() -> int {
    const int64_t blocks = (stride + 255) / 256;
    const int x = static_cast<int>(std::min<int64_t>(blocks, 16 * num_sms() / num_kv_heads + 1));
    const cudaError_t e = launch_pdl(weights_kernel, dim3(x, num_kv_heads), dim3(256), 0, s,
                                     static_cast<const float *>(logits), stride,
                                     static_cast<const float *>(row_lse), kv_indptr, kv_indices,
                                     kv_last_page_len, batch_size, group, num_qo_heads, page_size,
                                     num_kv_heads, num_pages, scores);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(MI_ERR_CUDA, "weights_kernel launch: %s", cudaGetErrorString(e));
    }
    return check_launch("weights_kernel");
  };
  const bool fast = decode_fast_shape(q, q_stride_b, q_stride_h, kv_data, out, head_dim, dtype,
                                      group, batch_size);
  if (fast) {
    SkArgs sk{q, q_stride_b, q_stride_h, kv_data, num_pages, page_size, num_kv_heads,
              head_dim, dtype, kv_indptr, kv_indices, kv_last_page_len, batch_size,
              num_qo_heads, sm_scale, out, lse, workspace, workspace_bytes, status, s};
    if (k_new) {
      sk.k_new = k_new;
      sk.ksb = k_stride_b;
      sk.ksh = k_stride_h;
      sk.v_new = v_new;
      sk.vsb = v_stride_b;
      sk.vsh = v_stride_h;
      sk.rope_cos = rope_cos;
      sk.rope_sin = rope_sin;
      sk.rope_max = rope_max_pos;
      sk.rope_pos = rope_positions;
    }
    sk.logits = logits;
    sk.lse2 = row_lse;
    sk.logit_stride = stride;
    const int rc = launch_decode_sk(sk);
    if (rc > 0) return rc;
    if (rc == 0) return launch_weights();
  }
  if (k_new)
    return fail(MI_ERR_UNSUPPORTED, "decode_scores: shape outside the fused append's coverage");
  ScoreParams p{q, q_stride_b, q_stride_h, nullptr, batch_size, kv_data, num_pages, page_size,
                num_kv_heads, head_dim, kv_indptr, kv_indices, kv_last_page_len, batch_size,
                num_qo_heads, group, 0, 0, sm_scale, nullptr, scores, status};
  if (!fast) {
    const int rc = launch_generic_decode(p, dtype, logits, stride, out, lse, row_lse, s);
    return rc ? rc : launch_weights();
  }
  p.lse = lse ? lse : row_lse;
  const int rc = mi_paged_decode(q, q_stride_b, q_stride_h, kv_data, num_pages, page_size,
                                 num_kv_heads, head_dim, dtype, kv_indptr, kv_indices,
                                 kv_last_page_len, batch_size, num_qo_heads, sm_scale, out,
                                 lse ? lse : row_lse, workspace, workspace_bytes, status, stream);
  if (rc != MI_OK) return rc;
  return launch_generic(p, dtype, s);
}

extern "C" int mi_paged_prefill_scores(
    const void *q, int64_t q_stride_n, int64_t q_stride_h,
    const int32_t *qo_indptr, int32_t total_q,
    const void *kv_data, int64_t num_pages, int32_t page_size, int32_t num_kv_heads,
    int32_t head_dim, int32_t dtype,
    const int32_t *kv_indptr, const int32_t *kv_indices, const int32_t *kv_last_page_len,
    int32_t batch_size, int32_t num_qo_heads, int32_t causal, int32_t window, float sm_scale,
    const float *lse, float *scores, void *workspace, size_t workspace_bytes, int32_t *status,
    mi_stream_t stream) {
  using namespace mi;
  MI_REQUIRE(total_q >= 0 && batch_size >= 0, "prefill_scores: negative total_q/batch_size");
  if (total_q == 0 || batch_size == 0) return MI_OK;
  MI_REQUIRE(q && qo_indptr && kv_data && kv_indptr && kv_indices && kv_last_page_len && lse &&
                 scores,
             "prefill_scores: null pointer argument");
  MI_REQUIRE(page_size > 0 && num_kv_heads > 0 && head_dim > 0 && head_dim <= 256 &&
                 num_pages > 0,
             "prefill_scores: bad pool geometry");
  MI_REQUIRE(num_qo_heads >= num_kv_heads && num_qo_heads % num_kv_heads == 0,
             "prefill_scores: num_qo_heads %d is not a multiple of num_kv_heads %d",
             num_qo_heads, num_kv_heads);
  MI_REQUIRE(dtype == MI_DTYPE_F32 || dtype == MI_DTYPE_F16 || dtype == MI_DTYPE_BF16,
             "prefill_scores: bad dtype %d", dtype);
  ScoreParams p{q, q_stride_n, q_stride_h, qo_indptr, total_q, kv_data, num_pages, page_size,
                num_kv_heads, head_dim, kv_indptr, kv_indices, kv_last_page_len, batch_size,
                num_qo_heads, num_qo_heads / num_kv_heads, causal != 0, window, sm_scale, lse,
                scores, status};
  // words 2 and 3 of the prefill workspace (0 and 1 are the prefill's own)
  unsigned *ctr = nullptr;
  if (workspace && workspace_bytes >= 256 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)
    ctr = static_cast<unsigned *>(workspace) + 2;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = launch_scores_tc(p, dtype, ctr, s);
  if (rc >= 0) return rc;
  return launch_generic(p, dtype, s);
}

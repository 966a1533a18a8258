// Eviction from the paged cache by accumulated attention weight.
//
// Per (layer, request, KV head) with n > budget cached tokens: kept are the
// first `sinks` slots, the last `recent` slots and, of the middle, the
// budget - sinks - recent tokens with the largest scores (equal scores: the
// lowest slot). The reference's cache only grows; no counterpart there.
//
// Attention does not depend on the order of a cache's tokens (keys carry
// their rotation), so the kept tokens are not packed in order: those of the
// middle that already lie below budget - recent stay, the others fill, in
// order, the holes the evicted ones left, and only the `recent` last tokens
// keep their order, as the new last ones. A cache that is cut back by a page
// every page_size steps thus moves about a page and the recent window per
// head instead of the whole cache.
//
// One CTA per (layer, request, head). The scores are read once, as ordered bits
// in shared memory (those of requests with no room for them there are read again
// in each pass).
// The threshold is found by radix select, 11 bits a pass: the first digit then
// has two bits of mantissa, and a few hundred scores of like size do not all
// meet in one counter. A bit per token in shared memory with running counts
// per 32-bit word gives the i-th hole and the i-th token to move by bisection.
// Rows move a pair (K and V) per warp step, 16 bytes a lane, kRows pairs loaded
// before any is stored. HBM traffic is the scores once and the moved rows twice.
// Bound by the rows' trip through the memory system, with 8-10 us of selection
// before each CTA's first row. Measured (8 heads of 128, bf16, CUDA graph): 8
// requests of up to 4096 -> 1024 tokens, 4 layers, 55.6 us (0.55 of the copy
// rate); 32 of 1025-1040 -> 1024, 8 layers, 94 us (0.50). With the scores read
// from memory in each pass and a row pair per warp at a time 129 and 140 us;
// with two or three CTAs per SM instead of four the second takes 110 us.
#include <algorithm>

#include "mi_common.cuh"

namespace mi {
namespace {

constexpr int kEThreads = 256;
constexpr int kEWarps = kEThreads / 32;
constexpr int kRows = 8;       // row pairs a warp holds in registers while they move
constexpr int kDigit = 11;     // radix select: 11, 11 and 10 bits
constexpr int kESmemMax = 200 * 1024;
// Room for the requests' ordered scores beside their bits, 4.25 bytes a token.
// Where max_len says that all fit while four CTAs do on an SM (56 KB each, 12.1
// KB of it static: 10360 tokens), that much: 64 requests of 8192 -> 8000 take 91
// us, and 128 with the scores read again in each pass. Else (longer requests, or
// a bound that says little, as a whole page table's) what leaves four CTAs' SM
// 92 KB of L1, 6504 tokens: with 28 KB of L1 the rows' moves are slower (8 of up
// to 4096 -> 1024 by their table's bound: 58 us for 48).
constexpr int kESmemFour = 43 * 1024;
constexpr int kESmemSome = 27 * 1024;

struct EvictParams {
  void *const *layer_kv;  // pointer per layer, or null: kv + layer * kv_stride bytes
  unsigned char *kv;
  int64_t kv_stride;
  float *scores;  // + layer * score_stride elements
  int64_t score_stride;
  int64_t num_pages;
  int ps, hkv, row_bytes;  // row: one head of one token of K (or V)
  const int32_t *indptr, *indices, *last;
  int batch, budget, recent, sinks, max_len, smem;
  int32_t *kept;
  int32_t *status;
};

// Scores in order as unsigned integers; NaN lowest, -0 equal to 0.
__device__ __forceinline__ uint32_t score_key(float x) {
  uint32_t b = __float_as_uint(x);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Position of the n-th (from 0) set bit of w, which has more than n.
__device__ __forceinline__ int nth_bit(uint32_t w, int n) {
  int at = 0;
#pragma unroll
  for (int half = 16; half > 0; half >>= 1) {
    const int c = __popc((w >> at) & ((1u << half) - 1u));
    if (n >= c) {
      n -= c;
      at += half;
    }
  }
  return at;
}

struct RowPair {
  const unsigned char *src;  // K rows of two slots
  unsigned char *dst;
};

// V: what a lane copies at once (16 bytes where rows and pointers allow).
template <typename V>
// four CTAs per SM (64 registers): most of a CTA's time is latency
__global__ void __launch_bounds__(kEThreads, 4) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t s_dyn[];
  __shared__ uint32_t s_hist[1 << kDigit];
  __shared__ int s_warp[kEWarps];
  __shared__ uint32_t s_digit, s_need, s_in;
  __shared__ int s_bad;
  __shared__ RowPair s_pair[kEWarps][32];
  const int b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv, layer = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = kv_len_of(p.indptr, p.last, b, p.ps);
  const int npages = p.indptr[b + 1] - p.indptr[b];
  const int32_t *table = p.indices + p.indptr[b];
  float *scores = p.scores + layer * p.score_stride + static_cast<int64_t>(h) * p.ps;
  int32_t *kept = p.kept ? p.kept + (static_cast<int64_t>(layer) * gridDim.x + blockIdx.x) * p.budget
                         : nullptr;
  if (n <= p.budget) {
    if (kept)
      for (int j = tid; j < p.budget; j += kEThreads) kept[j] = j < n ? j : -1;
    return;
  }
  // nothing of a request with a bad page, or longer than the bit map, is touched
  if (tid == 0) s_bad = n > p.max_len ? MI_STATUS_BAD_POSITION : 0;
  __syncthreads();
  for (int i = tid; i < npages; i += kEThreads)
    if (table[i] < 0 || table[i] >= p.num_pages) s_bad = MI_STATUS_BAD_PAGE;
  __syncthreads();
  if (s_bad) {
    if (tid == 0) flag(p.status, s_bad);
    if (kept)
      for (int j = tid; j < p.budget; j += kEThreads) kept[j] = -1;
    return;
  }
  const int64_t spage = static_cast<int64_t>(p.hkv) * p.ps;  // scores of a page
  auto score_at = [&](int t) -> float * { return scores + table[t / p.ps] * spage + t % p.ps; };

  const int recent = min(p.recent, p.budget), sinks = min(p.sinks, p.budget - recent);
  const int low = p.budget - recent, mid_end = n - recent;
  const int want = low - sinks;  // of the middle tokens [sinks, mid_end)

  unsigned char *kv = p.layer_kv ? static_cast<unsigned char *>(p.layer_kv[layer])
                                 : p.kv + layer * p.kv_stride;
  const int64_t slot_bytes = static_cast<int64_t>(p.hkv) * p.row_bytes;
  auto k_row = [&](int t) -> unsigned char * {
    return kv + (static_cast<int64_t>(table[t / p.ps]) * 2 * p.ps + t % p.ps) * slot_bytes +
           static_cast<int64_t>(h) * p.row_bytes;
  };
  const int64_t v_off = p.ps * slot_bytes;  // from a K row to its V row
  const int vec = p.row_bytes / static_cast<int>(sizeof(V));  // vectors of a row

  const int words = (n + 31) / 32;
  uint32_t *bits = s_dyn, *before = s_dyn + words;  // kept tokens in earlier words
  uint32_t *keys = before + words;
  const bool held = (2 * words + n) * 4 <= p.smem;  // (else: read again in each pass)
  auto key_of = [&](int t) { return held ? keys[t] : score_key(*score_at(t)); };
  if (held && want > 0) {
    for (int t = sinks + tid; t < mid_end; t += kEThreads) keys[t] = score_key(*score_at(t));
  }
  // ---- threshold: key of the want-th largest score, and how many ties to keep
  // (need < in: of `in` tokens with that key; else all with key >= cut are kept)
  uint32_t cut = 0, need = want, in = 0;
  int left = 32;  // bits not looked at yet
  while (want > 0 && left > 0 && need != in) {
    const int width = min(kDigit, left), shift = left - width;
    for (int i = tid; i < (1 << kDigit); i += kEThreads) s_hist[i] = 0;
    __syncthreads();
    for (int t = sinks + tid; t < mid_end; t += kEThreads) {
      const uint32_t k = key_of(t);
      if (left == 32 || (k >> left) == (cut >> left))
        atomicAdd(&s_hist[(k >> shift) & ((1u << width) - 1u)], 1u);
    }
    __syncthreads();
    // from the largest digit down, 8 a thread
    constexpr int kPer = (1 << kDigit) / kEThreads;
    const int top = (1 << kDigit) - 1 - tid * kPer;
    uint32_t c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += c[i] = s_hist[top - i];
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    for (int i = 0; i < warp; ++i) incl += s_warp[i];
    uint32_t first = incl - sum;
    if (first < need && need <= incl) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (first < need && need <= first + c[i]) {
          s_digit = top - i;
          s_need = need - first;
          s_in = c[i];
        }
        first += c[i];
      }
    }
    __syncthreads();
    cut |= s_digit << shift;
    need = s_need;
    in = s_in;
    left = shift;
    __syncthreads();
  }
  // ---- a bit per token: kept --------------------------------------------------
  const int per_warp = (words + kEWarps - 1) / kEWarps;
  const int w0 = min(words, warp * per_warp), w1 = min(words, w0 + per_warp);
  // ties with the threshold, where some are left out: their number per warp
  // segment, so that each segment knows its first's rank
  uint32_t rank = 0;
  const bool some = want > 0 && need < in;
  if (some) {
    int ties = 0;
    for (int w = w0; w < w1; ++w) {
      const int t = w * 32 + lane;
      const bool tie = t >= sinks && t < mid_end && key_of(t) == cut;
      ties += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) s_warp[warp] = ties;
    __syncthreads();
    for (int i = 0; i < warp; ++i) rank += s_warp[i];
    __syncthreads();
  }
  int count = 0;
  for (int w = w0; w < w1; ++w) {
    const int t = w * 32 + lane;
    const bool mid = t >= sinks && t < mid_end;
    const uint32_t k = mid && want > 0 ? key_of(t) : 0;
    bool keep = mid ? want > 0 && k >= cut : t < n;
    if (some) {
      const bool tie = mid && k == cut;
      const uint32_t tm = __ballot_sync(0xffffffffu, tie);
      if (tie) keep = rank + __popc(tm & ((1u << lane) - 1u)) < need;
      rank += __popc(tm);
    }
    const uint32_t m = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) {
      bits[w] = m;
      before[w] = count;
    }
    count += __popc(m);
  }
  if (lane == 0) s_warp[warp] = count;
  __syncthreads();
  {
    int add = 0;
    for (int i = 0; i < warp; ++i) add += s_warp[i];
    for (int w = w0 + lane; w < w1; w += 32) before[w] += add;
  }
  __syncthreads();
  auto kept_before = [&](int t) -> int {  // t <= n
    const int w = t >> 5;
    return w < words ? static_cast<int>(before[w]) + __popc(bits[w] & ((1u << (t & 31)) - 1u))
                     : p.budget;
  };
  const int moves = want - (kept_before(low) - sinks);  // holes below low = tokens to move there

  // ---- holes: the i-th takes the i-th kept token at or past `low` -------------
  for (int i0 = warp * 32; i0 < moves; i0 += kEWarps * 32) {
    const int i = i0 + lane;
    int dst = 0, src = 0;
    if (i < moves) {
      // the i-th slot not kept: the last word with fewer than i + 1 zeros before it
      int l = 0, r = words - 1;
      while (l < r) {
        const int m = (l + r + 1) >> 1;
        if (m * 32 - static_cast<int>(before[m]) <= i) l = m; else r = m - 1;
      }
      dst = l * 32 + nth_bit(~bits[l], i - (l * 32 - static_cast<int>(before[l])));
      const int q = kept_before(low) + i;  // the q-th kept token overall
      l = 0, r = words - 1;
      while (l < r) {
        const int m = (l + r + 1) >> 1;
        if (static_cast<int>(before[m]) <= q) l = m; else r = m - 1;
      }
      src = l * 32 + nth_bit(bits[l], q - static_cast<int>(before[l]));
      *score_at(dst) = *score_at(src);
      if (kept) kept[dst] = src;
      s_pair[warp][lane] = RowPair{k_row(src), k_row(dst)};
    }
    __syncwarp();
    const int cnt = min(32, moves - i0);
    for (int j = 0; j < cnt; j += kRows) {
      for (int e = lane; e < 2 * vec; e += 32) {
        const int64_t off = (e < vec ? 0 : v_off) +
                            static_cast<int64_t>(e < vec ? e : e - vec) * sizeof(V);
        V hold[kRows];
        // (row addresses come from each lane's own pair)
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (j + u < cnt) hold[u] = *reinterpret_cast<const V *>(s_pair[warp][j + u].src + off);
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (j + u < cnt) *reinterpret_cast<V *>(s_pair[warp][j + u].dst + off) = hold[u];
      }
    }
    __syncwarp();
  }
  if (kept)
    for (int j = tid; j < low; j += kEThreads)
      if ((bits[j >> 5] >> (j & 31)) & 1u) kept[j] = j;
  // ---- the recent window moves down by n - budget, lowest first ---------------
  // A slot may be written once it has been read, as the source of an earlier
  // one (or of a row above): rows go in chunks, a barrier between a chunk's
  // loads and its stores; the next chunk's loads follow its stores at once.
  const int by = n - p.budget;
  constexpr int kChunk = kEWarps * kRows;
  for (int c0 = 0; c0 < recent; c0 += kEWarps * 32) {
    {
      const int r = c0 + lane * kEWarps + warp;
      if (r < recent) s_pair[warp][lane] = RowPair{k_row(low + r + by), k_row(low + r)};
    }
    __syncwarp();
    // rows of this warp in this block of 256
    const int mine = max(0, min(32, (recent - c0 - warp + kEWarps - 1) / kEWarps));
    const int chunks = (min(recent - c0, kEWarps * 32) + kChunk - 1) / kChunk;
    for (int e0 = 0; e0 < 2 * vec; e0 += 32) {  // a row pair wider than a warp: in parts
      const int e = e0 + lane;
      const bool on = e < 2 * vec;
      const int64_t off = (e < vec ? 0 : v_off) +
                          static_cast<int64_t>(e < vec ? e : e - vec) * sizeof(V);
      V hold[kRows];
      auto load = [&](int c) {
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (on && c * kRows + u < mine)
            hold[u] = *reinterpret_cast<const V *>(s_pair[warp][c * kRows + u].src + off);
      };
      __syncthreads();  // (moves above, or the part or block before, have read)
      load(0);
      for (int c = 0; c < chunks; ++c) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (on && c * kRows + u < mine)
            *reinterpret_cast<V *>(s_pair[warp][c * kRows + u].dst + off) = hold[u];
        if (c + 1 < chunks) load(c + 1);
      }
    }
    __syncwarp();
  }
  for (int c0 = 0; c0 < recent; c0 += kEThreads) {
    const int r = c0 + tid;
    float sv = 0.f;
    if (r < recent) sv = *score_at(low + r + by);
    __syncthreads();
    if (r < recent) {
      *score_at(low + r) = sv;
      if (kept) kept[low + r] = low + r + by;
    }
  }
  __syncthreads();
  // ---- slots behind the kept ones have no score --------------------------------
  for (int t = p.budget + tid; t < npages * p.ps; t += kEThreads) *score_at(t) = 0.f;
}

template <typename V>
int launch_evict(const EvictParams &p, int layers, cudaStream_t s) {
  static std::atomic<unsigned long long> attr_set{0};
  if (smem_limit_once(attr_set, evict_kernel<V>, kESmemMax) != cudaSuccess)
    return check_launch("evict_kernel smem attribute");
  evict_kernel<V><<<dim3(p.batch * p.hkv, layers), kEThreads, p.smem, s>>>(p);
  return check_launch("evict_kernel");
}

}  // namespace
}  // namespace mi

extern "C" int mi_kv_evict(void *const *layer_pools, void *kv_data, int64_t kv_layer_stride,
                           float *scores, int32_t num_layers, int64_t num_pages,
                           int32_t page_size, int32_t num_kv_heads, int32_t head_dim,
                           int32_t dtype, const int32_t *kv_indptr, const int32_t *kv_indices,
                           const int32_t *kv_last_page_len, int32_t batch_size, int32_t max_len,
                           int32_t budget, int32_t recent, int32_t sinks, int32_t *kept,
                           int32_t *status, mi_stream_t stream) {
  using namespace mi;
  MI_REQUIRE(num_layers >= 0 && batch_size >= 0, "kv_evict: negative num_layers/batch_size");
  if (num_layers == 0 || batch_size == 0) return MI_OK;
  MI_REQUIRE((layer_pools || kv_data) && scores && kv_indptr && kv_indices && kv_last_page_len,
             "kv_evict: null pointer argument");
  MI_REQUIRE(num_pages > 0 && page_size > 0 && num_kv_heads > 0 && head_dim > 0,
             "kv_evict: bad pool geometry");
  MI_REQUIRE(dtype == MI_DTYPE_F32 || dtype == MI_DTYPE_F16 || dtype == MI_DTYPE_BF16,
             "kv_evict: bad dtype %d", dtype);
  MI_REQUIRE(budget > 0 && recent >= 0 && sinks >= 0 &&
                 static_cast<int64_t>(recent) + sinks <= budget,
             "kv_evict: budget %d below recent %d + sinks %d (or not positive)", budget, recent,
             sinks);
  MI_REQUIRE(max_len > 0, "kv_evict: max_len %d", max_len);
  MI_REQUIRE(num_layers <= 65535 &&
                 static_cast<int64_t>(batch_size) * num_kv_heads < (int64_t(1) << 31),
             "kv_evict: too many layers or heads");
  const int es = elt_size(dtype);
  const int64_t row = static_cast<int64_t>(head_dim) * es;
  MI_REQUIRE(row <= (1 << 20), "kv_evict: head_dim %d", head_dim);
  // the bit map and its counts: 8 bytes per 32 tokens
  const int64_t cap = static_cast<int64_t>(kESmemMax) / 8 * 32;
  EvictParams p{layer_pools, static_cast<unsigned char *>(kv_data), kv_layer_stride * es, scores,
                num_pages * num_kv_heads * page_size, num_pages, page_size, num_kv_heads,
                static_cast<int>(row), kv_indptr, kv_indices, kv_last_page_len, batch_size, budget,
                recent, sinks, static_cast<int>(std::min<int64_t>(max_len, cap)), 0, kept, status};
  const int map = (p.max_len + 31) / 32 * 8;  // the longest request's
  const int64_t full = map + int64_t(p.max_len) * 4;
  p.smem = full <= kESmemFour ? static_cast<int>(full) : std::max(map, kESmemSome);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // torch's pools are 256-byte aligned; a caller's own need only be aligned to
  // the element, and then the copies are narrower. (With layer_pools the
  // pointers are on the device: mi_page_release already asks 16 bytes of them.)
  const bool wide = row % 16 == 0 && (layer_pools || (reinterpret_cast<uintptr_t>(kv_data) % 16 == 0 &&
                                                      p.kv_stride % 16 == 0));
  if (wide) return launch_evict<uint4>(p, num_layers, s);
  if (es == 4) return launch_evict<uint32_t>(p, num_layers, s);
  return launch_evict<uint16_t>(p, num_layers, s);
}

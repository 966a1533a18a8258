// Token sampling from logits: temperature, top-k, top-p (nucleus), min-p,
// drawn with one given random number per row.
//
// Row x[0..V): d_i = x_i - max x (0 at the max), w_i = exp(d_i / T). Tokens are
// ordered by (x descending, index ascending). Kept are, in turn, the first k of
// the order, of those the shortest prefix holding at least p of their mass, and
// of those the ones with w_i >= m (the largest w is 1). The token drawn is the
// first kept one, by index, whose running mass exceeds u times the kept mass.
//
// All three filters keep a prefix of one total order, so a filter is a single
// threshold on the composite (ordered key of x, ~index): what follows finds
// that threshold without sorting the row. Weights are 45-bit fixed point (2^44
// = the largest), computed in 64-bit floating point from the logit alone, and
// summed as integers: sums are exact and the same in any order, so the result
// does not depend on how the row is split or on the order of atomics, and a
// near-flat row of 150,000 tokens still has 2^-44 of resolution per token.
//
// One thread-block cluster per row (1 to 8 CTAs); each CTA keeps its slice of
// the row in shared memory as ordered keys, read from HBM once. The passes
// exchange through distributed shared memory:
//   1. the largest composite (which is the greedy answer);
//   2. a 256-bin histogram of counts and masses over -log2 w in steps of 1/8
//      (linear in x: bins of the key's own bits would hold most of a row in a
//      few bins): the bin where the filter's prefix ends;
//   3. if no more than kCap tokens lie at or above that bin (the usual case),
//      they are gathered, sorted in registers, and every filter and the draw
//      happen on that list; else the range of composites the threshold lies in
//      is divided by 256 until kCap tokens are left in it, and the draw is one
//      more pass over the row: mass per warp, then the warp that holds u's
//      place scans its tokens.
#include <cooperative_groups.h>

#include <algorithm>

#include "mi_common.cuh"

namespace cg = cooperative_groups;

namespace mi {
namespace {

constexpr int kSThreads = 512;
constexpr int kSWarps = kSThreads / 32;
constexpr int kBins = 256;
constexpr int kCap = 512;        // tokens resolved by sorting (one per thread)
constexpr int kMaxCluster = 8;   // portable cluster size
constexpr int kIdxBits = 18;     // vocabulary <= 2^18
constexpr uint32_t kIdxMask = (1u << kIdxBits) - 1;
constexpr int kWeightBits = 44;  // the largest weight is 2^44
constexpr int kLimb = 15;        // histogram masses: three 15-bit limbs in 32-bit counters
constexpr int kMaxSlice = (1 << 17) - 1;  // limb sums: 2^17 tokens * 2^15 stay below 2^32

using u64 = unsigned long long;

struct SampleParams {
  const void *logits;
  int64_t row_stride;
  int rows, vocab, slice;  // slice: tokens per CTA (a multiple of 8)
  const float *uniform;
  const float *temperature, *top_p, *min_p;  // per row, or null: the scalar
  const int32_t *top_k;
  float temperature_s, top_p_s, min_p_s;
  int32_t top_k_s;
  int32_t *out;
  float *logprob;
  int32_t *status;
};

// Ordered keys: larger logit <=> larger key; NaN is key 0, -0 equals +0. Keys
// up to kNone (that of -inf) are never chosen.
template <typename T> struct KeyOf;
template <> struct KeyOf<__nv_bfloat16> {
  using K = uint16_t;
  static constexpr uint32_t kNone = 0x007F;
  __device__ static K key(uint16_t b) {
    if ((b & 0x7FFF) > 0x7F80) return 0;
    if (b == 0x8000) b = 0;
    return (b & 0x8000) ? static_cast<K>(~b) : static_cast<K>(b | 0x8000);
  }
  __device__ static float value(uint32_t k) {
    const uint32_t b = (k & 0x8000) ? (k & 0x7FFF) : (~k & 0xFFFF);
    return __uint_as_float(b << 16);
  }
};
template <> struct KeyOf<__half> {
  using K = uint16_t;
  static constexpr uint32_t kNone = 0x03FF;
  __device__ static K key(uint16_t b) {
    if ((b & 0x7FFF) > 0x7C00) return 0;
    if (b == 0x8000) b = 0;
    return (b & 0x8000) ? static_cast<K>(~b) : static_cast<K>(b | 0x8000);
  }
  __device__ static float value(uint32_t k) {
    const uint32_t b = (k & 0x8000) ? (k & 0x7FFF) : (~k & 0xFFFF);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(b)));
  }
};
template <> struct KeyOf<float> {
  using K = uint32_t;
  static constexpr uint32_t kNone = 0x007FFFFF;
  __device__ static K key(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;
    if (b == 0x80000000u) b = 0;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  __device__ static float value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
};

// (key, ~index): a total order of the row's tokens, largest first
__device__ __forceinline__ u64 composite(uint32_t key, uint32_t idx) {
  return (static_cast<u64>(key) << kIdxBits) | (kIdxMask - idx);
}
__device__ __forceinline__ uint32_t comp_key(u64 c) { return static_cast<uint32_t>(c >> kIdxBits); }
__device__ __forceinline__ uint32_t comp_idx(u64 c) {
  return kIdxMask - (static_cast<uint32_t>(c) & kIdxMask);
}

// A row's weights: functions of the key alone, the same in every pass.
struct RowW {
  double xmax, inv_t;
  float fmax, fscale;  // bins: 8 log2(e) / T

  __device__ double weight_f(float x) const {
    if (x == fmax) return 1.0;  // (also +inf among +inf)
    const double d = static_cast<double>(x) - xmax;
    return d == -INFINITY ? 0.0 : exp(d * inv_t);
  }
  __device__ u64 weight(float x) const {
    return __double2ull_rn(weight_f(x) * static_cast<double>(1ull << kWeightBits));
  }
  // monotone in x: each of the subtraction, product and truncation is
  __device__ int bin(float x) const {
    if (x == fmax) return 0;
    const float t = (fmax - x) * fscale;
    return t >= kBins - 1 ? kBins - 1 : static_cast<int>(t);
  }
};

struct __align__(16) Bin {
  uint32_t n, l0, l1, l2;  // count; mass limbs
};

struct Shared {
  Bin hist[2][kBins];
  u64 list[kCap];   // this CTA's gathered composites
  u64 sorted[kCap];
  u64 scan[kSWarps];
  u64 wsum[kSWarps];
  // read by the other CTAs of the cluster, each written once before a barrier
  u64 maxc;
  double lsum;
  u64 mass;
  uint32_t list_n[2];
  // block-wide results
  u64 r_u64[4];
  uint32_t r_u32[4];
  int token;
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
  return __shfl_up_sync(0xffffffffu, v, o);
}

// Inclusive block scan of one 64-bit integer per thread.
__device__ u64 block_scan(u64 v, u64 *s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = shfl_up64(v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // (s may still be read from an earlier call)
  if (lane == 31) s[warp] = v;
  __syncthreads();
  u64 before = 0;
#pragma unroll
  for (int i = 0; i < kSWarps; ++i)
    if (i < warp) before += s[i];
  return v + before;
}

// Sorts one 64-bit value per thread, descending over threadIdx.
__device__ u64 block_sort_desc(u64 v, u64 *buf) {
  const int t = threadIdx.x;
#pragma unroll 1
  for (int k = 2; k <= kSThreads; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64 o;
      if (j >= 32) {
        __syncthreads();
        buf[t] = v;
        __syncthreads();
        o = buf[t ^ j];
      } else {
        o = __shfl_xor_sync(0xffffffffu, v, j);
      }
      const bool keep_max = ((t & j) == 0) == ((t & k) == 0);
      v = keep_max ? (v > o ? v : o) : (v < o ? v : o);
    }
  }
  __syncthreads();
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kSThreads) sample_kernel(const SampleParams p) {
  using KO = KeyOf<T>;
  using K = typename KO::K;
  constexpr int VEC = 16 / sizeof(K);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared &sh = *reinterpret_cast<Shared *>(smem_raw);
  K *keys = reinterpret_cast<K *>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int nrank = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / nrank;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const int base = rank * p.slice;  // first token of this CTA's slice
  const int n = max(0, min(p.vocab - base, p.slice));
  const T *src = static_cast<const T *>(p.logits) + static_cast<int64_t>(row) * p.row_stride + base;
  // tokens before the first 16-byte boundary; keys[] is shifted so that vectors
  // of the row land on vectors of shared memory
  const int head = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T));
  const int pad = (VEC - head) & (VEC - 1);
  const int nvec = (pad + n + VEC - 1) / VEC;
  const int per_warp = (nvec + kSWarps - 1) / kSWarps;  // a warp's vectors are consecutive
  const int v0 = min(nvec, warp * per_warp), v1 = min(nvec, v0 + per_warp);

  for (int i = tid; i < 2 * kBins; i += kSThreads) sh.hist[0][i] = Bin{0, 0, 0, 0};
  if (tid < 2) sh.list_n[tid] = 0;
  if (tid == 0) sh.token = -1;

  // ---- 1. the slice into shared memory; its largest composite --------------
  u64 best = 0;
  for (int v = v0 + lane; v < v1; v += 32) {
    const int i0 = v * VEC - pad;  // first token of the vector
    K k[VEC];
    if (i0 >= 0 && i0 + VEC <= n) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(src + i0);
      const K *e = reinterpret_cast<const K *>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) k[j] = KO::key(e[j]);
    } else {
      const K *bits = reinterpret_cast<const K *>(src);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        k[j] = (i0 + j >= 0 && i0 + j < n) ? KO::key(bits[i0 + j]) : K(0);
    }
    uint32_t kb = k[0];
    int jb = 0;
#pragma unroll
    for (int j = 1; j < VEC; ++j)
      if (k[j] > kb) kb = k[j], jb = j;
    const u64 c = composite(kb, base + i0 + jb);
    if (kb > KO::kNone && c > best) best = c;
    *reinterpret_cast<uint4 *>(keys + v * VEC) = *reinterpret_cast<const uint4 *>(k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(0xffffffffu, best, o);
    best = y > best ? y : best;
  }
  if (lane == 0) sh.wsum[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSWarps; ++i) best = sh.wsum[i] > best ? sh.wsum[i] : best;
    sh.maxc = best;
  }
  cluster.sync();
  u64 gmax = 0;
  for (int r = 0; r < nrank; ++r) {
    const u64 c = *cluster.map_shared_rank(&sh.maxc, r);
    gmax = c > gmax ? c : gmax;
  }

  const float temp = p.temperature ? p.temperature[row] : p.temperature_s;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k_s;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_s;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p_s;
  float u = p.uniform[row];
  u = u > 0.f ? fminf(u, 1.f - 5.9604645e-8f) : 0.f;  // [0, 1); NaN: 0
  const bool greedy = !(temp > 0.f);
  const bool use_k = !greedy && top_k > 0 && top_k < p.vocab;
  const bool use_p = !greedy && top_p < 1.f;
  const double minw = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
  RowW rw;
  rw.fmax = KO::value(comp_key(gmax));
  rw.xmax = rw.fmax;
  rw.inv_t = greedy ? 1.0 : 1.0 / static_cast<double>(temp);
  rw.fscale = static_cast<float>(8.0 * 1.4426950408889634 * rw.inv_t);

  // visits this thread's tokens (vectors of its warp in order): f(key, token)
  auto each = [&](auto &&f) {
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
      const K *e = reinterpret_cast<const K *>(&raw);
      const int i0 = base + v * VEC - pad;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e[j] > KO::kNone) f(static_cast<uint32_t>(e[j]), static_cast<uint32_t>(i0 + j));
    }
  };

  // log-sum-exp of the row at temperature 1, for the log-probability
  if (p.logprob && gmax != 0) {
    float s = 0.f;
    each([&](uint32_t k, uint32_t) {
      const float x = KO::value(k);
      s += x == rw.fmax ? 1.f : exp2f((x - rw.fmax) * kLog2e);
    });
    double d = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    double *part = reinterpret_cast<double *>(sh.scan);
    if (lane == 0) part[warp] = d;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kSWarps; ++i) d += part[i];
      sh.lsum = d;
    }
    __syncthreads();
  }

  u64 thr = 0;        // tokens with a composite >= thr are kept
  bool done = false;  // resolved on a list (by every CTA alike)
  int sel = 0;        // threshold searches done (list_n buffer)
  int level = 0;      // histogram levels done (hist buffer)

  // Sums this level's histogram over the cluster and finds the first bin whose
  // running sum reaches the target: results in r_u32 = {bin, count above, count
  // in it}, r_u64 = {mass above, total mass, total count}. target < 0: the mass
  // target is frac * total mass.
  auto merge = [&](bool by_mass, double target, double frac, u64 have) {
    cluster.sync();
    Bin b{0, 0, 0, 0};
    u64 m = 0, c = 0;
    if (tid < kBins) {
      for (int r = 0; r < nrank; ++r) {
        b = *cluster.map_shared_rank(&sh.hist[level & 1][tid], r);
        c += b.n;
        m += static_cast<u64>(b.l0) + (static_cast<u64>(b.l1) << kLimb) +
             (static_cast<u64>(b.l2) << (2 * kLimb));
      }
    }
    const u64 cs = block_scan(c, sh.scan);
    const u64 ms = by_mass ? block_scan(m, sh.scan) : 0;
    if (tid == kSThreads - 1) {
      sh.r_u64[1] = ms;
      sh.r_u64[2] = cs;
    }
    if (tid == 0) sh.r_u32[0] = kBins;
    __syncthreads();
    if (by_mass && target < 0) target = frac * static_cast<double>(sh.r_u64[1]);
    // the first bin that reaches the target; a prefix of at least one token
    const double at = by_mass ? static_cast<double>(have + ms) : static_cast<double>(have + cs);
    const double was = by_mass ? static_cast<double>(have + ms - m)
                               : static_cast<double>(have + cs - c);
    if (tid < kBins && c > 0 && at >= target && (was < target || cs == c)) {
      sh.r_u32[0] = tid;
      sh.r_u32[1] = static_cast<uint32_t>(cs - c);
      sh.r_u32[2] = static_cast<uint32_t>(c);
      sh.r_u64[0] = ms - m;
    }
    __syncthreads();
    ++level;
    // the next level's buffer: every CTA has read it before this barrier
    if (tid < kBins) sh.hist[level & 1][tid] = Bin{0, 0, 0, 0};
    __syncthreads();
    return target;
  };
  auto add = [&](int b, bool by_mass, u64 w) {
    Bin *h = &sh.hist[level & 1][b];
    atomicAdd(&h->n, 1u);
    if (by_mass && w) {
      constexpr uint32_t mask = (1u << kLimb) - 1;
      if (const uint32_t l = static_cast<uint32_t>(w) & mask) atomicAdd(&h->l0, l);
      if (const uint32_t l = static_cast<uint32_t>(w >> kLimb) & mask) atomicAdd(&h->l1, l);
      if (const uint32_t l = static_cast<uint32_t>(w >> (2 * kLimb))) atomicAdd(&h->l2, l);
    }
  };
  // Gathers the tokens f accepts (at most kCap over the cluster), sorts them:
  // this thread's composite in descending order (0: none).
  auto gather = [&](auto &&f) {
    uint32_t *cnt = &sh.list_n[sel & 1];
    each([&](uint32_t k, uint32_t i) {
      const u64 c = composite(k, i);
      if (f(k, c)) {
        const uint32_t at = atomicAdd(cnt, 1u);
        if (at < kCap) sh.list[at] = c;
      }
    });
    cluster.sync();
    u64 mine = 0;
    uint32_t off = 0;
    for (int r = 0; r < nrank; ++r) {
      const uint32_t m = min(*cluster.map_shared_rank(cnt, r), static_cast<uint32_t>(kCap));
      if (tid >= off && tid < off + m) mine = *cluster.map_shared_rank(&sh.list[tid - off], r);
      off += m;
    }
    ++sel;
    return block_sort_desc(mine, sh.sorted);
  };
  auto weight_of = [&](u64 c) { return c ? rw.weight(KO::value(comp_key(c))) : 0ull; };

  // ---- 2., 3. the filters' thresholds ---------------------------------------
  const int nsel = (use_k ? 1 : 0) + (use_p ? 1 : 0);
  for (int s = 0; s < nsel && gmax != 0 && !done; ++s) {
    const bool by_mass = !(use_k && s == 0);
    each([&](uint32_t k, uint32_t i) {
      if (composite(k, i) < thr) return;
      const float x = KO::value(k);
      add(rw.bin(x), by_mass, by_mass ? rw.weight(x) : 0);
    });
    double target = merge(by_mass, by_mass ? -1.0 : static_cast<double>(top_k), top_p, 0);
    const uint32_t b = sh.r_u32[0];
    if (b == kBins) continue;  // fewer than k tokens: all are kept
    uint32_t above = sh.r_u32[1], inside = sh.r_u32[2];
    u64 above_m = sh.r_u64[0];
    __syncthreads();
    if (above + inside <= kCap) {
      // everything that may be kept fits the list
      const u64 c = gather([&](uint32_t k, u64 c) {
        return c >= thr && rw.bin(KO::value(k)) <= static_cast<int>(b);
      });
      u64 w = weight_of(c);
      bool keep = c != 0;
      if (!by_mass) keep = keep && tid < top_k;
      if (use_p) {
        const u64 upto = block_scan(keep ? w : 0, sh.scan);
        if (tid == kSThreads - 1) sh.r_u64[3] = upto;
        __syncthreads();
        // (mass search: the target is a share of all the row's mass)
        const double want = by_mass ? target : top_p * static_cast<double>(sh.r_u64[3]);
        keep = keep && (tid == 0 || static_cast<double>(upto - w) < want);
      }
      if (minw > 0.0) keep = keep && rw.weight_f(KO::value(comp_key(c))) >= minw;
      // by index, weight in the low bits (18 + 45 bits); ~: ascending
      const u64 packed =
          keep ? ~((static_cast<u64>(comp_idx(c)) << (kWeightBits + 1)) | w) : 0ull;
      const u64 sorted = block_sort_desc(packed, sh.sorted);
      w = sorted ? (~sorted & ((1ull << (kWeightBits + 1)) - 1)) : 0;
      const u64 cum = block_scan(w, sh.scan);
      if (tid == kSThreads - 1) sh.r_u64[3] = cum;
      __syncthreads();
      const u64 at = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sh.r_u64[3]));
      if (w && cum > at && cum - w <= at)
        sh.token = static_cast<int>((~sorted >> (kWeightBits + 1)) & kIdxMask);
      __syncthreads();
      done = true;
      break;
    }
    // the range of composites that bin b holds: its keys by a 32-way search
    // (bin() falls as the key grows), the same in every warp
    u64 lo, hi;
    {
      auto edge = [&](int limit) {  // smallest key above kNone with bin <= limit
        uint32_t l = KO::kNone + 1, h = comp_key(gmax);  // the answer is in [l, h]
        while (l < h) {
          const uint32_t step = (h - l + 31) / 32;
          const u64 at = static_cast<u64>(l) + static_cast<u64>(step) * lane;
          const bool in = at >= h || rw.bin(KO::value(static_cast<uint32_t>(at))) <= limit;
          const uint32_t m = __ballot_sync(0xffffffffu, in);
          const int first = m ? __ffs(m) - 1 : 32;
          const u64 nl = first ? static_cast<u64>(l) + static_cast<u64>(step) * (first - 1) + 1 : l;
          const u64 nh = first < 32 ? min(static_cast<u64>(h), static_cast<u64>(l) +
                                                                   static_cast<u64>(step) * first)
                                    : h;
          l = static_cast<uint32_t>(nl);
          h = static_cast<uint32_t>(nh);
        }
        return l;
      };
      const uint32_t klo = edge(static_cast<int>(b));
      const uint32_t khi = b == 0 ? comp_key(gmax) : edge(static_cast<int>(b) - 1) - 1;
      lo = static_cast<u64>(klo) << kIdxBits;
      hi = (static_cast<u64>(khi) << kIdxBits) | kIdxMask;
      if (lo < thr) lo = thr;
    }
    // divide the range until its tokens fit the list
    while (inside > kCap) {
      const int shift = max(0, 64 - __clzll(static_cast<long long>(hi - lo)) - 8);
      each([&](uint32_t k, uint32_t i) {
        const u64 c = composite(k, i);
        if (c >= lo && c <= hi)
          add(static_cast<int>((hi - c) >> shift), by_mass, by_mass ? rw.weight(KO::value(k)) : 0);
      });
      merge(by_mass, target, 0.0, by_mass ? above_m : above);
      const uint32_t q = sh.r_u32[0];
      above += sh.r_u32[1];
      inside = sh.r_u32[2];
      above_m += sh.r_u64[0];
      __syncthreads();
      hi -= static_cast<u64>(q) << shift;
      const u64 width = (1ull << shift) - 1;
      if (hi - lo > width) lo = hi - width;
    }
    const u64 c = gather([&](uint32_t, u64 c) { return c >= lo && c <= hi; });
    u64 w = by_mass ? weight_of(c) : (c ? 1 : 0);
    const u64 upto = (by_mass ? above_m : above) + block_scan(w, sh.scan);
    // the last kept: the first whose running sum reaches the target
    if (c && static_cast<double>(upto) >= target &&
        (tid == 0 || static_cast<double>(upto - w) < target))
      sh.r_u64[3] = c;
    __syncthreads();
    thr = sh.r_u64[3];
    __syncthreads();
  }

  // ---- 4. the draw ------------------------------------------------------------
  auto finish = [&](uint32_t key, int token) {  // one thread of the cluster
    p.out[row] = token;
    if (p.logprob) {
      double s = 0;
      for (int r = 0; r < nrank; ++r) s += *cluster.map_shared_rank(&sh.lsum, r);
      const float x = KO::value(key);
      const double d = x == rw.fmax ? 0.0 : static_cast<double>(x) - rw.xmax;
      p.logprob[row] = static_cast<float>(d - log(s));
    }
  };
  if (gmax == 0) {  // no finite or +inf logit
    if (rank == 0 && tid == 0) {
      p.out[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
      flag(p.status, MI_STATUS_NO_TOKEN);
    }
  } else if (greedy) {
    if (p.logprob) cluster.sync();  // every CTA's lsum is written
    if (rank == 0 && tid == 0) finish(comp_key(gmax), static_cast<int>(comp_idx(gmax)));
  } else if (done) {
    // the CTA that holds the token has its key
    const int t = sh.token;
    if (tid == 0 && t >= base && t < base + n) finish(keys[t - base + pad], t);
  } else {
    auto kept = [&](uint32_t k, uint32_t i) {
      if (composite(k, i) < thr) return 0ull;
      const double e = rw.weight_f(KO::value(k));
      return e >= minw ? __double2ull_rn(e * static_cast<double>(1ull << kWeightBits)) : 0ull;
    };
    u64 m = 0;
    each([&](uint32_t k, uint32_t i) { m += kept(k, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (lane == 0) sh.wsum[warp] = m;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int i = 0; i < kSWarps; ++i) s += sh.wsum[i];
      sh.mass = s;
    }
    cluster.sync();
    u64 total = 0, before = 0, own = 0;
    for (int r = 0; r < nrank; ++r) {
      const u64 x = *cluster.map_shared_rank(&sh.mass, r);
      if (r < rank) before += x;
      if (r == rank) own = x;
      total += x;
    }
    const u64 at = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
    if (at >= before && at < before + own) {
      u64 wb = before;
      int ww = 0;
      for (; ww < kSWarps - 1 && at >= wb + sh.wsum[ww]; ++ww) wb += sh.wsum[ww];
      if (warp == ww) {
        u64 run = wb;
        for (int v = v0; v < v1; v += 32) {
          uint4 raw = make_uint4(0, 0, 0, 0);
          if (v + lane < v1) raw = *reinterpret_cast<const uint4 *>(keys + (v + lane) * VEC);
          const K *e = reinterpret_cast<const K *>(&raw);
          const int i0 = base + (v + lane) * VEC - pad;
          u64 mine = 0;
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (e[j] > KO::kNone) mine += kept(e[j], i0 + j);
          u64 incl = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 y = shfl_up64(incl, o);
            if (lane >= o) incl += y;
          }
          const u64 sum = __shfl_sync(0xffffffffu, incl, 31);
          if (at < run + sum) {
            u64 c = run + incl - mine;
            if (at >= c && at < c + mine) {
              for (int j = 0; j < VEC; ++j) {
                if (e[j] <= KO::kNone) continue;
                const u64 w = kept(e[j], i0 + j);
                if (at < c + w) {
                  finish(e[j], i0 + j);
                  break;
                }
                c += w;
              }
            }
            break;
          }
          run += sum;
        }
      }
    }
  }
  cluster.sync();  // no CTA leaves while another may read its shared memory
}

template <typename T>
int launch_sample(SampleParams p, cudaStream_t s) {
  using K = typename KeyOf<T>::K;
  static std::atomic<unsigned long long> attr_set{0};
  constexpr int kSmemMax = 227 * 1024;
  if (smem_limit_once(attr_set, sample_kernel<T>, kSmemMax) != cudaSuccess)
    return check_launch("sample_kernel smem attribute");
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16 + 64;
  // CTAs per row: at least what the row needs of shared memory; more while
  // that adds CTAs up to two per SM and leaves 4096 tokens to each
  auto slice_of = [&](int c) { return ((p.vocab + c - 1) / c + 7) / 8 * 8; };
  int c = 1;
  while (c < kMaxCluster && fixed + size_t(slice_of(c)) * sizeof(K) > size_t(kSmemMax)) c *= 2;
  while (c < kMaxCluster && int64_t(p.rows) * c * 2 <= 2 * num_sms() && slice_of(2 * c) >= 2048)
    c *= 2;
  p.slice = slice_of(c);
  const size_t smem = fixed + size_t(p.slice) * sizeof(K);
  if (smem > size_t(kSmemMax) || p.slice > kMaxSlice)
    return fail(MI_ERR_UNSUPPORTED, "mi_sample_tokens: vocabulary of %d too large", p.vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * c);
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(MI_ERR_CUDA, "sample_kernel launch: %s", cudaGetErrorString(e));
  }
  return check_launch("sample_kernel");
}

}  // namespace
}  // namespace mi

extern "C" int mi_sample_tokens(const void *logits, int64_t row_stride, int32_t rows,
                                int32_t vocab, int32_t dtype, const float *uniform,
                                const float *temperature, float temperature_all,
                                const int32_t *top_k, int32_t top_k_all, const float *top_p,
                                float top_p_all, const float *min_p, float min_p_all,
                                int32_t *out, float *logprob, int32_t *status,
                                mi_stream_t stream) {
  using namespace mi;
  MI_REQUIRE(rows >= 0 && vocab > 0 && vocab <= (1 << kIdxBits),
             "mi_sample_tokens: rows = %d, vocab = %d (1 to %d)", rows, vocab, 1 << kIdxBits);
  if (rows == 0) return MI_OK;
  MI_REQUIRE(logits && uniform && out, "mi_sample_tokens: null pointer");
  MI_REQUIRE(rows <= (1 << 24), "mi_sample_tokens: rows = %d", rows);
  MI_REQUIRE(rows == 1 || row_stride >= vocab, "mi_sample_tokens: row stride");
  const int es = elt_size(dtype);
  MI_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0, "mi_sample_tokens: alignment");
  SampleParams p{logits, row_stride, rows, vocab, 0, uniform, temperature, top_p, min_p, top_k,
                 temperature_all, top_p_all, min_p_all, top_k_all, out, logprob, status};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MI_DTYPE_BF16: return launch_sample<__nv_bfloat16>(p, s);
    case MI_DTYPE_F16: return launch_sample<__half>(p, s);
    case MI_DTYPE_F32: return launch_sample<float>(p, s);
    default: return fail(MI_ERR_INVALID, "mi_sample_tokens: bad dtype %d", dtype);
  }
}

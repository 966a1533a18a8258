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
// = the largest), computed in 64-bit floating point from the logit alone (to
// 2^-39 of themselves: the series of the exponential), and summed as integers:
// sums are the same in any order, so the result does not depend on how the row
// is split or on the order of atomics. The rounding to whole units is half a
// unit a token: 2^-27 of the largest weight over 2^18 tokens at the most.
//
// One thread-block cluster per row (1 to 8 CTAs); each CTA keeps its slice of
// the row in shared memory, read from HBM once. The passes exchange through
// distributed shared memory:
//   1. the largest logit (packed maxima while the slice comes in);
//   2. a histogram over -log2 w in steps of 1/16, from which follows a bin at
//      or above which everything that may be kept lies: token counts for
//      top-k; for top-p counts times each bin's least or most weight, against
//      p times the row's mass. Only the tokens within 2^-16 of the largest
//      weight (for top-k, within 12 of the largest logit) are counted at first
//      (most of a row's are not, and an atomic a token would be the kernel's
//      largest cost); where that does not decide,
//      a second pass counts down to 2^-64 (nothing below 2^-45 can be drawn).
//      The mass is summed in the same pass, with the exact 64-bit exponential
//      within 2^-8, and below it with the hardware's exp2, good to mass_error.
//      Where a top-p edge may lie closer to the target than that, one more
//      pass sums the row in 64 bits (9 us at 152064 tokens);
//   3. if no more than kCap tokens lie at or above that bin (the usual case),
//      they are gathered, one per thread, and every filter and the draw happen
//      on that list with exact weights, each as a search for the token at which
//      a running sum crosses its target: by comparing with all others (tens of
//      tokens as a rule; sorting needs more barriers than that takes), on a long
//      list with those of the same 128th only;
//   4. else ("wide" sets) the histogram brackets the bin where the prefix ends
//      (exactly for counts; for masses between the bins' least and most
//      weights), and divisions of the bracket's range of composites by 256,
//      with exact masses, narrow the threshold down until kCap tokens are left
//      in it. The draw is then one more pass over the row: mass per warp, then
//      the warp that holds u's place scans its tokens.
// The histogram's bins are linear in x: bins of the key's own bits would hold
// most of a row in a few bins.
//
// Bound by latency, not by its one read of the row: a row is a chain of
// cluster barriers of 1-2 us with a few passes over shared memory between
// them. Measured (CUDA graph): 12.3 us for 1 x 32768, 13.4 for 9 x 50257; 70-75
// us for 64 x 152064 bf16 (nucleus of 0.9, by the rows drawn; those whose nucleus
// is wide take 50 us of it), 121 us for 200 x 152064 fp32 with mixed settings (1.01 TB/s;
// clusters of 8 with two CTAs per SM pass in 5.4 waves).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "mi_common.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace mi {
namespace {

constexpr int kSThreads = 512;
constexpr int kSWarps = kSThreads / 32;
constexpr int kBins = 256;
constexpr int kCap = 512;        // tokens resolved on a list (one per thread)
constexpr int kMaxCluster = 8;   // portable cluster size
constexpr int kIdxBits = 18;     // vocabulary <= 2^18
constexpr uint32_t kIdxMask = (1u << kIdxBits) - 1;
constexpr int kWeightBits = 44;  // the largest weight is 2^44
constexpr double kOne = 1ull << kWeightBits;
constexpr int kFine = 1024;      // bins of 1/16 of -log2 w (two per thread)
constexpr int kNear = 256;       // bins of the first pass by mass: down to 2^-16
constexpr float kNearX = 12.f;   // logits below the largest that it counts for top-k, at least
constexpr int kShort = 128;      // lists up to this are searched as one
constexpr float kExact = 128.f;  // exact weights down to 2^-8
// Error of the mass M that is summed with the hardware's exp2, all of it below
// 2^-8 of the largest weight: of a weight of 2^-o three roundings of o, 3 ln 2
// 2^-24 o, exp2's own 2^-22, and the seven fp32 additions of a vector's eight
// weights, 7 2^-24 (vectors are summed in 64 bits). The sum of w o is at most
// M log2(N / M) over N tokens (uniform weights have the largest), M in units of
// the largest weight.
__device__ __forceinline__ double mass_error(double m, int tokens) {
  return m * (1.3e-7 * log2f(static_cast<float>(tokens * kOne / fmax(m, kOne * 1e-6))) + 6.6e-7);
}
constexpr float kRound = 8388608.f;  // adding it rounds to an integer, in the low bits
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
  static constexpr K kEmpty = 0xFF80;  // -inf
  __device__ static K bits(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
  __device__ static float raw(K b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
  // larger of each pair of numbers in a word (a NaN loses)
  __device__ static uint32_t max_word(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162 *>(&a),
                                     *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ static float max_of(uint32_t w) {
    return fmaxf(raw(static_cast<K>(w)), raw(static_cast<K>(w >> 16)));
  }
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
  static constexpr K kEmpty = 0xFC00;
  __device__ static K bits(float x) { return __half_as_ushort(__float2half_rn(x)); }
  __device__ static float raw(K b) { return __half2float(__ushort_as_half(b)); }
  __device__ static uint32_t max_word(uint32_t a, uint32_t b) {
    const __half2 m =
        __hmax2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ static float max_of(uint32_t w) {
    return fmaxf(raw(static_cast<K>(w)), raw(static_cast<K>(w >> 16)));
  }
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
  static constexpr K kEmpty = 0xFF800000u;
  __device__ static K bits(float x) { return __float_as_uint(x); }
  __device__ static float raw(K b) { return __uint_as_float(b); }
  __device__ static uint32_t max_word(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ static float max_of(uint32_t w) { return __uint_as_float(w); }
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

// A row's weights: functions of the logit alone, the same in every pass.
struct RowW {
  double xmax, c;       // c: log2(e) / T
  float fmax_, fscale;  // fine bins: 16 log2(e) / T
  const double *table;  // 2^(j / 32), shared memory

  // exp((x - xmax) / T) * 2^44 as a 64-bit float, from 2^t = 2^n 2^(j/32) 2^r:
  // |r| <= 1/64, and the series of 2^r to r^4 leaves 2^-39. No branches, so
  // the chains of a vector's tokens overlap.
  __device__ double scaled(float x) const {
    const double t = fmax((static_cast<double>(x) - xmax) * c, -64.0);  // (NaN: -64)
    constexpr double kMagic = 6755399441055744.0 / 32;  // 1.5 * 2^52 in steps of 1/32
    const double kd = t + kMagic;
    const int k = __double2loint(kd);  // round(32 t)
    const double r = t - (kd - kMagic);
    double q = 0.009618129107628477;  // ln2^n / n!
    q = fma(q, r, 0.05550410866482158);
    q = fma(q, r, 0.2402265069591007);
    q = fma(q, r, 0.6931471805599453);
    const double m = table[k & 31];
    double w = fma(q * r, m, m);
    w = __hiloint2double(__double2hiint(w) + (((k >> 5) + kWeightBits) << 20),
                         __double2loint(w));
    return t > -64.0 ? w : 0.0;
  }
  static __device__ u64 whole(double w) {  // nearest integer, by adding 2^52 (w <= 2^44)
    return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & ((1ull << 52) - 1);
  }
  __device__ u64 weight(float x) const { return whole(scaled(x)); }
  // -log2 w in sixteenths (monotone in x: each of the subtraction and product
  // is); +inf or NaN for -inf and NaN logits, which no comparison takes in
  __device__ float steps(float x) const { return (fmax_ - x) * fscale; }
  // whether its bin, the nearest integer, is at most b
  __device__ bool within(float x, int b) const { return steps(x) + kRound <= kRound + b; }
};

// A place in the order, as a logit and a token: x is kept by a threshold when
// it is larger, or as large with no larger index.
struct Place {
  float x;
  uint32_t i;
  __device__ bool takes(float y, uint32_t j) const { return y > x || (y == x && j <= i); }
};

struct __align__(16) Bin {
  uint32_t n, l0, l1, l2;  // count; mass limbs
};

struct Shared {
  double table[32];
  uint32_t fine[2][kFine];  // one buffer per search
  union {  // a list is searched after the last read of any histogram
    Bin hist[2][kBins];
    ulonglong2 pairs[kCap];         // entries of the gathered list: order, weight
  };
  u64 list[kCap];   // this CTA's gathered composites
  u64 share[128];                   // a long list's sums per 128th
  u64 acc[4];                       // integer sums over the list; [3]: entries in pairs
  u64 cross;
  int close;
  u64 scan[kSWarps];
  uint32_t warp_n[kSWarps];
  float warp_hi[kSWarps];
  u64 wsum[kSWarps];
  double dsum[kSWarps], dsum2[kSWarps], msum[3][kSWarps];
  // read by the other CTAs of the cluster, each written once before a barrier
  float maxv;
  double lsum;       // sum of exp(x - max), temperature 1
  // per search: mass from 64-bit exponentials, from exp2, and what of both the
  // first pass counts
  double masses[2][3];
  double exact[2];   // all the mass from 64-bit exponentials alone
  u64 mass, over;
  uint32_t first;    // lowest token with the largest logit
  uint32_t list_n[2];
  // block-wide results
  u64 r_u64[4];
  uint32_t r_u32[4];
  int token;
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
  return __shfl_up_sync(0xffffffffu, v, o);
}

// Inclusive block scan of one 64-bit value per thread (in a fixed order).
template <typename V>
__device__ V block_scan(V v, void *buf) {
  V *s = static_cast<V *>(buf);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // (s may still be read from an earlier call)
  if (lane == 31) s[warp] = v;
  __syncthreads();
  V before = 0;
#pragma unroll
  for (int i = 0; i < kSWarps; ++i)
    if (i < warp) before += s[i];
  return v + before;
}

template <typename T>
__global__ void __launch_bounds__(kSThreads, 2) sample_kernel(const SampleParams p) {
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

  for (int i = tid; i < 2 * kFine; i += kSThreads) sh.fine[0][i] = 0;
  if (tid < 2) sh.list_n[tid] = 0;
  if (tid < 4) sh.acc[tid] = 0;
  if (tid < 32) sh.table[tid] = exp2(tid * (1.0 / 32));
  if (tid == 0) {
    sh.token = -1;
    sh.first = 0xFFFFFFFFu;
  }

  // ---- 1. the slice into shared memory; its largest logit ---------------------
  uint32_t top = sizeof(K) == 2 ? KO::kEmpty * 0x10001u : KO::kEmpty;
  const uint32_t empty = top;
  // (NaN becomes -inf, the number a maximum with -inf returns)
  auto clean = [&](uint4 r) {
    return make_uint4(KO::max_word(r.x, empty), KO::max_word(r.y, empty),
                      KO::max_word(r.z, empty), KO::max_word(r.w, empty));
  };
  auto vec_top = [](uint4 r) {
    return KO::max_word(KO::max_word(r.x, r.y), KO::max_word(r.z, r.w));
  };
  constexpr int kAhead = 4;  // vectors a lane has in flight
  for (int vb = v0 + lane; vb < v1; vb += 32 * kAhead) {
    uint4 raw[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int v = vb + 32 * a, i0 = v * VEC - pad;  // first token of the vector
      raw[a] = make_uint4(empty, empty, empty, empty);
      if (v < v1) {
        if (i0 >= 0 && i0 + VEC <= n) {
          raw[a] = __ldcs(reinterpret_cast<const uint4 *>(src + i0));
        } else {
          const K *bits = reinterpret_cast<const K *>(src);
          K *k = reinterpret_cast<K *>(&raw[a]);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (i0 + j >= 0 && i0 + j < n) k[j] = bits[i0 + j];
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const uint4 r = clean(raw[a]);
      top = KO::max_word(top, vec_top(r));
      if (vb + 32 * a < v1) *reinterpret_cast<uint4 *>(keys + (vb + 32 * a) * VEC) = r;
    }
  }
  float best = KO::max_of(top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sh.dsum[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSWarps; ++i) best = fmaxf(best, static_cast<float>(sh.dsum[i]));
    sh.maxv = best;
  }
  cluster.sync();
  // f(rank, that CTA's *field), four loads in flight together
  auto ranks = [&](auto *field, auto &&f) {
    for (int r0 = 0; r0 < nrank; r0 += 4) {
      std::remove_reference_t<decltype(*field)> v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = *cluster.map_shared_rank(field, min(r0 + r, nrank - 1));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + r < nrank) f(r0 + r, v[r]);
    }
  };
  float xmax = -INFINITY;
  ranks(&sh.maxv, [&](int, float v) { xmax = fmaxf(xmax, v); });
  const bool none = xmax == -INFINITY;
  if (xmax == INFINITY) {  // the limit: +inf logits weigh the same, all others nothing
    for (int v = v0 + lane; v < v1; v += 32) {
      K *e = keys + v * VEC;
      for (int j = 0; j < VEC; ++j) e[j] = KO::raw(e[j]) == INFINITY ? K(0) : KO::kEmpty;
    }
    __syncwarp();
    xmax = 0.f;
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
  // min-p on the scaled weights
  const double minw = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) * (1ull << kWeightBits)
                                  : 0.0;
  RowW rw;
  rw.fmax_ = xmax;
  rw.xmax = xmax;
  rw.c = greedy ? 1.0 : 1.4426950408889634 / static_cast<double>(temp);
  // (finite and not 0: 0 * it is 0, and inf * it is inf)
  rw.fscale = static_cast<float>(fmin(fmax(16.0 * rw.c, 1e-30), 3e38));
  rw.table = sh.table;

  // f(logit, token) for this thread's tokens above -inf that in(logit, token)
  // accepts, none of them below least_x: one test passes over a vector of VEC
  // tokens, as most are. The tests run over the whole vector, f over a mask of
  // what they found: f's code once (it may be long), and as often as a lane of
  // the warp needs it.
  auto each = [&](float least_x, auto &&in, auto &&f) {
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
      if (!(KO::max_of(vec_top(raw)) >= least_x)) continue;
      const K *e = reinterpret_cast<const K *>(&raw);
      const int i0 = base + v * VEC - pad;
      uint32_t found = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = KO::raw(e[j]);
        if (x > -INFINITY && in(x, static_cast<uint32_t>(i0 + j))) found |= 1u << j;
      }
      while (found) {
        const int j = __ffs(found) - 1;
        found &= found - 1;
        f(KO::raw(keys[v * VEC + j]), static_cast<uint32_t>(i0 + j));
      }
    }
  };
  auto comp_of = [&](float x, uint32_t i) { return composite(KO::key(KO::bits(x)), i); };
  // one value per thread summed over the CTA in a fixed order; thread 0 has it
  auto block_sum = [&](double d, double *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) part[warp] = d;
    __syncthreads();
    if (tid == 0)
      for (int i = 1; i < kSWarps; ++i) d += part[i];
    return d;
  };

  // log-sum-exp of the row at temperature 1, for the log-probability
  if (p.logprob && !none) {
    float s = 0.f;
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
      const K *e = reinterpret_cast<const K *>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += fast_exp2((KO::raw(e[j]) - rw.fmax_) * kLog2e);
    }
    const double d = block_sum(s, sh.dsum2);
    if (tid == 0) sh.lsum = d;
  }

  // the last token kept, once a search has found one (before: any above -inf)
  Place thr{-INFINITY, 0};
  bool cut = false;
  auto place_of = [&](u64 c) { return Place{KO::value(comp_key(c)), comp_idx(c)}; };
  bool done = false;  // resolved on a list (by every CTA alike)
  int sel = 0;        // this threshold search (fine, total and list_n buffers)
  int level = 0;      // wide histogram levels done (hist buffer)
  int listed = 0;     // tokens gathered

  // Sums this level's histogram over the cluster (after its barrier) and finds
  // the first bin whose running sum, past what lies above, reaches the target:
  // r_u32 = {bin or kBins, count in earlier bins, count in it}, r_u64[0] = mass
  // in earlier bins.
  auto merge = [&](bool by_mass, double target, double above, u64 above_m) {
    u64 m = 0, c = 0;
    if (tid < kBins)
      ranks(reinterpret_cast<uint4 *>(&sh.hist[level & 1][tid]), [&](int, uint4 b) {
        c += b.x;  // a Bin
        m += static_cast<u64>(b.y) + (static_cast<u64>(b.z) << kLimb) +
             (static_cast<u64>(b.w) << (2 * kLimb));
      });
    const u64 cs = block_scan(c, sh.scan);
    const u64 ms = by_mass ? block_scan(m, sh.scan) : 0;
    if (tid == 0) sh.r_u32[0] = kBins;
    __syncthreads();
    const double at = by_mass ? static_cast<double>(above_m + ms) : above + static_cast<double>(cs);
    const double was = by_mass ? static_cast<double>(above_m + ms - m)
                               : above + static_cast<double>(cs - c);
    // (nothing earlier anywhere: at least one token is kept)
    const bool only = cs == c && (by_mass ? above_m == 0 : above == 0.0);
    if (tid < kBins && c > 0 && at >= target && (was < target || only)) {
      sh.r_u32[0] = tid;
      sh.r_u32[1] = static_cast<uint32_t>(cs - c);
      sh.r_u32[2] = static_cast<uint32_t>(c);
      sh.r_u64[0] = ms - m;
    }
    __syncthreads();
    ++level;
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
  auto gather = [&](float least_x, auto &&in) {
    uint32_t *cnt = &sh.list_n[sel & 1];
    each(least_x, in, [&](float x, uint32_t i) {
      const uint32_t at = atomicAdd(cnt, 1u);
      if (at < kCap) sh.list[at] = comp_of(x, i);
    });
    cluster.sync();
    // this thread's entry of the ranks' lists, one after the other
    int src_rank = -1;
    uint32_t off = 0, at = 0;
    ranks(cnt, [&](int r, uint32_t m) {
      m = min(m, static_cast<uint32_t>(kCap));
      if (tid >= off && tid < off + m) src_rank = r, at = tid - off;
      off += m;
    });
    const u64 mine = src_rank >= 0 ? *cluster.map_shared_rank(&sh.list[at], src_rank) : 0;
    listed = min(off, static_cast<uint32_t>(kCap));
    return mine;
  };
  auto weight_of = [&](u64 c) { return c ? rw.weight(KO::value(comp_key(c))) : 0ull; };
  // The listed token at which the running sum of w, from `above` on and in
  // falling `order`, reaches the target (always one: the first, if none is
  // needed): its order. part: the entry's 128th, rising as the order falls.
  // With a slack: sh.close if the token's edges are not that far from the target.
  auto crossing = [&](bool has, u64 order, u64 w, uint32_t part, u64 above, double target,
                      float slack = -1.f) {
    const bool shorts = listed <= kShort;
    __syncthreads();  // (an earlier call's result has been read)
    if (tid < 128) sh.share[tid] = 0;
    if (tid == 0) {
      sh.acc[3] = 0;
      sh.cross = 0;
      sh.close = 0;
      sh.r_u32[0] = 0;
      sh.r_u64[0] = above;
    }
    __syncthreads();
    if (!shorts) {
      if (has) atomicAdd(&sh.share[part], w);
      __syncthreads();
      if (warp == 0) {  // four parts a lane
        u64 v[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += v[i] = sh.share[lane * 4 + i];
        u64 run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = shfl_up64(run, o);
          if (lane >= o) run += y;
        }
        run += above - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool first = run == 0;  // (nothing before it)
          if (v[i] && static_cast<double>(run + v[i]) >= target &&
              (first || static_cast<double>(run) < target)) {
            sh.r_u32[0] = lane * 4 + i;
            sh.r_u64[0] = run;
          }
          run += v[i];
        }
      }
      __syncthreads();
      has = has && part == sh.r_u32[0];
    }
    if (has) sh.pairs[atomicAdd(reinterpret_cast<uint32_t *>(&sh.acc[3]), 1u)] =
        make_ulonglong2(order, w);
    __syncthreads();
    if (has) {
      const int m = static_cast<int>(sh.acc[3]);
      u64 before = sh.r_u64[0];
#pragma unroll 4
      for (int j = 0; j < m; ++j) {
        const ulonglong2 o = sh.pairs[j];
        if (o.x > order) before += o.y;
      }
      if (w && static_cast<double>(before + w) >= target &&
          (before == 0 || static_cast<double>(before) < target)) {
        sh.cross = order;
        sh.close = target - static_cast<double>(before) <= slack ||
                   static_cast<double>(before + w) - target <= slack;
      }
    }
    __syncthreads();
    return sh.cross;
  };
  // sh.acc[slot] += v over the CTA (integers: in any order)
  auto accumulate = [&](u64 v, int slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0 && v) atomicAdd(&sh.acc[slot], v);
  };
  // the row's mass in 64-bit exponentials (of what a first search left)
  auto exact_mass = [&]() {
    double s = 0.0;
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
      const K *e = reinterpret_cast<const K *>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = KO::raw(e[j]);
        const double w = rw.scaled(x);
        s += !cut || thr.takes(x, base + v * VEC - pad + j) ? w : 0.0;
      }
    }
    s = block_sum(s, sh.dsum);
    if (tid == 0) sh.exact[sel] = s;
    cluster.sync();
    double all = 0.0;
    ranks(&sh.exact[sel], [&](int, double v) { all += v; });
    return all;
  };
  // ordered key of the largest logit (its float maps back to the type's bits)
  auto key_of_max = [&]() -> uint32_t { return KO::key(KO::bits(rw.fmax_)); };
  // ---- 2. to 4. the filters' thresholds ----------------------------------------
  const int nsel = (use_k ? 1 : 0) + (use_p ? 1 : 0);
  for (; sel < nsel && !none && !done; ++sel) {
    const bool by_mass = !(use_k && sel == 0);
    // -- 2. counts per bin, and the mass
    uint32_t *fine = sh.fine[sel];
    double sum = 0.0, fast = 0.0;  // mass; of exp2s (in units of the largest)
    float inside = 0.f;  // of it: what is counted, to fp32
    // weight at t sixteenths, for what lies below 2^-8 (t = inf: 0)
    auto far = [](float t) { return fast_exp2(t * -0.0625f); };
    auto count = [&](float z) { atomicAdd(&fine[__float_as_uint(z) & (kFine - 1)], 1u); };
    const int window =
        by_mass ? kNear
                : max(kNear, static_cast<int>(fminf(kNearX * rw.fscale, kFine - 2.f)) & ~1);
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
      const K *e = reinterpret_cast<const K *>(&raw);
      const float t0 = rw.steps(KO::max_of(vec_top(raw)));  // the vector's least
      const bool near = t0 + kRound <= kRound + (window - 1);
      if (!near && !by_mass) continue;
      float t[VEC], w[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) t[j] = rw.steps(KO::raw(e[j]));
      if (cut) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!thr.takes(KO::raw(e[j]), base + v * VEC - pad + j)) t[j] = INFINITY;
      }
      if (by_mass) {
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = far(t[j]);
        if (t0 < kExact) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const double x = rw.scaled(KO::raw(e[j]));
            sum += t[j] < kExact ? x : 0.0;
            part += t[j] < kExact ? 0.f : w[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) part += w[j];
        }
        fast += part;
      }
      if (near && by_mass) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float z = t[j] + kRound;
          if (z <= kRound + (window - 1)) {
            count(z);
            inside += w[j];
          }
        }
      } else if (near) {  // few: a mask, then a loop over what it found
        uint32_t found = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (t[j] + kRound <= kRound + (window - 1)) found |= 1u << j;
        while (found) {
          const int j = __ffs(found) - 1;
          found &= found - 1;
          count(rw.steps(KO::raw(keys[v * VEC + j])) + kRound);
        }
      }
    }
    if (by_mass) {
      // the three sums over the CTA, in a fixed order, a thread each
      double v[3] = {sum, fast, inside};
#pragma unroll
      for (int i = 0; i < 3; ++i) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        if (lane == 0) sh.msum[i][warp] = v[i];
      }
      __syncthreads();
      if (tid < 3) {
        double d = 0.0;
        for (int i = 0; i < kSWarps; ++i) d += sh.msum[tid][i];
        sh.masses[sel][tid] = tid == 0 ? d : d * kOne;
      }
    }
    double target = top_k, total = 0.0;
    float unsure = -1.f;  // error of the target
    float beyond = 0.f;  // mass not counted
    int fb = kFine, fa = kFine;
    uint32_t above_n = 0, upto_n = 0;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {  // undecided: the other bins
        for (int v = v0 + lane; v < v1; v += 32) {
          const uint4 raw = *reinterpret_cast<const uint4 *>(keys + v * VEC);
          const K *e = reinterpret_cast<const K *>(&raw);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float x = KO::raw(e[j]), z = rw.steps(x) + kRound;
            if (z > kRound + (window - 1) && z <= kRound + (kFine - 1) &&
                (!cut || thr.takes(x, base + v * VEC - pad + j)))
              count(z);
          }
        }
      }
      cluster.sync();
      if (by_mass && pass == 0) {
        struct Masses { double slow, fast, in; };
        double m = 0.0, in = 0.0;
        ranks(reinterpret_cast<Masses *>(sh.masses[sel]), [&](int, Masses v) {
          total += v.slow;
          m += v.fast;
          in += v.in;
        });
        total += m;
        target = total * top_p;
        unsure = static_cast<float>(mass_error(m, p.vocab));
        beyond = static_cast<float>(total - in);
      }
      // The first bin by which the prefix has certainly reached the target (fb),
      // and the first by which it may have (fa): exact for counts; by mass the
      // prefix lies between its counts times the bins' least and most weights,
      // and between the whole mass less the rest's most and least weights (1e-4:
      // the roundings of t, exp2f, fp32 sums). Thread t has bins 2 t, 2 t + 1.
      uint32_t c0 = 0, c1 = 0;
      if (pass || tid < window / 2)
        ranks(reinterpret_cast<uint2 *>(sh.fine[sel]) + tid, [&](int, uint2 v) {
          c0 += v.x;
          c1 += v.y;
        });
      constexpr float kLeast = 0.95760328f;  // 2^(-1/16): a bin's least weight over its most
      const float top = by_mass ? fast_exp2(-0.0625f * (2 * tid - 0.5f) + kWeightBits) : 0.f;
      const float h0 = c0 * top, h1 = c1 * (top * kLeast);
      uint32_t n_in = c0 + c1;
      float hi_in = h0 + h1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, n_in, o);
        const float z = __shfl_up_sync(0xffffffffu, hi_in, o);
        if (lane >= o) {
          n_in += y;
          hi_in += z;
        }
      }
      if (lane == 31) {
        sh.warp_n[warp] = n_in;
        sh.warp_hi[warp] = hi_in;
      }
      if (tid == 0) sh.r_u32[0] = sh.r_u32[2] = kFine;
      __syncthreads();
      uint32_t n_all = 0;
      float hi_all = 0.f;
#pragma unroll
      for (int i = 0; i < kSWarps; ++i) {
        if (i == warp) {
          n_in += n_all;
          hi_in += hi_all;
        }
        n_all += sh.warp_n[i];
        hi_all += sh.warp_hi[i];
      }
      const uint32_t n0 = n_in - c1;  // up to bin 2 t
      bool fb0, fb1, fa0, fa1;
      if (by_mass) {
        const float whole = static_cast<float>(total), goal = static_cast<float>(target);
        const float hi0 = hi_in - h1, slack = 1e-4f * whole;
        const float seen = whole - (pass ? 0.f : beyond);  // mass of the counted
        fb0 = fmaxf(hi0 * kLeast, seen - (hi_all - hi0)) - slack >= goal;
        fb1 = fmaxf(hi_in * kLeast, seen - (hi_all - hi_in)) - slack >= goal;
        fa0 = fminf(hi0, seen - (hi_all - hi0) * kLeast) + slack >= goal;
        fa1 = fminf(hi_in, seen - (hi_all - hi_in) * kLeast) + slack >= goal;
      } else {
        fb0 = fa0 = n0 >= static_cast<uint32_t>(top_k);
        fb1 = fa1 = n_in >= static_cast<uint32_t>(top_k);
      }
      // (a bin before the first token's does not count: one token is always kept)
      const int b0 = n0 > 0 ? 2 * tid : 2 * tid + 1;
      const uint32_t wb = __reduce_min_sync(
          0xffffffffu, n_in > 0 && (fb0 || fb1) ? (fb0 ? b0 : 2 * tid + 1) : kFine);
      const uint32_t wa = __reduce_min_sync(
          0xffffffffu, n_in > 0 && (fa0 || fa1) ? (fa0 ? b0 : 2 * tid + 1) : kFine);
      if (lane == 0) {  // (a warp at a time: an atomic a thread on one word costs microseconds)
        if (wb < kFine) atomicMin(&sh.r_u32[0], wb);
        if (wa < kFine) atomicMin(&sh.r_u32[2], wa);
      }
      __syncthreads();
      fb = static_cast<int>(sh.r_u32[0]), fa = static_cast<int>(sh.r_u32[2]);
      if (tid == fb >> 1) sh.r_u32[1] = fb & 1 ? n_in : n0;
      if (tid == min(fa, kFine - 1) >> 1)  // the count above bin fa
        sh.r_u32[3] = fa == kFine ? n_in : (fa & 1 ? n0 : n0 - c0);
      __syncthreads();
      upto_n = sh.r_u32[1], above_n = sh.r_u32[3];
      if (fb < window) break;
      __syncthreads();
    }
    // fewer than k tokens down to 2^-64: what lies below is never drawn
    if (!by_mass && fb == kFine) continue;
    if (fb < kFine && upto_n <= kCap) {
      // -- 3. everything that may be kept fits the list
      // (half a bin below what bin fb takes: more than the roundings)
      const float least_x = rw.fmax_ - (fb + 1.f) / rw.fscale;
      const u64 c = gather(least_x, [&](float x, uint32_t i) {
        return rw.within(x, fb) && (!cut || thr.takes(x, i));
      });
      const u64 w = weight_of(c);
      bool keep = c != 0;
      // a list's 128ths by bin (fb + 1 bins)
      const uint32_t part =
          c ? (__float_as_uint(rw.steps(KO::value(comp_key(c))) + kRound) & (kFine - 1)) * 128 /
                  (fb + 1)
            : 0;
      if (!by_mass && static_cast<int>(upto_n) > top_k) {
        const u64 last = crossing(keep, c, 1, part, 0, top_k);  // (every thread: it has barriers)
        keep = keep && c >= last;
      }
      if (use_p) {
        // (mass search: the target is a share of all the row's mass)
        double want = target;
        if (!by_mass) {
          accumulate(keep ? w : 0, 0);
          __syncthreads();
          want = top_p * static_cast<double>(sh.acc[0]);
        }
        u64 last = crossing(keep, c, w, part, 0, want, unsure);
        if (sh.close) {
          want = exact_mass() * top_p;
          last = crossing(keep, c, w, part, 0, want);
        }
        keep = keep && c >= last;
      }
      if (minw > 0.0) keep = keep && rw.scaled(KO::value(comp_key(c))) >= minw;
      accumulate(keep ? w : 0, 1);
      __syncthreads();
      // the first token, by index, whose running mass exceeds u's share (weights
      // are integers: reaches the share's floor and one)
      const u64 at = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sh.acc[1]));
      const u64 low = c & kIdxMask;  // falls as the index grows
      const uint32_t at_part = keep ? comp_idx(c) * 128 / p.vocab : 0;
      const u64 pick = crossing(keep, low, w, at_part, 0, static_cast<double>(at) + 1.0);
      if (tid == 0) sh.token = static_cast<int>(kIdxMask - pick);
      __syncthreads();
      done = true;
      break;
    }
    // -- 4. wide: the range of composites of bins fa to fb, or to the row's end;
    // its keys by a 32-way search (bins fall as the key grows), alike in every warp
    __syncthreads();
    u64 lo, hi;
    {
      const uint32_t kmax = key_of_max();
      auto edge = [&](int limit) {  // smallest key above kNone with bin <= limit
        uint32_t l = KO::kNone + 1, h = kmax;  // the answer is in [l, h]
        while (l < h) {
          const uint32_t step = (h - l + 31) / 32;
          const u64 at = static_cast<u64>(l) + static_cast<u64>(step) * lane;
          const bool in = at >= h || rw.within(KO::value(static_cast<uint32_t>(at)), limit);
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
      const uint32_t klo = fb < kFine ? edge(fb) : KO::kNone + 1;
      const uint32_t khi = fa == 0 ? kmax : edge(fa - 1) - 1;
      lo = static_cast<u64>(klo) << kIdxBits;
      hi = (static_cast<u64>(khi) << kIdxBits) | kIdxMask;
      if (cut) lo = max(lo, composite(KO::key(KO::bits(thr.x)), thr.i));
    }
    if (lo > hi) continue;  // no token past the bins: all are kept
    // With the mass in 64 bits: at once where an eighth of the edges or more lie
    // closer to the target than it is known (bin fb has the smallest tokens that
    // may be one), else only after a search that ended so close.
    const u64 lo0 = lo, hi0 = hi;
    bool all = false;  // the target is not reached: everything in the range is kept
    for (bool settle = by_mass && fast_exp2(-0.0625f * fb) * kOne < 16 * unsure;; settle = true) {
      if (settle) {  // (its cluster barrier: every CTA has read the lists)
        target = exact_mass() * top_p;
        unsure = -1.f;
        lo = lo0, hi = hi0;
        if (tid == 0) sh.list_n[sel & 1] = 0;
      }
      // divide the range until its tokens fit the list; the first time also the
      // mass above it (the count above is known)
      u64 above_m = 0;
      double above = above_n;
      all = false;
      for (uint32_t inside = UINT32_MAX; inside > kCap;) {
        const int shift = max(0, 64 - __clzll(static_cast<long long>(hi - lo)) - 8);
        for (int i = tid; i < kBins; i += kSThreads) sh.hist[level & 1][i] = Bin{0, 0, 0, 0};
        __syncthreads();
        u64 over = 0;
        const bool first = inside == UINT32_MAX;
        const Place least = place_of(lo), most = place_of(hi + 1);  // range: takes least, not most
        each(
            least.x,
            [&](float x, uint32_t i) {
              return least.takes(x, i) && ((by_mass && first) || !most.takes(x, i));
            },
            [&](float x, uint32_t i) {
              const u64 w = by_mass ? rw.weight(x) : 0;
              if (most.takes(x, i))
                over += w;
              else
                add(static_cast<int>((hi - comp_of(x, i)) >> shift), by_mass, w);
            });
        if (by_mass && first) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) over += __shfl_xor_sync(0xffffffffu, over, o);
          if (lane == 0) sh.wsum[warp] = over;
          __syncthreads();
          if (tid == 0) {
            for (int i = 1; i < kSWarps; ++i) over += sh.wsum[i];
            sh.over = over;
          }
        }
        cluster.sync();
        if (by_mass && first) {
          ranks(&sh.over, [&](int, u64 v) { above_m += v; });
          above = static_cast<double>(above_m);
        }
        merge(by_mass, target, above, above_m);
        const uint32_t q = sh.r_u32[0];
        if (q == kBins) {
          all = true;
          break;
        }
        above += sh.r_u32[1];  // (counts; by mass it is above_m that counts)
        inside = sh.r_u32[2];
        above_m += sh.r_u64[0];
        if (by_mass) above = static_cast<double>(above_m);
        __syncthreads();
        hi -= static_cast<u64>(q) << shift;
        const u64 width = (1ull << shift) - 1;
        if (hi - lo > width) lo = hi - width;
      }
      if (all && unsure < 0.f) break;
      if (all) continue;
      const Place least = place_of(lo), most = place_of(hi + 1);
      const u64 gc = gather(
          least.x, [&](float x, uint32_t i) { return least.takes(x, i) && !most.takes(x, i); });
      const u64 w = by_mass ? weight_of(gc) : (gc ? 1 : 0);
      const int shift = max(0, 64 - __clzll(static_cast<long long>(hi - lo)) - 7);
      const u64 last = crossing(gc != 0, gc, w, gc ? static_cast<uint32_t>((hi - gc) >> shift) : 0,
                                by_mass ? above_m : static_cast<u64>(above), target, unsure);
      if (sh.close && unsure >= 0.f) continue;
      if (last) thr = place_of(last);
      break;
    }
    if (all) thr = place_of(lo);
    cut = true;
    __syncthreads();
  }

  // ---- the draw -----------------------------------------------------------------
  auto finish = [&](float x, int token) {  // one thread of the cluster
    p.out[row] = token;
    if (p.logprob) {
      double s = 0;
      ranks(&sh.lsum, [&](int, double v) { s += v; });
      const double d = x == rw.fmax_ ? 0.0 : static_cast<double>(x) - rw.xmax;
      p.logprob[row] = static_cast<float>(d - log(s));
    }
  };
  if (none) {  // no logit above -inf
    if (rank == 0 && tid == 0) {
      p.out[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
      flag(p.status, MI_STATUS_NO_TOKEN);
    }
  } else if (greedy) {
    uint32_t first = 0xFFFFFFFFu;
    each(
        rw.fmax_, [&](float x, uint32_t) { return x == rw.fmax_; },
        [&](float, uint32_t i) { first = min(first, i); });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) atomicMin(&sh.first, first);
    cluster.sync();  // (every CTA's lsum is written, too)
    if (rank == 0 && tid == 0) {
      ranks(&sh.first, [&](int, uint32_t v) { first = min(first, v); });
      finish(rw.fmax_, static_cast<int>(first));
    }
  } else if (done) {
    // the CTA that holds the token has its logit
    const int t = sh.token;
    if (tid == 0 && t >= base && t < base + n) finish(KO::raw(keys[t - base + pad]), t);
  } else {
    // kept weights of a vector's tokens (0: not kept); any: some lane has one
    auto kept = [&](const K *e, int i0, u64 *w) {
      bool in[VEC], some = false;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = KO::raw(e[j]);
        in[j] = x > -INFINITY && (!cut || thr.takes(x, i0 + j));
        some = some || in[j];
      }
      if (!__any_sync(0xffffffffu, some)) return false;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const double d = rw.scaled(KO::raw(e[j]));
        w[j] = in[j] && d >= minw ? RowW::whole(d) : 0ull;
      }
      return true;
    };
    u64 m = 0;
    if (cut) {
      each(
          thr.x, [&](float x, uint32_t i) { return thr.takes(x, i); },
          [&](float x, uint32_t) {
            const double d = rw.scaled(x);
            m += d >= minw ? RowW::whole(d) : 0ull;
          });
    } else {  // all tokens: whole vectors
      for (int vw = v0; vw < v1; vw += 32) {
        uint4 raw = make_uint4(empty, empty, empty, empty);
        if (vw + lane < v1) raw = *reinterpret_cast<const uint4 *>(keys + (vw + lane) * VEC);
        u64 w[VEC];
        if (kept(reinterpret_cast<const K *>(&raw), base + (vw + lane) * VEC - pad, w)) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) m += w[j];
        }
      }
    }
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
    ranks(&sh.mass, [&](int r, u64 x) {
      if (r < rank) before += x;
      if (r == rank) own = x;
      total += x;
    });
    const u64 at = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
    if (at >= before && at < before + own) {
      u64 wb = before;
      int ww = 0;
      for (; ww < kSWarps - 1 && at >= wb + sh.wsum[ww]; ++ww) wb += sh.wsum[ww];
      if (warp == ww) {
        u64 run = wb;
        for (int v = v0; v < v1; v += 32) {
          uint4 raw = make_uint4(empty, empty, empty, empty);
          if (v + lane < v1) raw = *reinterpret_cast<const uint4 *>(keys + (v + lane) * VEC);
          const K *e = reinterpret_cast<const K *>(&raw);
          const int i0 = base + (v + lane) * VEC - pad;
          u64 w[VEC], mine = 0;
          if (!kept(e, i0, w)) continue;
#pragma unroll
          for (int j = 0; j < VEC; ++j) mine += w[j];
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
              bool open = true;
#pragma unroll
              for (int j = 0; j < VEC; ++j) {
                if (open && at < c + w[j]) {
                  finish(KO::raw(e[j]), i0 + j);
                  open = false;
                }
                c += w[j];
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
  constexpr int kSmemMax = 227 * 1024, kSmemTwo = 112 * 1024;
  if (smem_limit_once(attr_set, sample_kernel<T>, kSmemMax) != cudaSuccess)
    return check_launch("sample_kernel smem attribute");
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16 + 64;
  // CTAs per row: as many as bring the shared memory down to two CTAs per SM
  // (one CTA's barriers pass under the other's work); more while that adds CTAs
  // up to two per SM and leaves 2048 tokens to each (shorter slices gain less
  // than the wider barrier costs). 64 rows of 152064 bf16 take the same time
  // with 4 CTAs each and with 8.
  auto slice_of = [&](int c) { return ((p.vocab + c - 1) / c + 7) / 8 * 8; };
  int c = 1;
  while (c < kMaxCluster && fixed + size_t(slice_of(c)) * sizeof(K) > size_t(kSmemTwo)) c *= 2;
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

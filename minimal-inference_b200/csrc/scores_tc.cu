// Prompt scores on the tensor cores (see scores.cu for what is computed):
// bf16 / fp16, head_dim 64 / 128, page_size a multiple of 16.
//
// Work item: (request, KV head, 128 consecutive keys) and every query row that
// sees any of them, in tiles of up to 128 packed rows (query token x head of
// the group). The product is S^T = K Q^T: keys are the 128 TMEM lanes, query
// rows the columns, so a thread owns one key and the sum over queries stays in
// its registers (rows on the lanes would need a reduction across threads for
// every column). Per element that leaves a scale-and-subtract of the row's
// log-sum-exp, an exp2 and an addition. The exp2 unit (16 per clock and SM)
// takes 1024 clocks a tile; shared memory, which bounds the kernel, takes 512
// for the operands of the 128 x 128 x 128 product, 512 for the row terms (a
// clock per 32 lanes and column) and 256 for the Q tile's arrival. Measured
// (16 prompts of 100-1500 tokens, 32/8 heads of 128): 96 us, 1.4 times that
// bound of 1280 clocks a tile. Tried without gain: quarters or halves of a
// tile to a group, four groups, 256 keys to an item, K tiles an item ahead.
//
// Persistent, one CTA per SM, items from a counter in the workspace, a
// request's first keys (most queries) first. 10 warps:
//   warp 0     producer: TMA loads of the K tile (16-token boxes straight from
//              the pages) and the Q tiles, two K and three Q stages;
//   warp 1     MMA issuer, four 128-column TMEM accumulators;
//   warps 2-9  two groups of four take the tiles in turn: lane = key.
// Each warp keeps the tile's 128 row terms in a shared-memory slice of its own
// (read as broadcasts), loaded one tile ahead. The second group hands its sums
// to the first at the end of an item, so a key's sum has a fixed order.
// Every wait is bounded; TMEM is freed on every path.
#include <algorithm>
#include <type_traits>

#include "scores.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace mi {
namespace {

constexpr int kKeys = 128;      // keys per item (TMEM lanes)
constexpr int kRows = 128;      // packed query rows per tile (columns)
constexpr int kScThreads = 320;
constexpr int kScMaxBatch = 1024;
constexpr int kScSortBatch = 128;
constexpr int kQStages = 3, kKStages = 2, kAcc = 4, kRecs = 4;

template <int D> struct ScLayout {
  static constexpr int DH = D / 64;
  static constexpr int Q_BYTES = DH * kRows * 128;
  static constexpr int K_BYTES = DH * kKeys * 128;
  static constexpr int K_OFF = 0;
  static constexpr int Q_OFF = kKStages * K_BYTES;
  static constexpr int LSE_OFF = Q_OFF + kQStages * Q_BYTES;  // [8 warps][2][128] fp32
  static constexpr int PART_OFF = LSE_OFF + 8 * 2 * kRows * 4;  // [128] fp32
  static constexpr int REC_OFF = PART_OFF + kKeys * 4;
  static constexpr int BAR_OFF = REC_OFF + kRecs * 48;
  static constexpr int META_OFF = BAR_OFF + 64 * 8;
  static constexpr int SMEM = META_OFF + 5 * (kScMaxBatch + 1) * 4 + 1024;
};

// True for one lane of the (converged) warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(p));
  return p != 0;
}

struct __align__(16) ScItem {
  int b, h, j0, n_tiles;   // b < 0: no more items
  int q_start, i0, nq, kvlen;  // first query row; queries [i0, nq) of the request
  int page_base, off;      // causal: query i sees keys j <= off + i
  int pad[2];
};

struct ScArgs {
  ScoreParams p;
  float scale_log2;
  unsigned *ctr;  // [2]: next item, CTAs done; zero between calls. Or null.
};

template <typename T, int D>
__global__ void __launch_bounds__(kScThreads, 1)
    scores_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kvmap, const ScArgs a) {
  using L = ScLayout<D>;
  constexpr int DH = L::DH;
  const ScoreParams &p = a.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
  uint64_t *it_full = bars, *it_empty = bars + kRecs;
  uint64_t *k_full = bars + 8, *k_empty = bars + 10;
  uint64_t *q_full = bars + 12, *q_empty = bars + 15;
  uint64_t *s_full = bars + 18, *s_free = bars + 22;   // [accumulator]
  uint64_t *pt_full = bars + 26, *pt_free = bars + 30; // [lane quarter]
  uint64_t *drain = bars + 34;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 36);
  ScItem *recs = reinterpret_cast<ScItem *>(smem + L::REC_OFF);
  float *part = reinterpret_cast<float *>(smem + L::PART_OFF);
  int *tiles_pre = reinterpret_cast<int *>(smem + L::META_OFF);
  int *s_qo = tiles_pre + (kScMaxBatch + 1);
  int *s_ip = s_qo + (kScMaxBatch + 1);
  int *s_lk = s_ip + (kScMaxBatch + 1);
  int *s_order = s_lk + (kScMaxBatch + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = p.group, tq = kRows / g, m_used = tq * g;

  // ---- once per CTA: key tiles per request, barriers, TMEM --------------------
  auto qo_at = [&](int i) { return min(max(p.qo_indptr[i], 0), p.total_q); };
  for (int i = threadIdx.x; i <= p.batch; i += blockDim.x) {
    const int v = qo_at(i);
    if (blockIdx.x == 0 && (v != p.qo_indptr[i] || (i < p.batch && qo_at(i + 1) < v)))
      flag(p.status, MI_STATUS_BAD_POSITION);
    s_qo[i] = v;
    s_ip[i] = p.indptr[i];
    if (i < p.batch) s_lk[i] = kv_len_of(p.indptr, p.last, i, p.ps);
  }
  __syncthreads();
  // requests with the most keys first (ties by index), by counting
  for (int i = threadIdx.x; i < p.batch; i += blockDim.x) {
    int rank = i;
    if (p.batch <= kScSortBatch) {
      rank = 0;
      for (int j = 0; j < p.batch; ++j)
        rank += (s_lk[j] > s_lk[i] || (s_lk[j] == s_lk[i] && j < i)) ? 1 : 0;
    }
    s_order[rank] = i;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    if (lane == 0) tiles_pre[0] = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int bb = base + lane;
      const int rb = bb < p.batch ? s_order[bb] : 0;
      int x = bb < p.batch && s_qo[rb + 1] > s_qo[rb] ? cdiv(s_lk[rb], kKeys) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (bb < p.batch) tiles_pre[bb + 1] = carry + x;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < kRecs; ++i) {
        mbar_init(&it_full[i], 1);
        mbar_init(&it_empty[i], 9);  // the MMA thread and the 8 summing warps
        mbar_init(&s_full[i], 1);
        mbar_init(&s_free[i], 4);
        mbar_init(&pt_full[i], 1);
        mbar_init(&pt_free[i], 1);
      }
      for (int i = 0; i < kKStages; ++i) {
        mbar_init(&k_full[i], 1);
        mbar_init(&k_empty[i], 1);
      }
      for (int i = 0; i < kQStages; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 1);
      }
      mbar_init(drain, 1);
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // rows of a Q stage that no box covers (128 is no multiple of the group):
  // zero, so their columns stay finite
  for (int i = threadIdx.x; i < kQStages * DH * (kRows - m_used) * 8; i += blockDim.x) {
    const int blk = i / ((kRows - m_used) * 8), rem = i % ((kRows - m_used) * 8);
    *reinterpret_cast<uint4 *>(smem + L::Q_OFF + blk * (kRows * 128) + m_used * 128 + rem * 16) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  fence_mbar_init();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t n_items = static_cast<int64_t>(tiles_pre[p.batch]) * p.hkv;
  bool ok = true;

  if (warp == 0) {
    // ============================ producer ======================================
    const uint64_t pol_q = evict_last_policy(), pol_k = evict_first_policy();
    int kc = 0, qc = 0;  // K and Q tiles issued
    for (int it = 0; ok; ++it) {
      int64_t k = 0;
      if (lane == 0) k = a.ctr ? atomicAdd(a.ctr, 1u) : blockIdx.x + int64_t(it) * gridDim.x;
      k = __shfl_sync(0xffffffffu, k, 0);
      ScItem rec{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, {0, 0}};
      if (k < n_items) {
        int lo = 0, hi = p.batch - 1;  // last position with tiles_pre[pos] * hkv <= k
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (static_cast<int64_t>(tiles_pre[mid]) * p.hkv <= k) lo = mid; else hi = mid - 1;
        }
        const int b = s_order[lo];
        const int rem = static_cast<int>(k - static_cast<int64_t>(tiles_pre[lo]) * p.hkv);
        rec.b = b;
        rec.h = rem % p.hkv;
        rec.j0 = rem / p.hkv * kKeys;
        rec.q_start = s_qo[b];
        rec.nq = s_qo[b + 1] - rec.q_start;
        rec.kvlen = s_lk[b];
        rec.page_base = s_ip[b];
        rec.off = p.causal ? rec.kvlen - rec.nq : INT32_MAX / 2;
        rec.i0 = p.window > 0 ? max(0, rec.nq - p.window) : 0;
        if (p.causal) rec.i0 = max(rec.i0, rec.j0 - rec.off);
        rec.n_tiles = rec.nq > rec.i0 ? cdiv(rec.nq - rec.i0, tq) : 0;
      }
      const int slot = it % kRecs;
      if (it >= kRecs && !__all_sync(0xffffffffu, mbar_wait_bounded(&it_empty[slot],
                                                                    (it / kRecs - 1) & 1))) {
        ok = false;
        break;
      }
      if (lane == 0) {
        recs[slot] = rec;
        mbar_arrive(&it_full[slot]);
      }
      if (rec.b < 0) break;
      if (rec.n_tiles == 0) continue;
      {  // the keys: 16-token boxes up to the request's end (a lane past it is not used)
        const int st = kc % kKStages;
        const int nch = min(8, cdiv(rec.kvlen - rec.j0, 16));
        const int c = lane / DH, dh = lane % DH;
        int page = -1;
        if (c < nch) page = p.indices[rec.page_base + (rec.j0 + c * 16) / p.ps];
        if (kc >= kKStages && !__all_sync(0xffffffffu, mbar_wait_bounded(&k_empty[st],
                                                                         (kc / kKStages - 1) & 1))) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&k_full[st], nch * DH * 2048);
        __syncwarp();
        if (c < nch) {
          // a bad page's keys load from page 0 (in bounds); their sums are not stored
          const bool bad = page < 0 || page >= p.num_pages;
          tma_load_4d(smem + L::K_OFF + st * L::K_BYTES + dh * (kKeys * 128) + c * 2048, &kvmap,
                      dh * 64, rec.h, (rec.j0 + c * 16) % p.ps, (bad ? 0 : page) * 2, &k_full[st],
                      pol_k);
          if (bad && dh == 0) flag(p.status, MI_STATUS_BAD_PAGE);
        }
        ++kc;
      }
      for (int t = 0; t < rec.n_tiles; ++t, ++qc) {
        const int st = qc % kQStages;
        if (qc >= kQStages && !__all_sync(0xffffffffu, mbar_wait_bounded(&q_empty[st],
                                                                         (qc / kQStages - 1) & 1))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[st], DH * m_used * 128);
          for (int dh = 0; dh < DH; ++dh)
            tma_load_3d(smem + L::Q_OFF + st * L::Q_BYTES + dh * (kRows * 128), &qmap, dh * 64,
                        rec.h * g, rec.q_start + rec.i0 + t * tq, &q_full[st], pol_q);
        }
      }
    }
    // no copy may be in flight when the CTA retires
    for (int t = max(0, kc - kKStages); t < kc; ++t)
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&k_full[t % kKStages], (t / kKStages) & 1)))
        ok = false;
    for (int t = max(0, qc - kQStages); t < qc; ++t)
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&q_full[t % kQStages], (t / kQStages) & 1)))
        ok = false;
  } else if (warp == 1) {
    // ============================ MMA issuer ====================================
    // The whole warp runs the loop and one elected lane issues: descriptors are
    // warp-uniform that way (a loop inside one lane's branch took 1250 clocks to
    // issue a tile's eight products of 64 clocks each).
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = umma_idesc(fmt, false, kRows, kKeys);
    const uint64_t kdesc0 = umma_desc(smem_u32(smem + L::K_OFF), 16, 1024);
    const uint64_t qdesc0 = umma_desc(smem_u32(smem + L::Q_OFF), 16, 1024);
    int kc = 0, gt = 0;
    for (int it = 0; ok; ++it) {
      const int slot = it % kRecs;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&it_full[slot], (it / kRecs) & 1))) {
        ok = false;
        break;
      }
      const int b = __shfl_sync(0xffffffffu, recs[slot].b, 0);
      const int n = __shfl_sync(0xffffffffu, recs[slot].n_tiles, 0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&it_empty[slot]);
      if (b < 0) break;
      if (n == 0) continue;
      const int ks = kc % kKStages;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&k_full[ks], (kc / kKStages) & 1))) {
        ok = false;
        break;
      }
      const uint64_t kd = kdesc0 + ((ks * L::K_BYTES) >> 4);
      for (int t = 0; t < n; ++t, ++gt) {
        const int st = gt % kQStages, acc = gt % kAcc;
        const bool ready = mbar_wait_bounded(&q_full[st], (gt / kQStages) & 1) &&
                           (gt < kAcc || mbar_wait_bounded(&s_free[acc], (gt / kAcc - 1) & 1));
        if (!__all_sync(0xffffffffu, ready)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t qd = qdesc0 + ((st * L::Q_BYTES) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t koff = (kk >> 2) * (kKeys * 128) + (kk & 3) * 32;
            const uint32_t qoff = (kk >> 2) * (kRows * 128) + (kk & 3) * 32;
            umma(tmem + acc * kRows, kd + (koff >> 4), qd + (qoff >> 4), idesc, kk > 0);
          }
          umma_commit(&s_full[acc]);
          umma_commit(&q_empty[st]);
          if (t + 1 == n) umma_commit(&k_empty[ks]);
        }
        __syncwarp();
      }
      if (!ok) break;
      ++kc;
    }
    // every product must land before TMEM is freed (the same lane is elected:
    // a commit tracks the issuing thread's earlier products)
    if (gt > 0) {
      if (elect_one()) umma_commit(drain);
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(drain, 0))) ok = false;
    }
  } else {
    // ============================ sums (warps 2..9) ==============================
    const int wg = (warp - 2) >> 2;  // group: every other tile
    const int qd = warp & 3;         // the TMEM lane quarter this warp may access
    const int key = qd * 32 + lane;
    float *lse_s = reinterpret_cast<float *>(smem + L::LSE_OFF) + (warp - 2) * 2 * kRows;
    // rows lane, lane + 32, ... of a tile: query token and head offset
    int rt[4];
    int64_t ro[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = lane + 32 * i;
      rt[i] = r < m_used ? r / g : INT32_MAX / 2;
      ro[i] = r < m_used ? static_cast<int64_t>(r / g) * p.hq + r % g : 0;
    }
    int gt = 0, buf = 0, done = 0;
    for (int it = 0; ok; ++it) {
      const int slot = it % kRecs;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&it_full[slot], (it / kRecs) & 1))) {
        ok = false;
        break;
      }
      const ScItem rec = recs[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&it_empty[slot]);
      if (rec.b < 0) break;
      if (rec.n_tiles == 0) continue;
      const int j = rec.j0 + key;
      // row terms of tile t: log-sum-exp in log2 units; +inf for rows that are
      // not there or saw nothing, which makes their exp2 zero
      float lv[4];
      auto load_lse = [&](int t) {
        const int tok = rec.i0 + t * tq;
        const float *l = p.lse + static_cast<int64_t>(rec.q_start + tok) * p.hq + rec.h * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lv[i] = INFINITY;
          if (rt[i] < rec.nq - tok) lv[i] = l[ro[i]];
        }
      };
      float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
      const int first = (gt & 1) == wg ? 0 : 1;  // tiles of this item that are this group's
      if (first < rec.n_tiles) load_lse(first);
      for (int t = first; t < rec.n_tiles; t += 2) {
        const int u = gt + t, acc = u % kAcc;
        float *ls = lse_s + buf * kRows;
        buf ^= 1;
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (used here, a turn after its load, which no use waits for)
          ls[lane + 32 * i] = lv[i] == -INFINITY ? INFINITY : lv[i] * kLog2e;
        __syncwarp();
        if (t + 2 < rec.n_tiles) load_lse(t + 2);
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&s_full[acc], (u / kAcc) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t ta = tmem + (static_cast<uint32_t>(qd * 32) << 16) + acc * kRows;
        const int tok = rec.i0 + t * tq;
        // columns of rows that are there and see this key: [cmin, cmax)
        const int cmax = min(tq, rec.nq - tok) * g;
        const int cmin = max(0, min(j - rec.off - tok, kRows)) * g;
        const bool full = __all_sync(0xffffffffu, cmin == 0 && cmax == m_used);
        const float4 *l4 = reinterpret_cast<const float4 *>(ls);
        float v[2][32];
        tmem_ld32(ta, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_wait_ld();
          if (c < 3) tmem_ld32(ta + (c + 1) * 32, v[(c + 1) & 1]);
          const float *x = v[c & 1];
          if (full) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = l4[c * 8 + i / 4];
              s0 += fast_exp2(fmaf(x[i], a.scale_log2, -l.x));
              s1 += fast_exp2(fmaf(x[i + 1], a.scale_log2, -l.y));
              s2 += fast_exp2(fmaf(x[i + 2], a.scale_log2, -l.z));
              s3 += fast_exp2(fmaf(x[i + 3], a.scale_log2, -l.w));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = l4[c * 8 + i / 4];
              const int col = c * 32 + i;
              const float e0 = fast_exp2(fmaf(x[i], a.scale_log2, -l.x));
              const float e1 = fast_exp2(fmaf(x[i + 1], a.scale_log2, -l.y));
              const float e2 = fast_exp2(fmaf(x[i + 2], a.scale_log2, -l.z));
              const float e3 = fast_exp2(fmaf(x[i + 3], a.scale_log2, -l.w));
              s0 += col >= cmin && col < cmax ? e0 : 0.f;
              s1 += col + 1 >= cmin && col + 1 < cmax ? e1 : 0.f;
              s2 += col + 2 >= cmin && col + 2 < cmax ? e2 : 0.f;
              s3 += col + 3 >= cmin && col + 3 < cmax ? e3 : 0.f;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[acc]);
      }
      if (!ok) break;
      gt += rec.n_tiles;
      const float s = (s0 + s1) + (s2 + s3);
      if (wg == 1) {  // hand this group's sums to the first
        if (done > 0 && !__all_sync(0xffffffffu, mbar_wait_bounded(&pt_free[qd], (done - 1) & 1))) {
          ok = false;
          break;
        }
        part[key] = s;
        __syncwarp();
        if (lane == 0) mbar_arrive(&pt_full[qd]);
      } else {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&pt_full[qd], done & 1))) {
          ok = false;
          break;
        }
        const float sum = s + part[key];
        __syncwarp();
        if (lane == 0) mbar_arrive(&pt_free[qd]);
        if (j < rec.kvlen) {
          const int64_t page = p.indices[rec.page_base + j / p.ps];
          if (page >= 0 && page < p.num_pages)
            asm volatile("red.global.add.f32 [%0], %1;" ::"l"(
                             p.scores + (page * p.hkv + rec.h) * p.ps + j % p.ps),
                         "f"(sum)
                         : "memory");
        }
      }
      ++done;
    }
  }
  if (!ok && lane == 0) flag(p.status, MI_STATUS_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  // the last CTA out resets the shared counters for the next launch
  if (threadIdx.x == 0 && a.ctr) {
    __threadfence();
    if (atomicAdd(a.ctr + 1, 1u) + 1u == gridDim.x) {
      a.ctr[0] = 0u;
      a.ctr[1] = 0u;
      __threadfence();
    }
  }
}

template <typename T, int D>
int launch_tc(const ScoreParams &p, int dtype, unsigned *ctr, cudaStream_t s) {
  using L = ScLayout<D>;
  CUtensorMap qmap, kvmap;
  if (!rows_tensor_map(p.q, p.total_q, p.hq, D, p.qsn, p.qsh, p.group, kRows / p.group, dtype,
                       &qmap) ||
      !pool_tensor_map(p.kv, p.num_pages, p.ps, p.hkv, D, dtype, &kvmap))
    return -1;
  static std::atomic<unsigned long long> attr_set{0};
  if (smem_limit_once(attr_set, scores_tc_kernel<T, D>, L::SMEM) != cudaSuccess)
    return check_launch("scores_tc_kernel smem attribute");
  const ScArgs a{p, p.scale * kLog2e, ctr};
  scores_tc_kernel<T, D><<<num_sms(), kScThreads, L::SMEM, s>>>(qmap, kvmap, a);
  return check_launch("scores_tc_kernel");
}

}  // namespace

int launch_scores_tc(const ScoreParams &p, int dtype, unsigned *ctr, cudaStream_t s) {
  if (!(dtype == MI_DTYPE_BF16 || dtype == MI_DTYPE_F16)) return -1;
  if (!(p.d == 64 || p.d == 128)) return -1;
  if (p.group > kRows || p.ps % 16 != 0 || p.batch > kScMaxBatch) return -1;
  if (p.num_pages * 2 > (1LL << 31) || (reinterpret_cast<uintptr_t>(p.kv) & 15)) return -1;
  if (static_cast<int64_t>(p.total_q) + 2 * kRows > (1LL << 31)) return -1;
  if (dtype == MI_DTYPE_BF16)
    return p.d == 128 ? launch_tc<__nv_bfloat16, 128>(p, dtype, ctr, s)
                      : launch_tc<__nv_bfloat16, 64>(p, dtype, ctr, s);
  return p.d == 128 ? launch_tc<__half, 128>(p, dtype, ctr, s)
                    : launch_tc<__half, 64>(p, dtype, ctr, s);
}

}  // namespace mi

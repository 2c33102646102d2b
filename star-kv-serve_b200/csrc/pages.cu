// Page bounds and page selection over a paged full-rank cache.
//
// bounds_kernel: per page and KV head the smallest and largest value of every key
// channel. It reads each key once and writes 2 D values per page; the read is the cost.
// A warp takes one (page, head), 16 bytes per lane, whole rows at a time.
//
// Selection: for each (sequence, KV head) the `top` pages of the highest score
//   score(page) = sum_{g in group} sum_d max(q[g, d] lo[d], q[g, d] hi[d])
//               = sum_d up[d] hi[d] + down[d] lo[d],
//   up = sum_g max(q[g], 0),  down = sum_g min(q[g], 0),
// an upper bound of sum_g q[g] . k over the page's keys. The second form is the definition
// where a bound is infinite: on a side of weight 0 it gives NaN, which ranks first, so that a
// page whose keys overflowed is read and not hidden. One page costs 4 D bytes and 2 D
// multiply-adds whatever G is, so the read of the bounds is the cost.
//
// The selection is that of scores summed in 64 bits (products of two 16-bit values are
// exact there, so the order of two pages next to the border does not depend on how a sum
// is split; 32-bit sums put about one of a thousand selections on the other side). 64-bit
// conversions run at an eighth of the rate that the reads need, so score_kernel sums in
// f32 and also bounds the error, and pick_kernel sums again in 64 bits only the pages
// that lie within the error of the border, mostly none. The bound covers products too
// small for f32; sums too large for it have no bound, and pick_kernel sums all pages again.
//
// score_kernel takes the batch's pages in runs of 16, an equal number of runs per CTA
// whatever the mix of lengths, and writes order-preserving keys. pick_kernel takes a CTA
// per (sequence, KV head) and finds the border by radix selection from the highest bit in
// which the unit's keys differ (one or two passes of 8 bits on real scores). Ties go to
// the lowest page. Few units of few pages: pick_kernel scores them itself (kFused).
#include <algorithm>
#include <type_traits>

#include "flat_items.cuh"
#include "starkv_common.cuh"
#include "starkv_kernels.h"

namespace starkv {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ uint32_t min2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t min2(__half, uint32_t a, uint32_t b) {
  const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(__half, uint32_t a, uint32_t b) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void to_f32x8(__nv_bfloat16, const uint4& u, float (&f)[8]) { bf16x8_to_f32(u, f); }
__device__ __forceinline__ void to_f32x8(__half, const uint4& u, float (&f)[8]) { f16x8_to_f32(u, f); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) bounds_kernel(const PageBoundsParams p) {
  constexpr int kChunks = D / 8, kRowsPer = 32 / kChunks;
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * kWarps + (threadIdx.x >> 5);   // 64-bit divisions would show
  const unsigned bp = item / p.num_kv_heads;
  const int hk = (int)(item - bp * p.num_kv_heads);
  const int b = (int)(bp / p.max_pages), j = (int)(bp - b * p.max_pages);
  if (b >= p.n) return;
  const int L = min(max(p.seq_lens[b], 0), p.max_len);
  const int fresh = p.new_lens ? min(max(p.new_lens[b], 0), p.max_new) : p.max_new;
  const int page = max(L - fresh, 0) / p.block_size + j;
  if (fresh == 0 || (int64_t)page * p.block_size >= L) return;
  const int blk = p.block_table[b * p.bt_s0 + page * p.bt_s1];
  if ((unsigned)blk >= (unsigned)p.num_blocks) {
    if (lane == 0) record_status(p.status, STARKV_EBOUNDS);
    return;
  }
  const int rows = min(p.block_size, L - page * p.block_size);
  const int chunk = lane % kChunks, sub = lane / kChunks;
  const T* k = reinterpret_cast<const T*>(p.k) + (int64_t)blk * p.k_s0 + (int64_t)hk * p.k_s2 + chunk * 8;
  const uint32_t pinf = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  uint32_t lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = pinf;
    hi[i] = pinf | 0x80008000u;
  }
  constexpr int kUnroll = 8;   // rows in flight per lane
  for (int r0 = sub; r0 < rows; r0 += kRowsPer * kUnroll) {
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = min(r0 + u * kRowsPer, rows - 1);   // past the end: the last row once more
      v[u] = *reinterpret_cast<const uint4*>(k + (int64_t)r * p.k_s1);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = min2(T{}, lo[i], w[i]);
        hi[i] = max2(T{}, hi[i], w[i]);
      }
    }
  }
#pragma unroll
  for (int o = kChunks; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = min2(T{}, lo[i], __shfl_xor_sync(~0u, lo[i], o));
      hi[i] = max2(T{}, hi[i], __shfl_xor_sync(~0u, hi[i], o));
    }
  T* out = reinterpret_cast<T*>(p.bounds) + (int64_t)blk * p.b_s0 + (int64_t)hk * p.b_s1 + chunk * 8;
  if (sub == 0) *reinterpret_cast<uint4*>(out) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  if (sub == 1) *reinterpret_cast<uint4*>(out + D) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
}

// Order of numbers as order of unsigned integers; -0 as +0, every NaN above all numbers.
__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return ~0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | (1u << 31);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
        "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return d;
}

// The larger magnitude of two pairs (its sign means nothing); a NaN loses.
__device__ __forceinline__ uint32_t max_abs2(__nv_bfloat16, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_abs2(__half, uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// up (upper) or down of channels d .. d + 7 of a KV head's queries. In few instructions,
// as pick_kernel's steps are: each kernel of a selection runs its code once per CTA, so the
// time of its straight parts is that of fetching them (f32 compares in place of the packed
// max: 7000 cycles instead of 1000 at the start of score_kernel).
template <typename T, typename W>
__device__ __forceinline__ void query_side(const T* q, int64_t stride, int group, bool upper, W (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 0;
  const uint32_t flip = upper ? 0u : 0x80008000u;
  for (int h0 = 0; h0 < group; h0 += 4) {   // four rows at once: one after another they are four latencies
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = h0 + u < group ? *reinterpret_cast<const uint4*>(q + (h0 + u) * stride) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint4 r = v[u];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t& x = (&r.x)[i];
        x = max2(T{}, x ^ flip, 0u) ^ flip;              // -max(-x, 0) = min(x, 0); a NaN stays one
      }
      float f[8];
      to_f32x8(T{}, r, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] += (W)f[i];
    }
  }
}

// Pages of sequence b, and how many of them compete: all but the kept ones, none where
// every page is taken.
__device__ __forceinline__ int pages_of(const SelectPagesParams& p, int b) {
  const int L = min(max(p.seq_lens[b], 0), p.max_len);
  return (int)(((unsigned)L + (unsigned)p.block_size - 1u) / (unsigned)p.block_size);   // L <= 2^30
}
__device__ __forceinline__ int competing(const SelectPagesParams& p, int pages) {
  return pages <= p.top || p.sinks + p.recent == p.top ? 0 : pages - p.sinks - p.recent;
}

constexpr int kRun = 16;     // pages of a run
constexpr uint32_t kGaveUp = ~0u;   // in the place of a run's error: a wait ran out, it has no scores
constexpr int kBatch = 32;   // block ids that a warp holds
constexpr int kStep = 4;     // pages of a lane's step
constexpr int kRing = 3;     // steps in the copies' ring
constexpr int ring_bytes(int threads) { return kRing * kStep * 16 * threads; }

// One step's scores of a warp: v holds 16 bytes of each of kStep pages. Returns the lane's
// page number within the step (of the sub-warp's kStep pages) in `at` and its score in s[0];
// lanes with (lane & mask) == 0 hold one page each.
template <typename T, int LP>
__device__ __forceinline__ float step_scores(const uint4 (&v)[kStep], const float (&w)[8], int lane, uint32_t& largest,
                                             int& at, int& mask) {
  float s[kStep];
#pragma unroll
  for (int u = 0; u < kStep; ++u) {
    float f[8];
    to_f32x8(T{}, v[u], f);
    float2 a = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) a = fma2(make_float2(f[2 * i], f[2 * i + 1]), make_float2(w[2 * i], w[2 * i + 1]), a);
    s[u] = a.x + a.y;
    largest = max_abs2(T{}, max_abs2(T{}, max_abs2(T{}, largest, v[u].x), v[u].y), max_abs2(T{}, v[u].z, v[u].w));
  }
  // sums over the LP lanes of a page: first steps that also halve the pages a lane holds
  at = 0;
  int o = LP / 2;
#pragma unroll
  for (int h = kStep / 2; h >= 1; h >>= 1, o >>= 1) {
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const float give = lane & o ? s[i] : s[i + h], keep = lane & o ? s[i + h] : s[i];
      s[i] = keep + __shfl_xor_sync(~0u, give, o);
    }
    at += lane & o ? h : 0;
  }
  mask = 2 * o - 1;                                  // lanes below: copies of the same page
#pragma unroll
  for (; o; o >>= 1) s[0] += __shfl_xor_sync(~0u, s[0], o);
  return s[0];
}

// Error of f32 scores: a term passes at most G - 1 roundings of 2^-24 in its weight (of
// terms of one sign), 5 in the lane and 5 between lanes, so (G + 9) 2^-24 sum |w b|
// <= (G + 9) 2^-24 sum_lanes largest * size (size: the lane's sum of |w|); 1.125 times
// (G + 11) covers the roundings of the bound itself. Below 2^-126 a product is off by up to
// 2^-150 instead, 256 of them by 2^-142: 2^-120 times the factor is more. 0 only where every
// term is one of zeros. INFINITY where a sum may have left f32's range (it is at most the
// sum of |w b|) or a factor is not finite: then the scores say nothing, NaN ones neither.
template <typename T>
__device__ __forceinline__ float score_error(uint32_t largest, float size, int group) {
  float f[8];
  to_f32x8(T{}, make_uint4(largest, 0, 0, 0), f);
  const float most = fmaxf(fabsf(f[0]), fabsf(f[1]));
  float err = most * size;
  if (most > 0.f && size > 0.f) err += 0x1p-120f;
#pragma unroll
  for (int o = 16; o; o >>= 1) err += __shfl_xor_sync(~0u, err, o);   // D = 64: both halves, an upper bound
  return err < 1e38f ? err * (1.125f / (1 << 24) * (group + 11)) : INFINITY;   // a NaN too
}

// Keys of the f32 scores of the competing pages i0 .. i1 - 1 of a (sequence, KV head), by one
// warp of a CTA of kThr threads, to keys[i]; returns the scores' error, and the smallest and
// the largest key.
template <typename T, int D, int kThr>
__device__ float score_pages(const SelectPagesParams& p, int b, int hk, int i0, int i1, uint8_t* ring, uint32_t* keys,
                             uint32_t& k_lo, uint32_t& k_hi) {
  constexpr int LP = 2 * D / 8;                      // lanes of one page's bounds
  constexpr int kPer = kStep * (32 / LP);            // pages of a warp's step
  constexpr int kSteps = kBatch / kPer;              // steps of a batch of block ids
  const int tid = threadIdx.x, lane = tid & 31;
  const int e = lane % LP, sub = lane / LP;
  const int d = (e * 8) % D;
  const bool upper = e * 8 >= D;
  const int steps = (i1 - i0 + kPer - 1) / kPer;
  const int32_t* bt = p.block_table + b * p.bt_s0 + (int64_t)p.sinks * p.bt_s1;
  const T* bounds = reinterpret_cast<const T*>(p.bounds) + (int64_t)hk * p.b_s1 + e * 8;
  // A lane copies its own 16 bytes of a page into its own slots of the ring (cp.async,
  // two steps ahead): no barrier between copy and use. Block ids come 32 at a time.
  const uint32_t slots = smem_u32(ring) + tid * 16;
  auto blocks_from = [&](int i) {   // lane l: the block of competing page i + l
    int blk = bt[(int64_t)min(i + lane, i1 - 1) * p.bt_s1];   // past the end: the last page once more
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      record_status(p.status, STARKV_EBOUNDS);
      blk = 0;
    }
    return blk;
  };
  int cur = 0, nxt = blocks_from(i0);
  auto issue = [&](int j) {
    if (j % kSteps == 0) {
      cur = nxt;
      nxt = blocks_from(i0 + (j / kSteps + 1) * kBatch);
    }
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      const int blk = __shfl_sync(~0u, cur, j % kSteps * kPer + sub * kStep + u);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slots + (j % kRing * kStep + u) * kThr * 16),
                   "l"(bounds + (int64_t)blk * p.b_s0)
                   : "memory");
    }
  };
  // the queries before the copies, so that they do not wait behind them
  float w[8];
  query_side(reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)(hk * p.group) * p.q_s1 + d, p.q_s1, p.group,
             upper, w);
  float size = 0.f;                                // sum of |w| of this lane's channels
#pragma unroll
  for (int i = 0; i < 8; ++i) size += fabsf(w[i]);
#pragma unroll
  for (int j = 0; j < kRing - 1; ++j) {
    if (j < steps) issue(j);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  k_lo = ~0u;
  k_hi = 0;
  uint32_t largest = 0;                            // largest |bound| of this lane's channels, as a pair
  for (int j = 0; j < steps; ++j) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    if (j + kRing - 1 < steps) issue(j + kRing - 1);   // into the slots of step j - 1
    asm volatile("cp.async.commit_group;" ::: "memory");
    uint4 v[kStep];
#pragma unroll
    for (int u = 0; u < kStep; ++u)
      v[u] = *reinterpret_cast<const uint4*>(ring + ((j % kRing * kStep + u) * kThr + tid) * 16);
    int at, mask;
    const float s = step_scores<T, LP>(v, w, lane, largest, at, mask);
    at += i0 + j * kPer + sub * kStep;
    if ((lane & mask) == 0 && at < i1) {
      const uint32_t k = order_key(s);
      keys[at] = k;
      k_lo = min(k_lo, k);
      k_hi = max(k_hi, k);
    }
  }
  const float err = score_error<T>(largest, size, p.group);
  k_lo = __reduce_min_sync(~0u, k_lo);
  k_hi = __reduce_max_sync(~0u, k_hi);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  return err;
}

// Bulk copy of `bytes` (a multiple of 16, both addresses on 16 bytes) counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The scores of a batch. A CTA takes the same pages of up to eight neighbouring KV heads (a
// consumer warp per head; fewer heads: the warps share a stage's pages), so that a page's
// bounds come in one piece: a producer warp brings pages as bulk copies into a ring of
// stages. 64 sequences to 32768 tokens, 8 heads: 52 us, 5.4 TB/s, of which 4.7 us pass before
// the first page is scored. (512-byte pieces, a warp's own head copied by its lanes:
// 56 us, whatever the depth and the occupancy.)
constexpr int kScoreThreads = kThreads + 32;
constexpr int kScoreStages = 6;
constexpr int kStageBytes = 16 * 1024;

struct ScoreCtl {
  uint64_t full[kScoreStages], empty[kScoreStages];
  int abort_flag;
};
constexpr int kScoreSmem = kScoreStages * kStageBytes + (int)sizeof(ScoreCtl);

template <typename T, int D>
__global__ void __launch_bounds__(kScoreThreads, 2) score_kernel(const SelectPagesParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int LP = 2 * D / 8;                      // lanes of one page's bounds
  constexpr int kPer = kStep * (32 / LP);            // pages of a warp's step
  constexpr int kRowBytes = 4 * D;                   // bounds of one page and head
  ScoreCtl* ctl = reinterpret_cast<ScoreCtl*>(smem + kScoreStages * kStageBytes);
  volatile int* abort_flag = &ctl->abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // pick_kernel waits for all of this one
  const int abreast = min(p.num_kv_heads, kWarps), groups = (p.num_kv_heads + abreast - 1) / abreast;
  const int parts = p.parts;                         // warps of one head
  const int span = parts * kPer;                     // pages of a stage: 4 .. 32, a power of two
  if (threadIdx.x == 0) {
    for (int s = 0; s < kScoreStages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], parts * abreast);
    }
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  const bool producer = warp == kWarps;
  if (!producer && warp >= parts * abreast) return;
  const auto count = [&](int b) { return (competing(p, pages_of(p, b)) + kRun - 1) / kRun * groups; };
  FlatItems<decltype(count)> all(count, p.n, lane);
  const int shares = min((int)gridDim.x, all.total), share = blockIdx.x;
  if (share >= shares) return;
  const int g1 = share_begin(all.total, share + 1, shares);
  int g = share_begin(all.total, share, shares);
  int b, first;
  all.place(g, b, first);
  int N = competing(p, pages_of(p, b)), runs = (N + kRun - 1) / kRun;
  int group = (g - first) / runs, run = (g - first) % runs;
  const bool side_by_side = p.b_s1 == 2 * D;
  const int e = lane % LP, sub = lane / LP;
  const int d = (e * 8) % D;
  int stage = 0, phase = 0, issued = 0;              // of the ring, through all segments
  bool ok = true;                                    // no wait of this warp has run out

  while (g < g1) {
    // the share's runs of this (sequence, group of KV heads)
    const int here = min(runs - run, g1 - g);
    const int i0 = run * kRun, i1 = min(i0 + here * kRun, N);   // competing pages i0 .. i1 - 1
    const int head0 = group * abreast, heads = min(abreast, p.num_kv_heads - head0);
    const int steps = (i1 - i0 + span - 1) / span;
    if (producer) {
      const int32_t* bt = p.block_table + b * p.bt_s0 + (int64_t)p.sinks * p.bt_s1;
      const T* bounds = reinterpret_cast<const T*>(p.bounds) + (int64_t)head0 * p.b_s1;
      auto blocks_from = [&](int i) {   // lane l: the block of competing page i + l
        int blk = bt[(int64_t)min(i + lane, i1 - 1) * p.bt_s1];
        if ((unsigned)blk >= (unsigned)p.num_blocks) {
          record_status(p.status, STARKV_EBOUNDS);
          blk = 0;
        }
        return blk;
      };
      int cur = 0, nxt = blocks_from(i0);
      for (int j = 0; j < steps && !p.stall; ++j) {
        const int at = j * span;                     // first page of the stage, from i0
        if (at % kBatch == 0) {
          cur = nxt;
          nxt = blocks_from(i0 + at + kBatch);
        }
        const int blk = __shfl_sync(~0u, cur, (at + lane) % kBatch);
        const int pages = min(span, i1 - i0 - at);
        ok = __all_sync(~0u, mbar_wait(&ctl->empty[stage], phase ^ 1, abort_flag, p.status));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&ctl->full[stage], pages * heads * kRowBytes);
        __syncwarp();
        ++issued;
        if (lane < pages) {
          uint8_t* dst = smem + stage * kStageBytes + lane * abreast * kRowBytes;
          const T* src = bounds + (int64_t)blk * p.b_s0;
          if (side_by_side) {
            bulk_load(dst, src, heads * kRowBytes, &ctl->full[stage]);
          } else {
            for (int h = 0; h < heads; ++h)
              bulk_load(dst + h * kRowBytes, src + h * p.b_s1, kRowBytes, &ctl->full[stage]);
          }
        }
        if (++stage == kScoreStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    } else {
      const int h = warp % abreast, part = warp / abreast;
      const int hk = min(head0 + h, p.num_kv_heads - 1);
      float w[8];
      query_side(reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)(hk * p.group) * p.q_s1 + d, p.q_s1, p.group,
                 e * 8 >= D, w);
      float size = 0.f;                              // sum of |w| of this lane's channels
#pragma unroll
      for (int i = 0; i < 8; ++i) size += fabsf(w[i]);
      uint32_t k_lo = ~0u, k_hi = 0, largest = 0;    // largest |bound| of this lane's channels, as a pair
      uint32_t* keys = p.keys + ((int64_t)b * p.num_kv_heads + hk) * p.key_stride + i0;
      for (int j = 0; ok && j < steps; ++j) {        // after a wait that ran out no stage is what it should be
        ok = __all_sync(~0u, mbar_wait(&ctl->full[stage], phase, abort_flag, p.status));
        if (!ok) break;
        const int first_page = part * kPer + sub * kStep;   // of the stage
        const int left = i1 - i0 - j * span;
        const uint8_t* src = smem + stage * kStageBytes + (first_page * abreast + h) * kRowBytes + e * 16;
        uint4 v[kStep];
#pragma unroll
        for (int u = 0; u < kStep; ++u)              // a page past the end, a head past the last: nothing was copied
          v[u] = first_page + u < left && h < heads ? *reinterpret_cast<const uint4*>(src + u * abreast * kRowBytes)
                                                    : make_uint4(0, 0, 0, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->empty[stage]);
        if (++stage == kScoreStages) {
          stage = 0;
          phase ^= 1;
        }
        int at, mask;
        const float s = step_scores<T, LP>(v, w, lane, largest, at, mask);
        at += first_page;
        if ((lane & mask) == 0 && at < left && h < heads) {
          const uint32_t k = order_key(s);
          keys[j * span + at] = k;
          k_lo = min(k_lo, k);
          k_hi = max(k_hi, k);
        }
      }
      const float err = score_error<T>(largest, size, p.group);
      k_lo = __reduce_min_sync(~0u, k_lo);
      k_hi = __reduce_max_sync(~0u, k_hi);
      // an entry per run and warp of the head, on every path: pick_kernel reads all of them
      uint4* about = p.runs + (((int64_t)b * p.num_kv_heads + hk) * p.run_stride + run) * parts + part;
      if (h < heads)
        for (int r = lane; r < here; r += 32) about[r * parts] = make_uint4(ok ? __float_as_uint(err) : kGaveUp, k_lo, k_hi, 0);
    }
    if (producer && !ok) break;
    g += here;
    run = 0;
    if (g < g1 && ++group == groups) {
      group = 0;
      do N = ++b < p.n ? competing(p, pages_of(p, b)) : 0;
      while (N == 0 && b < p.n);
      if (b >= p.n) break;   // not reached: g < g1 <= total
      runs = (N + kRun - 1) / kRun;
    }
  }
  if (producer) {   // no copy may land in shared memory that is no longer this CTA's, whoever gave up
    for (int k = max(0, issued - kScoreStages); k < issued; ++k)
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(&ctl->full[k % kScoreStages], (k / kScoreStages) & 1); ++i) {
      }
  }
}

constexpr int kPickWarpsMost = 32;
constexpr int kAhead = 4;         // keys in flight per thread
constexpr int kPickCache = 8192;  // keys that are copied to shared memory
constexpr int kFusedPages = 512, kFusedThreads = 512;   // pages that pick_kernel scores itself

constexpr int kBins = 2048;
constexpr int kNear = 256;        // pages next to the border that are scored again one by one

struct PickShared {
  union {
    uint32_t hist[256];
    uint4 bins[kBins / 4];
  };
  uint64_t lo[kPickWarpsMost], hi[kPickWarpsMost];
  uint32_t scan[8], found[3];                 // bin, still needed in it, its count
  uint32_t sure[256], tied[256];                     // 32 pages a word
  int gt[8], eq[8];
  int above, near;
  uint32_t in, off;
  int near_page[kNear];
  uint64_t near_key[kNear];
  double side[256];                                  // query_side of the 2 D channels of a page's bounds
};

// The border of the `rest` largest of N > rest keys, all between k_lo and k_hi: those with
// key >> shift > border and, lowest index first, `rest` (as it comes back) of the `level`
// ones with key >> shift == border.
template <int kThr, typename K>
__device__ void find_border(const K* keys, int N, K k_lo, K k_hi, PickShared& sh, int& shift, K& border, int& rest,
                            int& level) {
  constexpr int kBits = sizeof(K) * 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 256) sh.hist[tid] = 0;
  __syncthreads();
  const int top_bit = k_lo == k_hi ? -1 : 63 - __clzll((long long)(k_lo ^ k_hi));
  shift = top_bit + 1;                               // bits above are the same in all keys
  border = shift >= kBits ? 0 : k_lo >> shift;
  level = N;
  while (shift > 0) {
    const int bits = min(8, shift), ns = shift - bits;
    for (int i = tid; i < N; i += kAhead * kThr) {
      K k[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) k[u] = keys[min(i + u * kThr, N - 1)];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * kThr < N && (shift >= kBits || (k[u] >> shift) == border))
          atomicAdd(&sh.hist[(uint32_t)(k[u] >> ns) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins from the highest down: thread t < 256 has bin 255 - t
    uint32_t mine = 0, incl = 0;
    if (warp < 8) {
      mine = incl = sh.hist[255 - tid];
      sh.hist[255 - tid] = 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sh.scan[warp] = incl;
    }
    __syncthreads();
    if (warp < 8) {
      for (int w = 0; w < warp; ++w) incl += sh.scan[w];
      if (incl >= (uint32_t)rest && incl - mine < (uint32_t)rest) {
        sh.found[0] = 255 - (uint32_t)tid;
        sh.found[1] = (uint32_t)rest - (incl - mine);
        sh.found[2] = mine;
      }
    }
    __syncthreads();
    border = (K)(border << bits) | (K)sh.found[0];
    rest = (int)sh.found[1];
    level = (int)sh.found[2];
    shift = ns;
    if (level == rest) break;                        // the whole bin is selected
  }
  __syncthreads();                                   // sh may be written again
}

// Writes the selected ones of N pages in ascending order, as base + index. cls(i): 1 for a
// selected page, 2 for one of those of which the first `rest` are selected, else 0. All
// threads; 8192 pages a round: a bit per page by ballots, then a thread per 32 pages.
template <int kThr, class Cls>
__device__ void write_selected(int N, PickShared& sh, const Cls& cls, int rest, int32_t* out, int base) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int gt0 = 0, eq0 = 0;                              // of the rounds before
  for (int r0 = 0; r0 < N; r0 += 32 * 256) {
    const int words = min(256, (N - r0 + 31) / 32);
#pragma unroll 1
    for (int w = warp; w < words; w += kThr / 32) {
      const int i = r0 + w * 32 + lane;
      const int c = i < N ? cls(i) : 0;
      const uint32_t g = __ballot_sync(~0u, c == 1), e = __ballot_sync(~0u, c == 2);
      if (lane == 0) {
        sh.sure[w] = g;
        sh.tied[w] = e;
      }
    }
    __syncthreads();
    uint32_t g = tid < words ? sh.sure[tid] : 0, e = tid < words ? sh.tied[tid] : 0;
    int gt = __popc(g), eq = __popc(e);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, gt, o), y = __shfl_up_sync(~0u, eq, o);
      if (lane >= o) {
        gt += x;
        eq += y;
      }
    }
    if (lane == 31 && warp < 8) {
      sh.gt[warp] = gt;
      sh.eq[warp] = eq;
    }
    __syncthreads();
    const int gt_w = lane < 8 ? sh.gt[lane] : 0, eq_w = lane < 8 ? sh.eq[lane] : 0;
    // before this thread's pages
    gt += gt0 - __popc(g) + __reduce_add_sync(~0u, lane < warp ? gt_w : 0);
    eq += eq0 - __popc(e) + __reduce_add_sync(~0u, lane < warp ? eq_w : 0);
    for (uint32_t m = g | e; m; m &= m - 1) {
      const uint32_t bit = m & -m;
      if (g & bit) out[gt++ + min(eq, rest)] = base + r0 + tid * 32 + __ffs(bit) - 1;
      else if (eq++ < rest) out[gt + eq - 1] = base + r0 + tid * 32 + __ffs(bit) - 1;
    }
    gt0 += __reduce_add_sync(~0u, gt_w);
    eq0 += __reduce_add_sync(~0u, eq_w);
    __syncthreads();
  }
}

// kFused: it scores the unit's pages itself (launch_select_typed says when).
// kThr: 256 threads where the units fill the GPU (four CTAs to an SM), 1024 where they do
// not and a unit's passes over many keys are the time (8192 pages: 20.9 -> 13.2 us).
template <typename T, int D, int kThr, bool kFused>
__global__ void __launch_bounds__(kThr, 1024 / kThr) pick_kernel(const SelectPagesParams p) {
  __shared__ PickShared sh;
  constexpr int kCache = kFused ? kFusedPages : kPickCache;
  __shared__ uint32_t cache[kCache];
  const int unit = blockIdx.x;
  const int hk = unit % p.num_kv_heads, b = unit / p.num_kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = pages_of(p, b), N = competing(p, P);
  // the attention over the lists may take the place of CTAs that are done; it waits for all
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int32_t* out = p.pages + b * p.pg_s0 + hk * p.pg_s1;
  if (P <= p.top) {   // every page, then -1
    for (int i = tid; i < p.top; i += kThr) out[i] = i < P ? i : -1;
  } else {
    for (int i = tid; i < p.sinks; i += kThr) out[i] = i;
    for (int i = tid; i < p.recent; i += kThr) out[p.top - p.recent + i] = P - p.recent + i;
  }
  constexpr int LP = 2 * D / 8;
  // for the scores in 64 bits, should there be any: before the wait it costs nothing, and the
  // last warp has the fewest pages to score
  if (N > 0 && warp == (kFused ? kThr / 32 - 1 : 0)) {
    const int d = (lane % LP * 8) % D;
    double w[8];
    query_side(reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)(hk * p.group) * p.q_s1 + d, p.q_s1, p.group,
               lane % LP * 8 >= D, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sh.side[lane % LP * 8 + i] = w[i];
  }
  for (int i = tid; i < kBins / 4; i += kThr) sh.bins[i] = make_uint4(0, 0, 0, 0);
  // keys of the scores, their largest error, smallest and largest key
  uint32_t* keys = p.keys + (int64_t)unit * p.key_stride;
  uint32_t k_lo = ~0u, k_hi = 0, e_bits = 0;
  if (kFused) {   // launched behind all earlier work, N <= kFusedPages
    extern __shared__ __align__(16) uint8_t ring[];
    if (N == 0) return;
    keys = cache;
    const int per = ((N + kThr / 32 - 1) / (kThr / 32) + 7) & ~7;
    if (warp * per < N)
      e_bits = __float_as_uint(score_pages<T, D, kThr>(p, b, hk, warp * per, min((warp + 1) * per, N), ring, cache, k_lo,
                                                       k_hi));
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the scores are written
    if (N == 0) return;
    const uint4* runs = p.runs + (int64_t)unit * p.run_stride * p.parts;
    const int n_runs = (N + kRun - 1) / kRun * p.parts;
    uint4 about = runs[min(tid, n_runs - 1)];
    if (N <= kCache) {
      for (int i = tid; i < N; i += 2 * kAhead * kThr) {
        uint32_t k[2 * kAhead];
#pragma unroll
        for (int u = 0; u < 2 * kAhead; ++u) k[u] = keys[min(i + u * kThr, N - 1)];
#pragma unroll
        for (int u = 0; u < 2 * kAhead; ++u)
          if (i + u * kThr < N) cache[i + u * kThr] = k[u];
      }
      keys = cache;
    }
    for (int r = tid;;) {
      e_bits = max(e_bits, about.x);                 // >= 0: ordered as integers
      k_lo = min(k_lo, about.y);
      k_hi = max(k_hi, about.z);
      if ((r += kThr) >= n_runs) break;
      about = runs[r];
    }
  }
  out += p.sinks;
  e_bits = __reduce_max_sync(~0u, e_bits);
  k_lo = __reduce_min_sync(~0u, k_lo);
  k_hi = __reduce_max_sync(~0u, k_hi);
  if (lane == 0) {
    sh.lo[warp] = (uint64_t)k_lo << 32 | e_bits;
    sh.hi[warp] = k_hi;
  }
  if (tid == 0) {
    sh.above = sh.near = 0;
    sh.in = ~0u;
    sh.off = 0;
  }
  __syncthreads();
  {
    const int w = min(lane, kThr / 32 - 1);
    e_bits = __reduce_max_sync(~0u, (uint32_t)sh.lo[w]);
    k_lo = __reduce_min_sync(~0u, (uint32_t)(sh.lo[w] >> 32));
    k_hi = __reduce_max_sync(~0u, (uint32_t)sh.hi[w]);
  }
  if (!kFused && e_bits == kGaveUp) {                // the same for the whole CTA: a list of no pages
    for (int i = tid; i < p.top; i += kThr) out[i - p.sinks] = -1;
    return;
  }
  const int need = p.top - p.sinks - p.recent;       // < N
  const float err = __uint_as_float(e_bits), reach = 2.01f * err;

  const int e = lane % LP;
  const int32_t* bt = p.block_table + b * p.bt_s0 + (int64_t)p.sinks * p.bt_s1;
  const T* bounds = reinterpret_cast<const T*>(p.bounds) + (int64_t)hk * p.b_s1 + e * 8;
  const auto score = [&](int i) {                    // in 64 bits, by a whole warp
    int blk = bt[(int64_t)i * p.bt_s1];
    if ((unsigned)blk >= (unsigned)p.num_blocks) blk = 0;   // recorded by score_kernel
    float f[8];
    to_f32x8(T{}, *reinterpret_cast<const uint4*>(bounds + (int64_t)blk * p.b_s0), f);
    double x = 0.0;
#pragma unroll
    for (int c = 0; c < 8; ++c) x = fma((double)f[c], sh.side[e * 8 + c], x);
#pragma unroll
    for (int o = LP / 2; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return order_key(x);
  };
  // Lists the pages with near_lo <= key <= near_hi (the first kNear) and counts those above.
  const auto list_near = [&](uint32_t near_lo, uint32_t near_hi) {
    for (int i0 = warp * 32; i0 < N; i0 += kThr) {
      const uint32_t k = i0 + lane < N ? keys[i0 + lane] : 0;
      const int up = __popc(__ballot_sync(~0u, i0 + lane < N && k > near_hi));
      if (lane == 0 && up) atomicAdd(&sh.above, up);
      if (i0 + lane < N && k >= near_lo && k <= near_hi) {
        const int c = atomicAdd(&sh.near, 1);
        if (c < kNear) sh.near_page[c] = i0 + lane;
      }
    }
    __syncthreads();
  };
  // How many of the listed pages come before listed page `tid`.
  const auto better = [&](int near, uint64_t mine) {
    const int page = sh.near_page[tid];
    int n = 0;
    for (int c = 0; c < near; ++c)
      n += sh.near_key[c] > mine || (sh.near_key[c] == mine && sh.near_page[c] < page);
    return n;
  };
  // The open ones of the listed pages by 64-bit scores; their keys become the largest, those
  // of the others the smallest (the scratch or its copy: this CTA's own).
  const auto settle = [&](int near, int open) {
    for (int c = warp; c < near; c += kThr / 32) {
      const uint64_t k = score(sh.near_page[c]);
      if (lane == 0) sh.near_key[c] = k;
    }
    __syncthreads();
    if (tid < near) keys[sh.near_page[tid]] = better(near, sh.near_key[tid]) < open ? ~0u : 0;
    __syncthreads();
  };

  // ---- ordinary scores: one histogram of 2048 equal parts of the keys' range, then the few
  // pages of the border's part, and those within reach of it, one by one ----
  if (N <= kCache && k_hi < ~0u && reach < INFINITY) {
    uint32_t* bins = reinterpret_cast<uint32_t*>(sh.bins);
    const int s = max(0, 21 - __clz(k_hi - k_lo));   // (k_hi - k_lo) >> s < 2048
    for (int i = tid; i < N; i += kThr) atomicAdd(&bins[(keys[i] - k_lo) >> s], 1u);
    __syncthreads();
    // from the highest bin down, eight bins to each of 256 threads
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (warp < 8) {
      x = sh.bins[kBins / 4 - 1 - 2 * tid];
      y = sh.bins[kBins / 4 - 2 - 2 * tid];
    }
    const uint32_t mine = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31 && warp < 8) sh.scan[warp] = incl;
    __syncthreads();
    incl += __reduce_add_sync(~0u, lane < min(warp, 8) ? sh.scan[lane] : 0u);
    if (warp < 8 && incl >= (uint32_t)need && incl - mine < (uint32_t)need) {
      const uint32_t c[8] = {x.w, x.z, x.y, x.x, y.w, y.z, y.y, y.x};
      uint32_t sum = incl - mine;
      int j = 0;
#pragma unroll
      for (int u = 0; u < 7; ++u) {
        sum += c[u];
        j += sum < (uint32_t)need;
      }
      sh.found[0] = kBins - 1 - 8 * tid - j;
    }
    __syncthreads();
    const uint32_t first = k_lo + (sh.found[0] << s), last = first + ((1u << s) - 1);
    const uint32_t near_lo = max(order_key(key_value(first) - reach), 1u) - 1;
    const uint32_t near_hi = min(order_key(key_value(min(last, k_hi)) + reach), ~0u - 2) + 1;
    list_near(near_lo, near_hi);
    const int near = sh.near, open = need - sh.above;
    if (near <= kNear) {
      bool chosen = false;
      if (tid < near) sh.near_key[tid] = keys[sh.near_page[tid]];
      __syncthreads();
      if (tid < near) {
        chosen = better(near, sh.near_key[tid]) < open;
        if (chosen) atomicMin(&sh.in, (uint32_t)sh.near_key[tid]);
        else atomicMax(&sh.off, (uint32_t)sh.near_key[tid]);
      }
      __syncthreads();
      if (near == open || err == 0.f || key_value(sh.in) - key_value(sh.off) > reach) {
        if (tid < near) keys[sh.near_page[tid]] = chosen ? ~0u : 0;
        __syncthreads();
      } else {
        settle(near, open);
      }
      write_selected<kThr>(N, sh, [&](int i) { return keys[i] > near_hi ? 1 : 0; }, 0, out, p.sinks);
      return;
    }
    __syncthreads();
    if (tid == 0) sh.above = sh.near = 0;
    __syncthreads();
  }

  // ---- long units, many equal scores, infinities: the border by radix selection; the keys
  // >= border are selected, all of them or, lowest index first, `rest` of the equal ones ----
  int shift, rest = need, level;
  uint32_t border;
  find_border<kThr>(keys, N, k_lo, k_hi, sh, shift, border, rest, level);
  const bool whole = level == rest;
  border = shift < 32 ? border << shift : 0;
  // the scores next to the border on both sides
  uint32_t in = ~0u, off = 0;
  for (int i = tid; i < N; i += kThr) {
    const uint32_t k = keys[i];
    if (k >= border) in = min(in, k);
    else off = max(off, k);
  }
  in = __reduce_min_sync(~0u, in);
  off = __reduce_max_sync(~0u, off);
  if (lane == 0) {
    sh.lo[warp] = in;
    sh.hi[warp] = off;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThr / 32; ++w) {
    in = min(in, (uint32_t)sh.lo[w]);
    off = max(off, (uint32_t)sh.hi[w]);
  }
  // the border lies among NaN scores: all the same, if the scores are to be believed
  const bool nan = in == ~0u && reach < INFINITY;
  const float at = key_value(in);
  // sure: every selected score is further above every other than the error can move them
  if (err == 0.f || nan || (whole && at - key_value(off) > reach)) {
    write_selected<kThr>(N, sh, [&](int i) {
      const uint32_t k = keys[i];
      return k > border || (whole && k == border) ? 1 : k == border ? 2 : 0;
    }, rest, out, p.sinks);
    return;
  }

  // 64-bit scores of the pages within reach of the border; above it all are selected,
  // below it none. No bound of the error: of every page, the keys of NaN scores among them.
  uint32_t near_lo = 0, near_hi = ~0u - 1;
  if (reach < INFINITY) {
    near_lo = max(order_key(at - reach), 1u) - 1;
    near_hi = min(order_key(at + reach), ~0u - 2) + 1;
  } else {
    for (int i = tid; i < N; i += kThr) keys[i] = min(keys[i], near_hi);
    __syncthreads();
  }
  list_near(near_lo, near_hi);
  const int near = sh.near, open = need - sh.above;  // pages to be told apart, and how many of them are selected
  if (near <= kNear) {
    settle(near, open);
    write_selected<kThr>(N, sh, [&](int i) { return keys[i] > near_hi ? 1 : 0; }, 0, out, p.sinks);
    return;
  }
  // many of them (equal pages, or no usable error): all keys in 64 bits
  uint64_t* exact = p.exact + (int64_t)unit * p.key_stride;
  uint64_t lo64 = ~0ull, hi64 = 0;
  for (int i0 = warp * 32; i0 < N; i0 += kThr) {
    const uint32_t k = i0 + lane < N ? keys[i0 + lane] : 0;
    uint64_t x = k > near_hi ? ~0ull : 0;
    for (uint32_t m = __ballot_sync(~0u, i0 + lane < N && k >= near_lo && k <= near_hi); m; m &= m - 1) {
      const uint64_t y = score(i0 + __ffs(m) - 1);
      if (lane == __ffs(m) - 1) x = y;
    }
    if (i0 + lane < N) {
      exact[i0 + lane] = x;
      lo64 = min(lo64, x);
      hi64 = max(hi64, x);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo64 = min(lo64, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)lo64, o));
    hi64 = max(hi64, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)hi64, o));
  }
  if (lane == 0) {
    sh.lo[warp] = lo64;
    sh.hi[warp] = hi64;
  }
  __syncthreads();                                   // also orders this CTA's writes of `exact` before its reads
#pragma unroll
  for (int v = 0; v < kThr / 32; ++v) {
    lo64 = min(lo64, sh.lo[v]);
    hi64 = max(hi64, sh.hi[v]);
  }
  uint64_t border64;
  rest = need;
  find_border<kThr>(exact, N, lo64, hi64, sh, shift, border64, rest, level);
  write_selected<kThr>(N, sh, [&](int i) {
    const uint64_t k = exact[i] >> shift;
    return k > border64 ? 1 : k == border64 ? 2 : 0;
  }, rest, out, p.sinks);
}

template <typename T, int D>
int launch_select_typed(SelectPagesParams p, int num_sms, cudaStream_t stream) {
  const int64_t units = (int64_t)p.n * p.num_kv_heads;
  p.run_stride = (p.key_stride + kRun - 1) / kRun;
  p.parts = std::min(kWarps / std::min(p.num_kv_heads, kWarps), 32 / (kStep * (128 / D)));
  if (units * p.run_stride > 0x7fffffff) return STARKV_EINVAL;   // 32-bit run numbers
  p.runs = reinterpret_cast<uint4*>(p.scratch);
  p.exact = reinterpret_cast<uint64_t*>(p.runs + units * p.run_stride * p.parts);
  p.keys = reinterpret_cast<uint32_t*>(p.exact + units * p.key_stride);
  void* args[] = {&p};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)units);
  cfg.stream = stream;
  cfg.attrs = attr;
  // One kernel where a CTA per unit, one to an SM, is enough for the reads. Its time grows
  // with the pages of a unit, that of two kernels with all pages: 8 units of 128 / 375 / 512
  // / 1024 pages 7.2 / 8.9 / 11.5 / 15.8 us against 9.4 / 9.1 / 10.3 / 10.0 in two; 128 units
  // of 256 / 512 pages 9.3 / 11.5 against 12.2 / 15.0. The launch less is 4 us of the host's.
  if (units <= num_sms && p.key_stride <= kFusedPages) {
    const void* fn = (const void*)pick_kernel<T, D, kFusedThreads, true>;
    if (const int st = allow_smem(fn, ring_bytes(kFusedThreads))) return st;
    cfg.blockDim = dim3(kFusedThreads);
    cfg.dynamicSmemBytes = ring_bytes(kFusedThreads);
    return cudaLaunchKernelExC(&cfg, fn, args) == cudaSuccess ? STARKV_OK : STARKV_ECUDA;
  }
  if (p.key_stride > p.top) {   // else no sequence has pages to choose from
    const void* fn = (const void*)score_kernel<T, D>;
    if (const int st = allow_smem(fn, kScoreSmem)) return st;
    const int64_t grid = std::min<int64_t>(2 * num_sms, units * p.run_stride);
    if (cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kScoreThreads), args, kScoreSmem, stream) != cudaSuccess)
      return STARKV_ECUDA;
  }
  const bool few = units <= num_sms && p.key_stride > 1024;
  cfg.blockDim = dim3(few ? 1024 : 256);
  cfg.numAttrs = p.key_stride > p.top;   // behind score_kernel alone may the launch come early
  const void* pick = few ? (const void*)pick_kernel<T, D, 1024, false> : (const void*)pick_kernel<T, D, 256, false>;
  return cudaLaunchKernelExC(&cfg, pick, args) == cudaSuccess ? STARKV_OK : STARKV_ECUDA;
}

template <typename T, int D>
int launch_bounds_typed(PageBoundsParams p, cudaStream_t stream) {
  const int64_t items = (int64_t)p.n * p.max_pages * p.num_kv_heads;
  const int64_t blocks = (items + kWarps - 1) / kWarps;
  if (items > 0x7fffffff) return STARKV_EINVAL;
  void* args[] = {&p};
  return cudaLaunchKernel((const void*)bounds_kernel<T, D>, dim3((unsigned)blocks), dim3(kThreads), args, 0, stream) ==
                 cudaSuccess
             ? STARKV_OK
             : STARKV_ECUDA;
}

}  // namespace

size_t select_scratch_bytes(int64_t units, int64_t pages) {
  return (size_t)units * (pages * 12 + (pages + kRun - 1) / kRun * 16 * kWarps);   // at most kWarps entries a run
}

int launch_page_bounds(const PageBoundsParams& p, int dtype, int head_dim, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_bounds_typed<__nv_bfloat16, 64>(p, stream)
                          : launch_bounds_typed<__nv_bfloat16, 128>(p, stream);
  return head_dim == 64 ? launch_bounds_typed<__half, 64>(p, stream) : launch_bounds_typed<__half, 128>(p, stream);
}

int launch_select_pages(SelectPagesParams p, int dtype, int head_dim, int num_sms, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_select_typed<__nv_bfloat16, 64>(p, num_sms, stream)
                          : launch_select_typed<__nv_bfloat16, 128>(p, num_sms, stream);
  return head_dim == 64 ? launch_select_typed<__half, 64>(p, num_sms, stream)
                        : launch_select_typed<__half, 128>(p, num_sms, stream);
}

}  // namespace starkv

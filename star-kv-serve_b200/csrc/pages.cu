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
// an upper bound of sum_g q[g] . k over the page's keys. One page costs 4 D bytes and 2 D
// multiply-adds whatever G is, so the read of the bounds is the cost. Scores are summed
// in 64 bits: the products of two 16-bit values are exact there and the order of two
// pages next to the border does not depend on how the sum was split (32-bit sums put
// about one of a thousand selections on the other side).
//
// score_kernel takes the batch's pages in runs of 32, an equal number of runs per warp
// whatever the mix of lengths, and writes order-preserving 64-bit keys. pick_kernel takes
// a CTA per (sequence, KV head) and finds the border by radix selection from the highest
// bit in which the unit's keys differ (one or two passes of 8 bits on real scores). Ties
// go to the lowest page.
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
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int hk = (int)(item % p.num_kv_heads);
  const int64_t bp = item / p.num_kv_heads;
  const int b = (int)(bp / p.max_pages), j = (int)(bp % p.max_pages);
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

// Order of doubles as order of unsigned integers; -0 as +0, every NaN above all numbers.
__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Pages of sequence b, and how many of them compete: all but the kept ones, none where
// every page is taken.
__device__ __forceinline__ int pages_of(const SelectPagesParams& p, int b) {
  const int L = min(max(p.seq_lens[b], 0), p.max_len);
  return (int)(((int64_t)L + p.block_size - 1) / p.block_size);
}
__device__ __forceinline__ int competing(const SelectPagesParams& p, int pages) {
  return pages <= p.top || p.sinks + p.recent == p.top ? 0 : pages - p.sinks - p.recent;
}

constexpr int kRun = 32;     // pages of a run
constexpr int kStep = 4;     // pages of a lane's step
constexpr int kRing = 3;     // steps in the copies' ring
constexpr int kRingBytes = kRing * kStep * 16 * kThreads;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 3) score_kernel(const SelectPagesParams p) {
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int LP = 2 * D / 8;                      // lanes of one page's bounds
  constexpr int kPer = kStep * (32 / LP);            // pages of a warp's step
  constexpr int kSteps = kRun / kPer;                // steps of a run
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int e = lane % LP, sub = lane / LP;
  const int d = (e * 8) % D;
  const bool upper = e * 8 >= D;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // pick_kernel waits for all of this one
  const auto count = [&](int b) { return (competing(p, pages_of(p, b)) + kRun - 1) / kRun * p.num_kv_heads; };
  FlatItems<decltype(count)> all(count, p.n, lane);
  const int shares = min((int)gridDim.x * kWarps, all.total);
  const int share = blockIdx.x + warp * gridDim.x;   // a warp of every CTA before the second of one
  if (share >= shares) return;
  const int g1 = share_begin(all.total, share + 1, shares);
  int g = share_begin(all.total, share, shares);
  int b, first;
  all.place(g, b, first);
  int N = competing(p, pages_of(p, b)), runs = (N + kRun - 1) / kRun;
  int hk = (g - first) / runs, run = (g - first) % runs;

  while (g < g1) {
    // the share's runs of this (sequence, KV head)
    const int here = min(runs - run, g1 - g);
    const int i0 = run * kRun, i1 = min(i0 + here * kRun, N);   // competing pages i0 .. i1 - 1
    const int steps = (i1 - i0 + kPer - 1) / kPer;
    const int32_t* bt = p.block_table + b * p.bt_s0 + (int64_t)p.sinks * p.bt_s1;
    const T* bounds = reinterpret_cast<const T*>(p.bounds) + (int64_t)hk * p.b_s1 + e * 8;
    // A lane copies its own 16 bytes of a page into its own slots of the ring (cp.async,
    // two steps ahead): no barrier between copy and use. Block ids come 32 at a time.
    const uint32_t slots = smem_u32(ring) + tid * 16;
    auto blocks_from = [&](int i) {   // lane l: the block of competing page i + l
      if (i + lane >= i1) return 0;
      int blk = bt[(int64_t)(i + lane) * p.bt_s1];
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
        nxt = blocks_from(i0 + (j / kSteps + 1) * kRun);
      }
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const int blk = __shfl_sync(~0u, cur, j % kSteps * kPer + sub * kStep + u);   // a page past the end: block 0
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slots + (j % kRing * kStep + u) * kThreads * 16),
                     "l"(bounds + (int64_t)blk * p.b_s0)
                     : "memory");
      }
    };
    issue(0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (steps > 1) issue(1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    double w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0.0;
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)(hk * p.group) * p.q_s1 + d;
#pragma unroll 4
    for (int h = 0; h < p.group; ++h) {
      float f[8];
      to_f32x8(T{}, *reinterpret_cast<const uint4*>(q + h * p.q_s1), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] += (double)(upper ? (f[i] < 0.f ? 0.f : f[i]) : (f[i] > 0.f ? 0.f : f[i]));
    }
    uint64_t* keys = p.keys + ((int64_t)b * p.num_kv_heads + hk) * p.key_stride + i0;
    for (int j = 0; j < steps; ++j) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      double s[kStep];
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const uint4 v = *reinterpret_cast<const uint4*>(ring + ((j % kRing * kStep + u) * kThreads + tid) * 16);
        float f[8];
        to_f32x8(T{}, v, f);
        s[u] = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[u] = fma((double)f[i], w[i], s[u]);
      }
      if (j + 2 < steps) issue(j + 2);   // into the slots of step j - 1
      asm volatile("cp.async.commit_group;" ::: "memory");
      // sums over the LP lanes of a page: first steps that also halve the pages a lane holds
      int at = j * kPer + sub * kStep, o = LP / 2;
#pragma unroll
      for (int h = kStep / 2; h >= 1; h >>= 1, o >>= 1) {
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const double give = lane & o ? s[i] : s[i + h], keep = lane & o ? s[i + h] : s[i];
          s[i] = keep + __shfl_xor_sync(~0u, give, o);
        }
        at += lane & o ? h : 0;
      }
      const int last = o;                            // lanes below: copies of the same page
#pragma unroll
      for (; o; o >>= 1) s[0] += __shfl_xor_sync(~0u, s[0], o);
      if ((lane & (2 * last - 1)) == 0 && i0 + at < i1) keys[at] = order_key(s[0]);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    g += here;
    run = 0;
    if (g < g1 && ++hk == p.num_kv_heads) {
      hk = 0;
      do N = ++b < p.n ? competing(p, pages_of(p, b)) : 0;
      while (N == 0 && b < p.n);
      if (b >= p.n) break;   // not reached: g < g1 <= total
      runs = (N + kRun - 1) / kRun;
    }
  }
}

constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32;

__global__ void __launch_bounds__(kPickThreads) pick_kernel(const SelectPagesParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint64_t warp_lo[kPickWarps], warp_hi[kPickWarps];
  __shared__ uint32_t scan[8], found[3];             // bin, still needed in it, its count
  __shared__ int n_gt[kPickWarps], n_eq[kPickWarps];
  const int unit = blockIdx.x;
  const int hk = unit % p.num_kv_heads, b = unit / p.num_kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = pages_of(p, b), N = competing(p, P);
  // the attention over the lists may take the place of CTAs that are done; it waits for all
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int32_t* out = p.pages + b * p.pg_s0 + hk * p.pg_s1;
  if (P <= p.top) {   // every page, then -1
    for (int i = tid; i < p.top; i += kPickThreads) out[i] = i < P ? i : -1;
  } else {
    for (int i = tid; i < p.sinks; i += kPickThreads) out[i] = i;
    for (int i = tid; i < p.recent; i += kPickThreads) out[p.top - p.recent + i] = P - p.recent + i;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the scores are written
  if (N == 0) return;
  const uint64_t* keys = p.keys + (int64_t)unit * p.key_stride;
  constexpr int kAhead = 4;                          // keys in flight per thread

  uint64_t k_lo = ~0ull, k_hi = 0;
  for (int i = tid; i < N; i += kAhead * kPickThreads) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint64_t k = keys[min(i + u * kPickThreads, N - 1)];
      k_lo = min(k_lo, k);
      k_hi = max(k_hi, k);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    k_lo = min(k_lo, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)k_lo, o));
    k_hi = max(k_hi, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)k_hi, o));
  }
  if (lane == 0) {
    warp_lo[warp] = k_lo;
    warp_hi[warp] = k_hi;
  }
  if (tid < 256) hist[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPickWarps; ++w) {
    k_lo = min(k_lo, warp_lo[w]);
    k_hi = max(k_hi, warp_hi[w]);
  }

  // ---- the border: key >> shift == border for the last selected ones, `rest` of them ----
  const int top_bit = k_lo == k_hi ? -1 : 63 - __clzll((long long)(k_lo ^ k_hi));
  int shift = top_bit + 1;                           // bits above are the same in all keys
  uint64_t border = shift >= 64 ? 0 : k_lo >> shift;
  int rest = p.top - p.sinks - p.recent;             // < N
  while (shift > 0) {
    const int bits = min(8, shift), ns = shift - bits;
    for (int i = tid; i < N; i += kAhead * kPickThreads) {
      uint64_t k[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) k[u] = keys[min(i + u * kPickThreads, N - 1)];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * kPickThreads < N && (shift >= 64 || (k[u] >> shift) == border))
          atomicAdd(&hist[(uint32_t)(k[u] >> ns) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins from the highest down: thread t < 256 has bin 255 - t
    uint32_t mine = 0, incl = 0;
    if (warp < 8) {
      mine = incl = hist[255 - tid];
      hist[255 - tid] = 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) scan[warp] = incl;
    }
    __syncthreads();
    if (warp < 8) {
      for (int w = 0; w < warp; ++w) incl += scan[w];
      if (incl >= (uint32_t)rest && incl - mine < (uint32_t)rest) {
        found[0] = 255 - (uint32_t)tid;
        found[1] = (uint32_t)rest - (incl - mine);
        found[2] = mine;
      }
    }
    __syncthreads();
    border = (border << bits) | found[0];
    rest = (int)found[1];
    shift = ns;
    if (found[2] == found[1]) break;                 // the whole bin is selected
  }

  // ---- the selected pages in ascending order: a warp per consecutive part ----
  const int per = ((N + kPickWarps - 1) / kPickWarps + 31) & ~31;
  const int w0 = min(warp * per, N), w1 = min(w0 + per, N);
  int gt = 0, eq = 0;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint64_t k = in ? keys[i0 + lane] >> shift : 0;
    gt += __popc(__ballot_sync(~0u, in && k > border));
    eq += __popc(__ballot_sync(~0u, in && k == border));
  }
  if (lane == 0) {
    n_gt[warp] = gt;
    n_eq[warp] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < warp; ++w) {
    gt += n_gt[w];
    eq += n_eq[w];
  }
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint64_t k = in ? keys[i0 + lane] >> shift : 0;
    const uint32_t mg = __ballot_sync(~0u, in && k > border), me = __ballot_sync(~0u, in && k == border);
    const uint32_t below = (1u << lane) - 1u;
    const int gb = gt + __popc(mg & below), eb = eq + __popc(me & below);
    if (in && (k > border || (k == border && eb < rest))) out[p.sinks + gb + min(eb, rest)] = p.sinks + i0 + lane;
    gt += __popc(mg);
    eq += __popc(me);
  }
}

template <typename T, int D>
int launch_select_typed(SelectPagesParams p, int num_sms, cudaStream_t stream) {
  const int64_t units = (int64_t)p.n * p.num_kv_heads;
  if (units * ((p.key_stride + kRun - 1) / kRun) > 0x7fffffff) return STARKV_EINVAL;   // 32-bit run numbers
  const void* fn = (const void*)score_kernel<T, D>;
  if (const int st = allow_smem(fn, kRingBytes)) return st;
  void* args[] = {&p};
  if (p.key_stride > p.top) {   // else no sequence has pages to choose from
    const int64_t runs = units * ((p.key_stride + kRun - 1) / kRun);
    const int64_t grid = std::min<int64_t>(3 * num_sms, runs);
    if (cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kThreads), args, kRingBytes, stream) != cudaSuccess)
      return STARKV_ECUDA;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)units);
  cfg.blockDim = dim3(kPickThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.key_stride > p.top;   // behind score_kernel alone may the launch come early
  return cudaLaunchKernelExC(&cfg, (const void*)pick_kernel, args) == cudaSuccess ? STARKV_OK : STARKV_ECUDA;
}

template <typename T, int D>
int launch_bounds_typed(PageBoundsParams p, cudaStream_t stream) {
  const int64_t items = (int64_t)p.n * p.max_pages * p.num_kv_heads;
  const int64_t blocks = (items + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return STARKV_EINVAL;
  void* args[] = {&p};
  return cudaLaunchKernel((const void*)bounds_kernel<T, D>, dim3((unsigned)blocks), dim3(kThreads), args, 0, stream) ==
                 cudaSuccess
             ? STARKV_OK
             : STARKV_ECUDA;
}

}  // namespace

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

// Page bounds and page selection over a paged full-rank cache.
//
// bounds_kernel: per page and KV head the smallest and largest value of every key
// channel. It reads each key once and writes 2 D values per page; the read is the cost.
// A warp takes one (page, head), 16 bytes per lane, whole rows at a time.
//
// select_kernel: for each (sequence, KV head) the `top` pages of the highest score
//   score(page) = sum_{g in group} sum_d max(q[g, d] lo[d], q[g, d] hi[d])
//               = sum_d up[d] hi[d] + down[d] lo[d],
//   up = sum_g max(q[g], 0),  down = sum_g min(q[g], 0),
// an upper bound of sum_g q[g] . k over the page's keys. One page costs 4 D bytes and 2 D
// multiply-adds whatever G is, so the read of the bounds is the cost. Scores are summed
// in 64 bits: the products of two 16-bit values are exact there and the order of two
// pages next to the border does not depend on how the sum was split (32-bit sums put
// about one of a thousand selections on the other side).
//
// A cluster of CTAs takes one (sequence, KV head), each CTA a run of pages whose scores
// stay in its shared memory as order-preserving 64-bit keys; the border is found by
// radix selection from the highest bit in which the keys differ, the histograms added
// through distributed shared memory. Ties go to the lowest page index.
#include <cooperative_groups.h>
#include <type_traits>

#include "starkv_common.cuh"
#include "starkv_kernels.h"

namespace starkv {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr size_t kKeyBytes = 192 * 1024;

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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectPagesParams p) {
  extern __shared__ __align__(16) uint64_t keys[];
  __shared__ uint32_t hist[2][256];
  __shared__ uint64_t range[2];                      // smallest, largest key of this CTA
  __shared__ uint64_t warp_lo[kWarps], warp_hi[kWarps];
  __shared__ uint32_t scan[kWarps], found[3];        // bin, still needed in it, its count
  __shared__ int n_gt[kWarps], n_eq[kWarps], cta_counts[2], before[2];
  constexpr int LP = 2 * D / 8;                      // lanes of one page's bounds
  constexpr int kPer = 8 * (32 / LP);                // pages of a warp's step
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t unit = blockIdx.x / C;
  const int hk = (int)(unit % p.num_kv_heads), b = (int)(unit / p.num_kv_heads);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int L = min(max(p.seq_lens[b], 0), p.max_len);
  const int P = (int)(((int64_t)L + p.block_size - 1) / p.block_size);
  int32_t* out = p.pages + b * p.pg_s0 + hk * p.pg_s1;
  if (P <= p.top) {   // every page, then -1
    if (rank == 0)
      for (int i = tid; i < p.top; i += kThreads) out[i] = i < P ? i : -1;
    return;
  }
  const int need = p.top - p.sinks - p.recent;       // >= 0; P > top: the kept pages do not overlap
  if (rank == 0) {
    for (int i = tid; i < p.sinks; i += kThreads) out[i] = i;
    for (int i = tid; i < p.recent; i += kThreads) out[p.top - p.recent + i] = P - p.recent + i;
  }
  if (need == 0) return;
  const int N = P - p.sinks - p.recent;              // pages that compete, > need
  const int c0 = (int)((int64_t)N * rank / C), cnt = (int)((int64_t)N * (rank + 1) / C) - c0;

  // ---- scores of this CTA's pages ----
  uint64_t k_lo = ~0ull, k_hi = 0;
  {
    const int e = lane % LP, sub = lane / LP;
    const int d = (e * 8) % D;
    const bool upper = e * 8 >= D;
    double w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0.0;
    for (int g = 0; g < p.group; ++g) {
      const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)(hk * p.group + g) * p.q_s1 + d;
      float f[8];
      to_f32x8(T{}, *reinterpret_cast<const uint4*>(q), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] += (double)(upper ? (f[i] < 0.f ? 0.f : f[i]) : (f[i] > 0.f ? 0.f : f[i]));
    }
    const int32_t* bt = p.block_table + b * p.bt_s0;
    const T* bounds = reinterpret_cast<const T*>(p.bounds) + (int64_t)hk * p.b_s1 + e * 8;
    auto block_of = [&](int i0) {   // lanes 0 .. kPer-1: the blocks of pages i0 .. i0 + kPer - 1
      const int i = i0 + lane;
      if (lane >= kPer || i >= cnt) return 0;
      int blk = bt[(int64_t)(p.sinks + c0 + i) * p.bt_s1];
      if ((unsigned)blk >= (unsigned)p.num_blocks) {
        record_status(p.status, STARKV_EBOUNDS);
        blk = 0;
      }
      return blk;
    };
    int nxt = block_of(warp * kPer);
    for (int i0 = warp * kPer; i0 < cnt; i0 += kWarps * kPer) {
      const int cur = nxt;
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = *reinterpret_cast<const uint4*>(bounds + (int64_t)__shfl_sync(~0u, cur, sub * 8 + u) * p.b_s0);
      nxt = block_of(i0 + kWarps * kPer);
      double s[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float f[8];
        to_f32x8(T{}, v[u], f);
        s[u] = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[u] = fma((double)f[i], w[i], s[u]);
      }
      // sums over the LP lanes of a page: three steps that also halve the pages a lane holds
#pragma unroll
      for (int h = 4, o = LP / 2; h >= 1; h >>= 1, o >>= 1)
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const double give = lane & o ? s[i] : s[i + h], keep = lane & o ? s[i + h] : s[i];
          s[i] = keep + __shfl_xor_sync(~0u, give, o);
        }
#pragma unroll
      for (int o = LP / 16; o; o >>= 1) s[0] += __shfl_xor_sync(~0u, s[0], o);
      const int at = i0 + sub * 8 + (lane & (LP / 2) ? 4 : 0) + (lane & (LP / 4) ? 2 : 0) + (lane & (LP / 8) ? 1 : 0);
      if ((lane & (LP / 8 - 1)) == 0 && at < cnt) {
        const uint64_t key = order_key(s[0]);
        keys[at] = key;
        k_lo = min(k_lo, key);
        k_hi = max(k_hi, key);
      }
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
  hist[0][tid] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) {
      k_lo = min(k_lo, warp_lo[w]);
      k_hi = max(k_hi, warp_hi[w]);
    }
    range[0] = k_lo;
    range[1] = k_hi;
  }
  cluster.sync();
  k_lo = ~0ull;
  k_hi = 0;
  for (int r = 0; r < C; ++r) {
    const uint64_t* o = cluster.map_shared_rank(range, r);
    k_lo = min(k_lo, o[0]);
    k_hi = max(k_hi, o[1]);
  }

  // ---- the border: key >> shift == border for the last selected ones, `rest` of them ----
  const int top_bit = k_lo == k_hi ? -1 : 63 - __clzll((long long)(k_lo ^ k_hi));
  int shift = top_bit + 1;                           // bits above are the same in all keys
  uint64_t border = shift >= 64 ? 0 : k_lo >> shift;
  int rest = need;
  for (int pass = 0; shift > 0; ++pass) {
    const int bits = min(8, shift), ns = shift - bits;
    uint32_t* h = hist[pass & 1];
    for (int i = tid; i < cnt; i += kThreads) {
      const uint64_t k = keys[i];
      if (shift >= 64 || (k >> shift) == border) atomicAdd(&h[(uint32_t)(k >> ns) & ((1u << bits) - 1)], 1u);
    }
    cluster.sync();
    // bins from the highest down: thread t has bin 255 - t
    const int bin = 255 - tid;
    uint32_t mine = 0;
    for (int r = 0; r < C; ++r) mine += cluster.map_shared_rank(h, r)[bin];
    hist[(pass + 1) & 1][tid] = 0;                   // its readers passed the barrier above
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) incl += scan[w];
    if (incl >= (uint32_t)rest && incl - mine < (uint32_t)rest) {
      found[0] = (uint32_t)bin;
      found[1] = (uint32_t)rest - (incl - mine);
      found[2] = mine;
    }
    __syncthreads();
    border = (border << bits) | found[0];
    rest = (int)found[1];
    shift = ns;
    if (found[2] == found[1]) break;                 // the whole bin is selected
  }

  // ---- the selected pages in ascending order ----
  const int per = ((cnt + kWarps - 1) / kWarps + 31) & ~31;
  const int w0 = min(warp * per, cnt), w1 = min(w0 + per, cnt);
  int gt = 0, eq = 0;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const uint64_t k = i0 + lane < w1 ? keys[i0 + lane] >> shift : 0;
    gt += __popc(__ballot_sync(~0u, i0 + lane < w1 && k > border));
    eq += __popc(__ballot_sync(~0u, i0 + lane < w1 && k == border));
  }
  if (lane == 0) {
    n_gt[warp] = gt;
    n_eq[warp] = eq;
  }
  __syncthreads();
  if (tid == 0) {
    int a = 0, c = 0;
    for (int w = 0; w < kWarps; ++w) {
      a += n_gt[w];
      c += n_eq[w];
    }
    cta_counts[0] = a;
    cta_counts[1] = c;
  }
  cluster.sync();
  if (tid == 0) {
    int a = 0, c = 0;
    for (int r = 0; r < rank; ++r) {
      const int* o = cluster.map_shared_rank(cta_counts, r);
      a += o[0];
      c += o[1];
    }
    before[0] = a;
    before[1] = c;
  }
  __syncthreads();
  gt = before[0];
  eq = before[1];
  for (int w = 0; w < warp; ++w) {
    gt += n_gt[w];
    eq += n_eq[w];
  }
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint64_t k = in ? keys[i0 + lane] >> shift : 0;
    const uint32_t mg = __ballot_sync(~0u, in && k > border), me = __ballot_sync(~0u, in && k == border);
    const uint32_t below = (1u << lane) - 1u;
    const int g = gt + __popc(mg & below), e = eq + __popc(me & below);
    if (in && (k > border || (k == border && e < rest))) out[p.sinks + g + min(e, rest)] = p.sinks + c0 + i0 + lane;
    gt += __popc(mg);
    eq += __popc(me);
  }
  cluster.sync();   // no CTA leaves while another reads its counts
}

template <typename T, int D>
int launch_select_typed(SelectPagesParams p, int num_sms, cudaStream_t stream) {
  const int64_t most = ((int64_t)p.max_len + p.block_size - 1) / p.block_size;
  const int64_t units = (int64_t)p.n * p.num_kv_heads;
  // a cluster per unit: more CTAs while the units alone leave SMs idle and a CTA keeps
  // at least 64 pages, and as many as the scores need in shared memory
  int C = 1;
  while (C < kMaxCluster && units * C < 2 * num_sms && most / (2 * C) >= 64) C *= 2;
  while (C < kMaxCluster && (size_t)((most + C - 1) / C + 1) * 8 > kKeyBytes) C *= 2;
  const size_t smem = (size_t)((most + C - 1) / C + 1) * 8;
  if (smem > kKeyBytes || units * C > 0x7fffffff) return STARKV_EINVAL;
  p.keys = (int)((most + C - 1) / C + 1);
  const void* fn = (const void*)select_kernel<T, D>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kKeyBytes) != cudaSuccess)
    return STARKV_ECUDA;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(units * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&p};
  return cudaLaunchKernelExC(&cfg, fn, args) == cudaSuccess ? STARKV_OK : STARKV_ECUDA;
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

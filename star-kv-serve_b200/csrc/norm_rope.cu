// Per-head RMS norm of queries and keys, the rotation by position, and the write of keys
// and values into a paged cache, in one pass:
//   y = x * rsqrt(mean(x^2) + eps) * w                 (no weight: y = x)
//   out[i]         = y[i] cos[i] - y[i + rot/2] sin[i]
//   out[i + rot/2] = y[i + rot/2] cos[i] + y[i] sin[i]      i < rot / 2, channels >= rot as they are
// Everything between the load and the store is f32 and rounded once.
//
// Each row of head_dim values is read once and written once, and that traffic is the
// cost; the table row and the weights are shared by a token's heads and stay in L1 / L2.
// D / 8 lanes hold a row, 16 bytes each; the sum of squares and the partner channel come
// by shuffles.
#include <type_traits>

#include "starkv_common.cuh"
#include "starkv_kernels.h"

namespace starkv {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerGroup = 4;

__device__ __forceinline__ void load8(const void* p, int64_t i, int dtype, float (&f)[8]) {
  if (dtype == STARKV_F32) {
    const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = s[0], b = s[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
  if (dtype == STARKV_BF16) bf16x8_to_f32(u, f);
  else f16x8_to_f32(u, f);
}

__device__ __forceinline__ uint4 round8(__nv_bfloat16, const float (&f)[8]) {
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return u;
}
__device__ __forceinline__ uint4 round8(__half, const float (&f)[8]) {
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return u;
}

// A group of D / 8 lanes takes up to kPer consecutive heads of the queries, keys or values
// of one token: the position's table values and the weight are loaded once for them, and
// kPer rows are in flight.
template <typename T, int D, int kPer>
__global__ void __launch_bounds__(kThreads, 3) norm_rope_kernel(const NormRopeParams p, unsigned q_chunks,
                                                                unsigned k_chunks, unsigned chunks, unsigned items) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  constexpr int dtype = std::is_same<T, __half>::value ? STARKV_F16 : STARKV_BF16;
  const int j = threadIdx.x % kLanes;
  const unsigned item = blockIdx.x * kGroups + threadIdx.x / kLanes;
  const bool live = item < items;                      // groups share a warp: all take part in the shuffles
  const unsigned t = live ? item / chunks : 0, chunk = live ? item - t * chunks : 0;
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;   // query, key, value
  const int h0 = kPer * (int)(chunk - (kind == 0 ? 0 : kind == 1 ? q_chunks : q_chunks + k_chunks));
  const int count = live ? min(kPer, (kind == 0 ? p.num_heads : p.num_kv_heads) - h0) : 0;
  const int64_t step = kind == 0 ? p.q_s1 : kind == 1 ? p.k_s1 : p.v_s1;
  const T* src = reinterpret_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                 t * (kind == 0 ? p.q_s0 : kind == 1 ? p.k_s0 : p.v_s0) + h0 * step + j * 8;
  uint4 raw[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    raw[u] = u < count ? *reinterpret_cast<const uint4*>(src + u * step) : make_uint4(0, 0, 0, 0);

  const int half = p.rot / 16;                         // lanes of half the rotated channels
  const bool low = j < half, turns = j < 2 * half && kind < 2;
  const int other = (threadIdx.x & 31 & ~(kLanes - 1)) + (j < 2 * half ? (low ? j + half : j - half) : j);
  float c[8], s[8], g[8];
  const void* w = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = g[i] = 1.f;
    s[i] = 0.f;
  }
  if (w) load8(w, j * 8, p.w_dtype, g);
  if (turns && live) {
    int64_t pos = load_slot(p.positions, t, p.pos_dtype);
    if (pos < 0 || pos >= p.table_rows) {
      record_status(p.status, STARKV_EBOUNDS);
      pos = pos < 0 ? 0 : p.table_rows - 1;
    }
    const int64_t at = pos * p.t_s0 + (low ? j : j - half) * 8;
    load8(p.table, at, p.table_dtype, c);
    load8(p.table, at + p.rot / 2, p.table_dtype, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = low ? -s[i] : s[i];   // x c - y s below, x c + y s above
  }
  // where the rows go: q_out, or k_out and the cache
  T* out = kind == 0   ? reinterpret_cast<T*>(p.q_out) + t * p.qo_s0 + h0 * p.qo_s1 + j * 8
           : kind == 1 ? reinterpret_cast<T*>(p.k_out) + t * p.ko_s0 + h0 * p.ko_s1 + j * 8
                       : nullptr;
  if (kind == 1 && !p.k_out) out = nullptr;
  const int64_t out_step = kind == 0 ? p.qo_s1 : p.ko_s1;
  T* cache = nullptr;
  const int64_t cache_step = kind == 1 ? p.kc_s2 : p.vc_s2;
  if (p.k_cache && kind > 0 && live) {
    const int64_t slot = load_slot(p.slots, t, p.slot_dtype);
    if (slot >= (int64_t)p.num_blocks * p.block_size) {
      record_status(p.status, STARKV_EBOUNDS);
    } else if (slot >= 0) {                            // negative: padding, not written
      // a 64-bit division is some hundred instructions
      const int64_t blk = slot <= 0x7fffffff ? (unsigned)slot / (unsigned)p.block_size : slot / p.block_size;
      const int64_t off = slot - blk * p.block_size;
      cache = kind == 1 ? reinterpret_cast<T*>(p.k_cache) + blk * p.kc_s0 + off * p.kc_s1 + h0 * p.kc_s2 + j * 8
                        : reinterpret_cast<T*>(p.v_cache) + blk * p.vc_s0 + off * p.vc_s1 + h0 * p.vc_s2 + j * 8;
    }
  }
  const bool norms = p.q_weight || p.k_weight;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    float x[8];
    if (dtype == STARKV_BF16) bf16x8_to_f32(raw[u], x);
    else f16x8_to_f32(raw[u], x);
    if (norms) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
      const float inv = w ? 1.f / sqrtf(ss * (1.f / D) + p.eps) : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(~0u, x[i], other);
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + y[i] * s[i];
    }
    if (u >= count) continue;
    const uint4 res = kind < 2 ? round8(T{}, x) : raw[u];
    if (out) *reinterpret_cast<uint4*>(out + u * out_step) = res;
    if (cache) *reinterpret_cast<uint4*>(cache + u * cache_step) = res;
  }
}

template <typename T, int D>
int launch_typed(NormRopeParams p, cudaStream_t stream) {
  constexpr int kGroups = kThreads / (D / 8);
  unsigned qc = (p.num_heads + kRowsPerGroup - 1) / kRowsPerGroup;
  unsigned kc = (p.num_kv_heads + kRowsPerGroup - 1) / kRowsPerGroup;
  unsigned chunks = qc + kc * (p.v ? 2 : 1);
  const int64_t all = (int64_t)p.n * chunks;
  if (all > 0x7fffffff) return STARKV_EINVAL;
  unsigned items = (unsigned)all;
  void* args[] = {&p, &qc, &kc, &chunks, &items};
  return cudaLaunchKernel((const void*)norm_rope_kernel<T, D, kRowsPerGroup>, dim3((items + kGroups - 1) / kGroups),
                          dim3(kThreads), args, 0, stream) == cudaSuccess
             ? STARKV_OK
             : STARKV_ECUDA;
}

}  // namespace

int launch_norm_rope(const NormRopeParams& p, int dtype, int head_dim, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_typed<__nv_bfloat16, 64>(p, stream) : launch_typed<__nv_bfloat16, 128>(p, stream);
  return head_dim == 64 ? launch_typed<__half, 64>(p, stream) : launch_typed<__half, 128>(p, stream);
}

}  // namespace starkv

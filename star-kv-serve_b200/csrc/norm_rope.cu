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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRopeParams p) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  constexpr int dtype = std::is_same<T, __half>::value ? STARKV_F16 : STARKV_BF16;
  const int per = p.num_heads + p.num_kv_heads * (p.v ? 2 : 1);   // rows of a token
  const int j = threadIdx.x % kLanes;
  const int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  const bool live = r < (int64_t)p.n * per;
  const int64_t t = live ? r / per : 0;
  const int row = live ? (int)(r - t * per) : 0;
  // which of q, k, v
  const int kind = row < p.num_heads ? 0 : row < p.num_heads + p.num_kv_heads ? 1 : 2;
  const int h = kind == 0 ? row : kind == 1 ? row - p.num_heads : row - p.num_heads - p.num_kv_heads;
  const T* src = kind == 0 ? reinterpret_cast<const T*>(p.q) + t * p.q_s0 + h * p.q_s1
                 : kind == 1 ? reinterpret_cast<const T*>(p.k) + t * p.k_s0 + h * p.k_s1
                             : reinterpret_cast<const T*>(p.v) + t * p.v_s0 + h * p.v_s1;
  const uint4 raw = *reinterpret_cast<const uint4*>(src + j * 8);
  uint4 res = raw;
  // lanes of values and lanes of another token share a warp: all take part in the shuffles
  {
    float x[8];
    if (dtype == STARKV_BF16) bf16x8_to_f32(raw, x);
    else f16x8_to_f32(raw, x);
    const void* w = kind == 0 ? p.q_weight : p.k_weight;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    if (w) {
      const float inv = 1.f / sqrtf(ss * (1.f / D) + p.eps);
      float g[8];
      load8(w, j * 8, p.w_dtype, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
    }
    const int half = p.rot / 16;                    // lanes of half the rotated channels
    const bool low = j < half, turns = j < 2 * half;
    const int other = (threadIdx.x & 31 & ~(kLanes - 1)) + (turns ? (low ? j + half : j - half) : j);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(~0u, x[i], other);
    if (turns && kind < 2) {
      int64_t pos = load_slot(p.positions, t, p.pos_dtype);
      if (pos < 0 || pos >= p.table_rows) {
        if (live) record_status(p.status, STARKV_EBOUNDS);
        pos = pos < 0 ? 0 : p.table_rows - 1;
      }
      float c[8], s[8];
      const int64_t at = pos * p.t_s0 + (low ? j : j - half) * 8;
      load8(p.table, at, p.table_dtype, c);
      load8(p.table, at + p.rot / 2, p.table_dtype, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = low ? x[i] * c[i] - y[i] * s[i] : x[i] * c[i] + y[i] * s[i];
    }
    if (kind < 2) res = round8(T{}, x);
  }
  if (!live) return;
  if (kind == 0) {
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + t * p.qo_s0 + h * p.qo_s1 + j * 8) = res;
    return;
  }
  if (kind == 1 && p.k_out)
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.k_out) + t * p.ko_s0 + h * p.ko_s1 + j * 8) = res;
  if (!p.k_cache) return;
  const int64_t slot = load_slot(p.slots, t, p.slot_dtype);
  if (slot < 0) return;   // padding: not written
  const int64_t blk = slot / p.block_size, off = slot - blk * p.block_size;
  if (blk >= p.num_blocks) {
    record_status(p.status, STARKV_EBOUNDS);
    return;
  }
  T* dst = kind == 1 ? reinterpret_cast<T*>(p.k_cache) + blk * p.kc_s0 + off * p.kc_s1 + h * p.kc_s2
                     : reinterpret_cast<T*>(p.v_cache) + blk * p.vc_s0 + off * p.vc_s1 + h * p.vc_s2;
  *reinterpret_cast<uint4*>(dst + j * 8) = res;
}

template <typename T, int D>
int launch_typed(NormRopeParams p, cudaStream_t stream) {
  constexpr int kRows = kThreads / (D / 8);
  const int64_t rows = (int64_t)p.n * (p.num_heads + p.num_kv_heads * (p.v ? 2 : 1));
  const int64_t blocks = (rows + kRows - 1) / kRows;
  if (blocks > 0x7fffffff) return STARKV_EINVAL;
  void* args[] = {&p};
  return cudaLaunchKernel((const void*)norm_rope_kernel<T, D>, dim3((unsigned)blocks), dim3(kThreads), args, 0,
                          stream) == cudaSuccess
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

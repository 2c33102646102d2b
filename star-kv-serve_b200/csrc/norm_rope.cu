// Per-head RMS norm of queries and keys, the rotation by position, and the write of keys
// and values into a paged cache, in one pass:
//   y = x * rsqrt(mean(x^2) + eps) * w                 (no weight: y = x)
//   out[i]         = y[i] cos[i] - y[i + rot/2] sin[i]
//   out[i + rot/2] = y[i + rot/2] cos[i] + y[i] sin[i]      i < rot / 2, channels >= rot as they are
// Everything between the load and the store is f32 and rounded once.
//
// Each row of head_dim values is read once and written once, and that traffic is the
// cost; the table row and the weights are shared by a token's heads and stay in L1 / L2.
// D / 8 lanes hold a row; a lane holds four channels of the first rotated half and their
// four partners of the second (8 bytes each), so the rotation needs no other lane, and
// only the sum of squares comes by shuffles.
#include "starkv_common.cuh"
#include "starkv_kernels.h"

namespace starkv {

namespace {

constexpr int kThreads = 256;
constexpr int kManyRows = 256;   // rows per SM from which a group takes 8 rows and not 2

__device__ __forceinline__ float4 load4(const void* p, int64_t i, int dtype) {
  if (dtype == STARKV_F32) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
  if (dtype == STARKV_BF16)
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ float2 unpack(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t round2(__nv_bfloat16, float2 f) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t round2(__half, float2 f) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// two f32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
        "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return d;
}

// A group of D / 8 lanes takes up to kPer consecutive heads of the queries, keys or values
// of one token: the position's table values and the weight are loaded once for them, and
// kPer rows are in flight.
template <typename T, int D, int kPer>
__global__ void __launch_bounds__(kThreads, 3) norm_rope_kernel(const NormRopeParams p, unsigned q_chunks,
                                                                unsigned k_chunks, unsigned chunks, unsigned items) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  const int j = threadIdx.x % kLanes;
  const unsigned item = blockIdx.x * kGroups + threadIdx.x / kLanes;
  const bool live = item < items;                      // groups share a warp: all take part in the shuffles
  const unsigned t = live ? item / chunks : 0, chunk = live ? item - t * chunks : 0;
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;   // query, key, value
  const int h0 = kPer * (int)(chunk - (kind == 0 ? 0 : kind == 1 ? q_chunks : q_chunks + k_chunks));
  const int count = live ? min(kPer, (kind == 0 ? p.num_heads : p.num_kv_heads) - h0) : 0;
  const int64_t step = kind == 0 ? p.q_s1 : kind == 1 ? p.k_s1 : p.v_s1;
  // this lane's channels: lo .. lo + 3 and hi .. hi + 3; behind the rotated width eight in a row
  const int pairs = p.rot / 8;
  const bool turns = j < pairs && kind < 2;
  const int lo = j < pairs ? 4 * j : p.rot + 8 * (j - pairs), hi = j < pairs ? lo + p.rot / 2 : lo + 4;
  const T* src = reinterpret_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                 t * (kind == 0 ? p.q_s0 : kind == 1 ? p.k_s0 : p.v_s0) + h0 * step;
  uint2 raw_lo[kPer], raw_hi[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    raw_lo[u] = u < count ? *reinterpret_cast<const uint2*>(src + u * step + lo) : make_uint2(0, 0);
    raw_hi[u] = u < count ? *reinterpret_cast<const uint2*>(src + u * step + hi) : make_uint2(0, 0);
  }

  // out_lo = inv * (x_lo a + x_hi b), out_hi = inv * (x_hi c + x_lo d): the weight is in a .. d already
  float4 a = make_float4(1.f, 1.f, 1.f, 1.f), b = make_float4(0.f, 0.f, 0.f, 0.f), c = a, d = b;
  const void* w = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
  if (turns && live) {
    int64_t pos = load_slot(p.positions, t, p.pos_dtype);
    if (pos < 0 || pos >= p.table_rows) {
      record_status(p.status, STARKV_EBOUNDS);
      pos = pos < 0 ? 0 : p.table_rows - 1;
    }
    const int64_t at = pos * p.t_s0 + lo;
    a = c = load4(p.table, at, p.table_dtype);
    d = load4(p.table, at + p.rot / 2, p.table_dtype);
    b = make_float4(-d.x, -d.y, -d.z, -d.w);
  }
  if (w) {
    const float4 gl = load4(w, lo, p.w_dtype), gh = load4(w, hi, p.w_dtype);
    a = make_float4(a.x * gl.x, a.y * gl.y, a.z * gl.z, a.w * gl.w);
    b = make_float4(b.x * gh.x, b.y * gh.y, b.z * gh.z, b.w * gh.w);
    c = make_float4(c.x * gh.x, c.y * gh.y, c.z * gh.z, c.w * gh.w);
    d = make_float4(d.x * gl.x, d.y * gl.y, d.z * gl.z, d.w * gl.w);
  }
  // where the rows go: q_out, or k_out and the cache
  T* out = kind == 0   ? reinterpret_cast<T*>(p.q_out) + t * p.qo_s0 + h0 * p.qo_s1
           : kind == 1 ? reinterpret_cast<T*>(p.k_out) + t * p.ko_s0 + h0 * p.ko_s1
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
      cache = kind == 1 ? reinterpret_cast<T*>(p.k_cache) + blk * p.kc_s0 + off * p.kc_s1 + h0 * p.kc_s2
                        : reinterpret_cast<T*>(p.v_cache) + blk * p.vc_s0 + off * p.vc_s1 + h0 * p.vc_s2;
    }
  }
  const bool norms = p.q_weight || p.k_weight;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    uint2 res_lo = raw_lo[u], res_hi = raw_hi[u];
    const float2 l0 = unpack(T{}, res_lo.x), l1 = unpack(T{}, res_lo.y);
    const float2 h0 = unpack(T{}, res_hi.x), h1 = unpack(T{}, res_hi.y);
    float inv = 1.f;
    if (norms) {
      const float2 q = fma2(h1, h1, fma2(h0, h0, fma2(l1, l1, mul2(l0, l0))));
      float ss = q.x + q.y;
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
      if (w) inv = rsqrtf(ss * (1.f / D) + p.eps);     // within 2^-22
    }
    if (u >= count) continue;
    if (kind < 2) {
      const float2 iv = make_float2(inv, inv);
      const float2 a0 = make_float2(a.x, a.y), a1 = make_float2(a.z, a.w), b0 = make_float2(b.x, b.y),
                   b1 = make_float2(b.z, b.w), c0 = make_float2(c.x, c.y), c1 = make_float2(c.z, c.w),
                   d0 = make_float2(d.x, d.y), d1 = make_float2(d.z, d.w);
      res_lo.x = round2(T{}, mul2(iv, fma2(h0, b0, mul2(l0, a0))));
      res_lo.y = round2(T{}, mul2(iv, fma2(h1, b1, mul2(l1, a1))));
      res_hi.x = round2(T{}, mul2(iv, fma2(l0, d0, mul2(h0, c0))));
      res_hi.y = round2(T{}, mul2(iv, fma2(l1, d1, mul2(h1, c1))));
    }
    if (out) {
      *reinterpret_cast<uint2*>(out + u * out_step + lo) = res_lo;
      *reinterpret_cast<uint2*>(out + u * out_step + hi) = res_hi;
    }
    if (cache) {
      *reinterpret_cast<uint2*>(cache + u * cache_step + lo) = res_lo;
      *reinterpret_cast<uint2*>(cache + u * cache_step + hi) = res_hi;
    }
  }
}

template <typename T, int D, int kPer>
int launch_per(NormRopeParams p, cudaStream_t stream) {
  constexpr int kGroups = kThreads / (D / 8);
  unsigned qc = (p.num_heads + kPer - 1) / kPer;
  unsigned kc = (p.num_kv_heads + kPer - 1) / kPer;
  unsigned chunks = qc + kc * (p.v ? 2 : 1);
  const int64_t all = (int64_t)p.n * chunks;
  if (all > 0x7fffffff) return STARKV_EINVAL;
  unsigned items = (unsigned)all;
  void* args[] = {&p, &qc, &kc, &chunks, &items};
  return cudaLaunchKernel((const void*)norm_rope_kernel<T, D, kPer>, dim3((items + kGroups - 1) / kGroups),
                          dim3(kThreads), args, 0, stream) == cudaSuccess
             ? STARKV_OK
             : STARKV_ECUDA;
}

template <typename T, int D>
int launch_typed(const NormRopeParams& p, int num_sms, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.n * (p.num_heads + p.num_kv_heads * (p.v ? 2 : 1));
  return rows > (int64_t)num_sms * kManyRows ? launch_per<T, D, 8>(p, stream) : launch_per<T, D, 2>(p, stream);
}

}  // namespace

int launch_norm_rope(const NormRopeParams& p, int dtype, int head_dim, int num_sms, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_typed<__nv_bfloat16, 64>(p, num_sms, stream) : launch_typed<__nv_bfloat16, 128>(p, num_sms, stream);
  return head_dim == 64 ? launch_typed<__half, 64>(p, num_sms, stream) : launch_typed<__half, 128>(p, num_sms, stream);
}

}  // namespace starkv

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

constexpr int kThreads = 128;
// rows per SM from which a warp takes 4 steps and not one (48 rows a token: one token 3.0
// against 3.4 us, 64 tokens the same, 256 tokens 4.2 against 3.5, 4096 tokens 37 against 22)
constexpr int kManyRows = 24;

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

// A warp takes up to kSteps * G heads of the queries, keys or values of one token, G = 32 *
// 8 / D heads a step: token, kind, table row and cache slot are the warp's, so a row costs
// little more than its own arithmetic (8191 tokens of 48 heads, f16: 41 us, 5.0 TB/s; with
// token and heads chosen per group of lanes 193 instructions a warp and step, and 51 us).
// kPart: the table is narrower than a head (asked in the loop of every call: 45 us).
template <typename T, int D, int kSteps, bool kPart>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRopeParams p, unsigned q_chunks,
                                                             unsigned k_chunks, unsigned chunks, unsigned items) {
  constexpr int kLanes = D / 8, G = 32 / kLanes;
  constexpr int kAhead = kSteps < 4 ? kSteps : 4;      // steps in flight
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (item >= items) return;
  const unsigned t = item / chunks, chunk = item - t * chunks;
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;   // query, key, value
  const int j = lane % kLanes, g = lane / kLanes;
  const int h0 = kSteps * G * (int)(chunk - (kind == 0 ? 0 : kind == 1 ? q_chunks : q_chunks + k_chunks)) + g;
  const int heads = (kind == 0 ? p.num_heads : p.num_kv_heads) - h0 + G - 1;
  const int count = heads / G, most = (heads + g) / G;   // heads of this group (also <= 0), of group 0
  // this lane's channels: lo .. lo + 3 and hi .. hi + 3; behind the rotated width eight in a row
  const int pairs = p.rot / 8;
  const int lo = j < pairs ? 4 * j : p.rot + 8 * (j - pairs), hi = j < pairs ? lo + p.rot / 2 : lo + 4;
  const int64_t s0 = kind == 0 ? p.q_s0 : kind == 1 ? p.k_s0 : p.v_s0;
  const int64_t s1 = kind == 0 ? p.q_s1 : kind == 1 ? p.k_s1 : p.v_s1;
  const T* src = reinterpret_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + t * s0 + h0 * s1 + lo;
  const int64_t step = G * s1;
  uint2 raw[kAhead][2];
  const auto load = [&](int s) {                       // steps s .. s + kAhead - 1
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      raw[u][0] = raw[u][1] = make_uint2(0, 0);
      if (s + u < count) {
        raw[u][0] = *reinterpret_cast<const uint2*>(src);
        raw[u][1] = *reinterpret_cast<const uint2*>(src + (hi - lo));
      }
      src += step;
    }
  };
  load(0);

  // where the rows go: queries to q_out, keys and values to the cache, keys to k_out as well
  T *to = nullptr, *also = nullptr;
  int64_t to_step = 0, also_step = 0;
  if (kind == 0) {
    to = reinterpret_cast<T*>(p.q_out) + t * p.qo_s0 + h0 * p.qo_s1 + lo;
    to_step = G * p.qo_s1;
  } else {
    if (p.k_cache) {
      const int64_t slot = load_slot(p.slots, t, p.slot_dtype);
      if (slot >= (int64_t)p.num_blocks * p.block_size) {
        record_status(p.status, STARKV_EBOUNDS);
      } else if (slot >= 0) {                          // negative: padding, not written
        // a 64-bit division is some hundred instructions
        const int64_t blk = slot <= 0x7fffffff ? (unsigned)slot / (unsigned)p.block_size : slot / p.block_size;
        const int64_t off = slot - blk * p.block_size;
        const int64_t c2 = kind == 1 ? p.kc_s2 : p.vc_s2;
        to = reinterpret_cast<T*>(kind == 1 ? p.k_cache : p.v_cache) + blk * (kind == 1 ? p.kc_s0 : p.vc_s0) +
             off * (kind == 1 ? p.kc_s1 : p.vc_s1) + h0 * c2 + lo;
        to_step = G * c2;
      }
    }
    if (kind == 1 && p.k_out) {
      also = reinterpret_cast<T*>(p.k_out) + t * p.ko_s0 + h0 * p.ko_s1 + lo;
      also_step = G * p.ko_s1;
    }
  }
  if (kind == 2) {
    if (!to) return;
#pragma unroll
    for (int s = 0; s < kSteps; s += kAhead) {
      if (s) load(s);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u < count) {
          *reinterpret_cast<uint2*>(to) = raw[u][0];
          *reinterpret_cast<uint2*>(to + (hi - lo)) = raw[u][1];
        }
        to += to_step;
      }
    }
    return;
  }
  const bool has_to = to != nullptr, has_also = also != nullptr;

  // out_lo = inv * (x_lo a + x_hi b), out_hi = inv * (x_hi c + x_lo d): the weight is in a .. d already
  float4 a = make_float4(1.f, 1.f, 1.f, 1.f), b = make_float4(0.f, 0.f, 0.f, 0.f), c = a, d = b;
  if (!kPart || j < pairs) {
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
  const void* w = kind == 0 ? p.q_weight : p.k_weight;
  if (w) {
    const float4 gl = load4(w, lo, p.w_dtype), gh = load4(w, hi, p.w_dtype);
    a = make_float4(a.x * gl.x, a.y * gl.y, a.z * gl.z, a.w * gl.w);
    b = make_float4(b.x * gh.x, b.y * gh.y, b.z * gh.z, b.w * gh.w);
    c = make_float4(c.x * gh.x, c.y * gh.y, c.z * gh.z, c.w * gh.w);
    d = make_float4(d.x * gl.x, d.y * gl.y, d.z * gl.z, d.w * gl.w);
  }
  const float2 a0 = make_float2(a.x, a.y), a1 = make_float2(a.z, a.w), b0 = make_float2(b.x, b.y),
               b1 = make_float2(b.z, b.w), c0 = make_float2(c.x, c.y), c1 = make_float2(c.z, c.w),
               d0 = make_float2(d.x, d.y), d1 = make_float2(d.z, d.w);
#pragma unroll
  for (int s = 0; s < kSteps; s += kAhead) {
    if (s) {
      if (s >= most) break;
      load(s);
    }
    float inv[kAhead];
    if (w) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float2 l0 = unpack(T{}, raw[u][0].x), l1 = unpack(T{}, raw[u][0].y);
        const float2 h0v = unpack(T{}, raw[u][1].x), h1v = unpack(T{}, raw[u][1].y);
        const float2 q = fma2(h1v, h1v, fma2(h0v, h0v, fma2(l1, l1, mul2(l0, l0))));
        inv[u] = q.x + q.y;
      }
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1)
#pragma unroll
        for (int u = 0; u < kAhead; ++u) inv[u] += __shfl_xor_sync(~0u, inv[u], o);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) inv[u] = rsqrtf(inv[u] * (1.f / D) + p.eps);   // within 2^-22
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float2 l0 = unpack(T{}, raw[u][0].x), l1 = unpack(T{}, raw[u][0].y);
      const float2 h0v = unpack(T{}, raw[u][1].x), h1v = unpack(T{}, raw[u][1].y);
      float2 x0 = mul2(l0, a0), x1 = mul2(l1, a1), y0 = mul2(h0v, c0), y1 = mul2(h1v, c1);
      // not by zeros in b and d: behind the rotated width an infinity stays its own channel's
      if (!kPart || j < pairs) {
        x0 = fma2(h0v, b0, x0);
        x1 = fma2(h1v, b1, x1);
        y0 = fma2(l0, d0, y0);
        y1 = fma2(l1, d1, y1);
      }
      if (w) {
        const float2 iv = make_float2(inv[u], inv[u]);
        x0 = mul2(iv, x0);
        x1 = mul2(iv, x1);
        y0 = mul2(iv, y0);
        y1 = mul2(iv, y1);
      }
      const uint2 x = make_uint2(round2(T{}, x0), round2(T{}, x1)), y = make_uint2(round2(T{}, y0), round2(T{}, y1));
      if (s + u < count) {
        if (has_to) {
          *reinterpret_cast<uint2*>(to) = x;
          *reinterpret_cast<uint2*>(to + (hi - lo)) = y;
        }
        if (has_also) {
          *reinterpret_cast<uint2*>(also) = x;
          *reinterpret_cast<uint2*>(also + (hi - lo)) = y;
        }
      }
      to += to_step;
      also += also_step;
    }
  }
}

template <typename T, int D, int kSteps>
int launch_steps(const NormRopeParams& p, cudaStream_t stream) {
  constexpr int heads = kSteps * (256 / D);            // of a warp
  unsigned qc = (p.num_heads + heads - 1) / heads, kc = (p.num_kv_heads + heads - 1) / heads;
  unsigned chunks = qc + kc * (p.v ? 2 : 1);
  if ((int64_t)p.n * chunks > 0x7fffffff) return STARKV_EINVAL;
  unsigned items = (unsigned)p.n * chunks;
  void* args[] = {const_cast<NormRopeParams*>(&p), &qc, &kc, &chunks, &items};
  const void* fn = p.rot < D ? (const void*)norm_rope_kernel<T, D, kSteps, true>
                             : (const void*)norm_rope_kernel<T, D, kSteps, false>;
  return cudaLaunchKernel(fn, dim3((items + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), args, 0, stream) ==
                 cudaSuccess
             ? STARKV_OK
             : STARKV_ECUDA;
}

template <typename T, int D>
int launch_typed(const NormRopeParams& p, int num_sms, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.n * (p.num_heads + p.num_kv_heads * (p.v ? 2 : 1));
  return rows > (int64_t)num_sms * kManyRows ? launch_steps<T, D, 4>(p, stream) : launch_steps<T, D, 1>(p, stream);
}

}  // namespace

int launch_norm_rope(const NormRopeParams& p, int dtype, int head_dim, int num_sms, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_typed<__nv_bfloat16, 64>(p, num_sms, stream) : launch_typed<__nv_bfloat16, 128>(p, num_sms, stream);
  return head_dim == 64 ? launch_typed<__half, 64>(p, num_sms, stream) : launch_typed<__half, 128>(p, num_sms, stream);
}

}  // namespace starkv

// Attention of one new token per sequence over a paged full-rank K/V cache:
//   out[b, h] = sum_t softmax_t(scale q[b, h] . K[t, h / G]) V[t, h / G],  t < seq_lens[b]
// (G = query heads per KV head), over all tokens or over a list of pages per (sequence,
// KV head).
//
// What bounds it: a K or V row is read once for up to 16 query heads (the M of an MMA; more
// heads of a KV head are units of their own, which read it again), 4 FLOP per head and
// element of 2 bytes, so the cache read is the cost. The tokens of all (sequence, KV
// head) units are laid end to end in items of 64 tokens and every CTA of one wave takes an
// equal run of them, whatever the mix of lengths. A unit that lies inside one CTA's run
// is finished there; a unit that crosses CTA borders leaves one partial (max, sum,
// unnormalised output) per CTA, and join_kernel adds them in the order of the CTAs, so
// results do not depend on timing.
//
// A warp owns 16 tokens of each 64-token tile and a private ring of cp.async stages in
// shared memory (no block barrier between tiles). 16 query heads are the M of
// mma.sync.m16n8k16: S = Q K^T (B from ldmatrix), P from the accumulators' own layout,
// O += P V (B from ldmatrix.trans). mma.sync and not tcgen05: a tile is 16 tokens x at
// most 16 heads, the tensor pipe is idle most of the time either way, and P stays in
// registers instead of a round trip through tensor memory. Cache rows past a sequence's
// end are filled with zeros by the copy itself, so whatever they hold cannot reach the
// sums.
//
// Precision of the weights and of the sums. P is split into parts of the cache's type, so
// that its rounding (2^-9 for bf16) does not show. With G <= 8 two parts share one MMA (rows
// 0-7 and 8-15), with G <= 4 three do (rows 0-3, 8-11 and 4-7, whose scores come from the
// queries of rows 0-3 once more). The tensor core's own accumulation cuts off instead of
// rounding. Shares of outputs that are not the nearest to the exact value, of 1000:
//   f16 in two parts (22 bits), sums of the tensor core                 4.2, f32 operations 7.0
//   bf16, G <= 4: three parts (24 bits), every MMA of P V added to zero
//     and its result to the sum by a rounded f32 addition               0.5, f32 operations 1.0
//     (in two parts and by the tensor core's sums 2.4, at the same time)
//   bf16, G > 4: two parts (16 bits), sums of the tensor core           1.6, f32 operations 0.9
//     (as above, with a third MMA: 0.4, but 192 against 168 us for 32 x 8160 tokens of 64 / 8
//     heads, 116 against 95 with heads of 64: not worth a last place of a bf16 in a thousand)
// The partial form, whose output is f32, is always of the second kind.
#include <algorithm>
#include <type_traits>

#include "flat_items.cuh"
#include "starkv_common.cuh"
#include "starkv_kernels.h"

namespace starkv {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSub = 16;                 // tokens of a warp's share of a tile
constexpr int kTileTok = kWarps * kSub;  // tokens of a tile
constexpr int kTileShift = 6, kWholeShift = 8;
// Units of at most this many tokens are not split and not joined (8 KV heads, 256 tokens:
// one sequence 7.4 us whole and 7.0 split but a launch less for the host, 8 sequences 7.6 and
// 9.3, 64 sequences 15.6 and 20.1; 512 tokens: 10.7 and 7.1, 11.1 and 11.8, 29.5 and 31.6).
constexpr int kWholeTokens = 1 << kWholeShift;
constexpr int kStages = 3;
constexpr int kMaxShares = 384;          // CTAs of one call at most
constexpr int kRowsM = 16;               // query heads of one MMA

template <int D>
struct Ring {
  static constexpr int row_bytes = D * 2;
  static constexpr int op_bytes = kSub * row_bytes;      // K or V of a subtile
  static constexpr int stage_bytes = 2 * op_bytes;
  static constexpr int warp_bytes = kStages * stage_bytes;
  static constexpr int bytes = kWarps * warp_bytes;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (a, b) as two 16-bit values in one register, and what that rounding left over
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Weights are kept times 2^kBias: f16 has no value below 2^-24, so that weights under
// 2^-25 of the largest would leave the output but not the sum (at 131072 tokens up to
// 2^-8 of it); times 2^10 that is 2^-18 and the largest weight, 1024, is far from f16's
// end. The factor is the same in output and sum.
template <typename T>
constexpr float weight_bias() {
  return std::is_same<T, __half>::value ? 10.f : 0.f;
}

// (a, b) += (c, d)
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  asm("{.reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %3}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}"
      : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ bool finite4(float4 v) {
  return fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < INFINITY;
}
// An infinite V meets parts of its weight that are 0 or below it, and weights of shares that
// have become 0: NaN. With weights > 0 the sum is that of the channel's infinities and NaN,
// so where a result of a finite denominator is not finite those alone are added up:
// `odd` takes what of v is not finite, and replaces what it has of acc.
__device__ __forceinline__ void add_odd(float4& odd, float4 v) {
  odd.x += fabsf(v.x) < INFINITY ? 0.f : v.x;
  odd.y += fabsf(v.y) < INFINITY ? 0.f : v.y;
  odd.z += fabsf(v.z) < INFINITY ? 0.f : v.z;
  odd.w += fabsf(v.w) < INFINITY ? 0.f : v.w;
}
__device__ __forceinline__ void take_odd(float4& acc, float4 odd) {
  acc.x = odd.x == 0.f ? acc.x : odd.x;
  acc.y = odd.y == 0.f ? acc.y : odd.y;
  acc.z = odd.z == 0.f ? acc.z : odd.z;
  acc.w = odd.w == 0.f ? acc.w : odd.w;
}

// Tokens that a (sequence, KV head) unit of sequence b covers.
__device__ __forceinline__ int unit_tokens(const PagedAttnParams& p, int b) {
  const int L = min(max(p.seq_lens[b], 0), p.max_len);
  if (!p.pages) return L;
  return min(p.top, (int)(((unsigned)L + (unsigned)p.block_size - 1u) / (unsigned)p.block_size)) * p.block_size;
}
// Work items (runs of 2^item_shift tokens) of a unit of sequence b.
__device__ __forceinline__ int unit_items(const PagedAttnParams& p, int b) {
  return b < p.n ? (unit_tokens(p, b) + (1 << p.item_shift) - 1) >> p.item_shift : 0;
}

// f32 partials: per share two slots (its first unit, its last one) of
// [rows][D] outputs, then [rows] max and [rows] sum, padded to whole 16-byte pieces.
__host__ __device__ constexpr int part_floats(int rows, int D) { return rows * D + ((2 * rows + 3) & ~3); }
__device__ __forceinline__ float* part_slot(const PagedAttnParams& p, int D, int share, int which) {
  return p.part + (int64_t)(2 * share + which) * part_floats(p.part_rows, D);
}

template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 v) {
  uint2 u;
  u.x = pack2(T{}, v.x, v.y);
  u.y = pack2(T{}, v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = u;
}

// Final output of query head `head` of sequence b, four channels from column c.
// `o` unnormalised, `m` the largest raw q . k.
template <typename T>
__device__ __forceinline__ void store_out(const PagedAttnParams& p, int b, int head, int c, float4 o, float m, float l) {
  const int64_t at = b * p.o_s0 + head * p.o_s1 + c;
  if (p.m_out) {
    constexpr float back = std::is_same<T, __half>::value ? 1.f / 1024.f : 1.f;   // 2^-weight_bias
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) =
        make_float4(o.x * back, o.y * back, o.z * back, o.w * back);
    if (c == 0) {
      p.m_out[(int64_t)b * p.num_heads + head] = m * p.scale;
      p.l_out[(int64_t)b * p.num_heads + head] = l * back;
    }
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // no token: 0; a NaN sum stays NaN
  store4(reinterpret_cast<T*>(p.out) + at, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// kHeads: 4, 8 or 16, the most query heads of a unit; 4 for bf16 alone (24 x 8192 tokens of
// 32 / 32 heads back to back under the power cap: three parts in one MMA 488 us, the third
// in one of its own 542, two parts 483). kF32: the partial form; the MMAs of Q K^T add to
// zero as well (131071 tokens: 4.8e-7 off, relative in norm, against 6.1e-7), which does not
// show in 16 bits (the 24 x 8192 tokens 483 us, with it 495).
template <typename T, int D, int kHeads, bool kSparse, bool kF32>
__global__ void __launch_bounds__(kThreads, 2) paged_attn_kernel(const PagedAttnParams p) {
  using R = Ring<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red_m[kWarps][kRowsM], red_l[kWarps][kRowsM];
  constexpr int kChunks = D / 8;             // 16-byte pieces of a row
  constexpr int kRowsPer = 32 / kChunks;     // rows of one warp-wide copy
  constexpr int kKSteps = D / 16;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int qr = lane >> 2, qc = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * R::warp_bytes;
  const float c_log2 = p.scale * 1.4426950408889634f;
  constexpr float kBias = weight_bias<T>();
  constexpr bool kTwo = kHeads > 8, kFour = kHeads <= 4;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kRounded = kFour || kF32, kThird = kRounded && kBf16;
  static_assert(!kFour || kBf16, "rows 4-7 hold the third part");

  // the joining kernel's blocks may take the place of CTAs that are done; they wait for all
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // sequences without a token have no tile: their outputs are written here
  for (int b = blockIdx.x; b < p.n; b += gridDim.x) {
    if (unit_tokens(p, b) > 0) continue;
    for (int i = threadIdx.x; i < p.num_heads * (D / 4); i += kThreads)
      store_out<T>(p, b, i / (D / 4), (i % (D / 4)) * 4, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
  }

  const auto count = [&](int b) { return unit_items(p, b) * p.units; };
  FlatItems<decltype(count)> all(count, p.n, lane);
  const int shares = min((int)gridDim.x, all.total);
  if (kSparse && p.after_select) asm volatile("griddepcontrol.wait;" ::: "memory");   // the lists are written
  if ((int)blockIdx.x >= shares) return;
  const int g0 = share_begin(all.total, blockIdx.x, shares), g1 = share_begin(all.total, blockIdx.x + 1, shares);
  int b, first;
  all.place(g0, b, first);
  int items = unit_items(p, b);
  int unit = (g0 - first) / items;
  int t0 = (g0 - first) % items;

  for (int g = g0; g < g1;) {
    const int t1 = min(items, t0 + (g1 - g));
    const int hk = unit / p.head_groups, hg = unit % p.head_groups;
    const int head0 = hk * p.group + hg * kRowsM;
    const int rows = min(kRowsM, p.group - hg * kRowsM);
    const int L = min(max(p.seq_lens[b], 0), p.max_len);
    const int tokens = unit_tokens(p, b);
    const int32_t* bt = p.block_table + b * p.bt_s0;
    const int32_t* list = kSparse ? p.pages + b * p.pg_s0 + hk * p.pg_s1 : nullptr;
    const char* kbase = reinterpret_cast<const char*>(p.k) + hk * p.k_s2 * 2;
    const char* vbase = reinterpret_cast<const char*>(p.v) + hk * p.v_s2 * 2;
    // this warp's 16-token subtiles of the segment
    const int base0 = (t0 << p.item_shift) + warp * kSub;
    const int end = (int)min((int64_t)t1 << p.item_shift, (int64_t)tokens);
    const int subs = max(end - base0 + kTileTok - 1, 0) / kTileTok;

    // Q as A fragments
    uint32_t qa[kKSteps][4];
    {
      const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_s0 + (int64_t)head0 * p.q_s1;
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        const int d = kk * 16 + 2 * qc;
        const int row0 = kFour ? qr & 3 : qr;
        const T* r0 = q + (int64_t)row0 * p.q_s1 + d;
        const T* r1 = q + (int64_t)(qr + 8) * p.q_s1 + d;
        qa[kk][0] = row0 < rows ? *reinterpret_cast<const uint32_t*>(r0) : 0u;
        qa[kk][2] = row0 < rows ? *reinterpret_cast<const uint32_t*>(r0 + 8) : 0u;
        qa[kk][1] = kTwo && qr + 8 < rows ? *reinterpret_cast<const uint32_t*>(r1) : 0u;
        qa[kk][3] = kTwo && qr + 8 < rows ? *reinterpret_cast<const uint32_t*>(r1 + 8) : 0u;
      }
    }

    // Block of the page that holds position `pos`-style index `idx` of the unit's token
    // list, and that position (-1: not a token).
    auto locate = [&](int idx, int& pos) -> int {
      pos = -1;
      if (idx >= tokens) return 0;
      const int at = idx / p.block_size, off = idx - at * p.block_size;
      int page = at;
      if (kSparse) {
        page = list[at];
        if (page < 0 || page >= p.max_blocks) return 0;
      }
      const int64_t ps = (int64_t)page * p.block_size + off;
      if (ps >= L) return 0;
      int blk = bt[page * p.bt_s1];
      if ((unsigned)blk >= (unsigned)p.num_blocks) {
        record_status(p.status, STARKV_EBOUNDS);
        blk = 0;
      }
      pos = (int)ps;
      return blk;
    };
    // pages of whole subtiles: one lookup per subtile, 32 of them ahead by the lanes
    int cur_blk = 0, cur_pos = -1, nxt_blk = 0, nxt_pos = -1;
    if (p.page16) nxt_blk = locate((int)min((int64_t)base0 + lane * kTileTok, (int64_t)tokens), nxt_pos);

    auto issue = [&](int i) -> uint32_t {   // returns the subtile's valid-token bits
      const uint32_t dst = ring + (i % kStages) * R::stage_bytes;
      const int base = base0 + i * kTileTok;
      const int chunk = lane % kChunks, sub = lane / kChunks;
      uint32_t valid;
      if (p.page16) {
        if ((i & 31) == 0) {
          cur_blk = nxt_blk;
          cur_pos = nxt_pos;
          nxt_blk = locate((int)min((int64_t)base + (int64_t)(32 + lane) * kTileTok, (int64_t)tokens), nxt_pos);
        }
        const int blk = __shfl_sync(~0u, cur_blk, i & 31), pos = __shfl_sync(~0u, cur_pos, i & 31);
        const int nv = pos < 0 ? 0 : min(kSub, L - pos);
        valid = (1u << nv) - 1u;
        const int off = pos < 0 ? 0 : pos % p.block_size;
        const char* ks = kbase + ((int64_t)blk * p.k_s0 + (int64_t)(off + sub) * p.k_s1) * 2 + chunk * 16;
        const char* vs = vbase + ((int64_t)blk * p.v_s0 + (int64_t)(off + sub) * p.v_s1) * 2 + chunk * 16;
#pragma unroll
        for (int r = 0; r < kSub; r += kRowsPer) {
          const int row = r + sub;
          const uint32_t o = dst + row * R::row_bytes + ((chunk ^ (row & 7)) << 4);
          const int n = row < nv ? 16 : 0;
          cp_async16(o, n ? ks + (int64_t)r * p.k_s1 * 2 : kbase, n);
          cp_async16(o + R::op_bytes, n ? vs + (int64_t)r * p.v_s1 * 2 : vbase, n);
        }
      } else {
        int pos;
        const int blk = locate(base + (lane & 15), pos);
        valid = __ballot_sync(~0u, pos >= 0) & 0xffffu;
        const int off = pos < 0 ? 0 : pos % p.block_size;
        const int64_t ko = ((int64_t)blk * p.k_s0 + (int64_t)off * p.k_s1) * 2;
        const int64_t vo = ((int64_t)blk * p.v_s0 + (int64_t)off * p.v_s1) * 2;
#pragma unroll
        for (int r = 0; r < kSub; r += kRowsPer) {
          const int row = r + sub;
          const int64_t kr = __shfl_sync(~0u, ko, row), vr = __shfl_sync(~0u, vo, row);
          const uint32_t o = dst + row * R::row_bytes + ((chunk ^ (row & 7)) << 4);
          const int n = (valid >> row) & 1 ? 16 : 0;
          cp_async16(o, n ? kbase + kr + chunk * 16 : kbase, n);
          cp_async16(o + R::op_bytes, n ? vbase + vr + chunk * 16 : vbase, n);
        }
      }
      return valid;
    };

    float o[2 * kKSteps][4];
#pragma unroll
    for (int j = 0; j < 2 * kKSteps; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    // valid bits of the kStages - 1 = 2 subtiles in flight
    uint32_t va = 0, vb = 0;
    static_assert(kStages == 3, "two subtiles in flight");
    // (one place that issues: the kernel's first pass over its code is fetched from memory)
    for (int i = -2; i < subs; ++i) {
      cp_wait<kStages - 2>();
      __syncwarp();   // every lane's copies of subtile i are in; every lane is done with subtile i - 1
      const uint32_t valid = va;
      va = vb;
      if (i + 2 < subs) vb = issue(i + 2);
      cp_commit();
      if (i < 0) continue;
      const uint32_t kt = ring + (i % kStages) * R::stage_bytes, vt = kt + R::op_bytes;
      const int mi = lane >> 3, rr = lane & 7;
      // ---- S = Q K^T, 16 tokens ----
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      {
        const int row = (mi >> 1) * 8 + rr;
        const uint32_t a = kt + row * R::row_bytes;
#pragma unroll
        for (int kk = 0; kk < kKSteps; ++kk) {
          uint32_t r[4];
          ldsm4(a + (((2 * kk + (mi & 1)) ^ rr) << 4), r);
          if (kF32) {
            float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816<T>(t0, qa[kk], r[0], r[1]);
            mma16816<T>(t1, qa[kk], r[2], r[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s0[e] += t0[e];
              s1[e] += t1[e];
            }
          } else {
            mma16816<T>(s0, qa[kk], r[0], r[1]);
            mma16816<T>(s1, qa[kk], r[2], r[3]);
          }
        }
      }
      if (valid != 0xffffu) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (!((valid >> (2 * qc + e)) & 1)) s0[e] = s0[2 + e] = -INFINITY;
          if (!((valid >> (8 + 2 * qc + e)) & 1)) s1[e] = s1[2 + e] = -INFINITY;
        }
      }
      // ---- online softmax ----
      float x0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1]));
      float x1 = kTwo ? fmaxf(fmaxf(s0[2], s0[3]), fmaxf(s1[2], s1[3])) : -INFINITY;
      x0 = fmaxf(x0, __shfl_xor_sync(~0u, x0, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(~0u, x0, 2));
      if (kTwo) {
        x1 = fmaxf(x1, __shfl_xor_sync(~0u, x1, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(~0u, x1, 2));
      }
      if (__any_sync(~0u, x0 > m0 || (kTwo && x1 > m1))) {
        // the maxima move: what is there so far is scaled down (-inf - -inf only before the first token)
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float f0 = n0 == m0 ? 1.f : ex2((m0 - n0) * c_log2), f1 = n1 == m1 ? 1.f : ex2((m1 - n1) * c_log2);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
        const float fr = kTwo ? f1 : f0;   // G <= 8: rows 8-15 hold the low parts of rows 0-7
#pragma unroll
        for (int j = 0; j < 2 * kKSteps; ++j) {
          o[j][0] *= f0;
          o[j][1] *= f0;
          o[j][2] *= fr;
          o[j][3] *= fr;
        }
      }
      const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
      const float p00 = ex2(fmaf(s0[0] - u0, c_log2, kBias)), p01 = ex2(fmaf(s0[1] - u0, c_log2, kBias));
      const float p02 = ex2(fmaf(s1[0] - u0, c_log2, kBias)), p03 = ex2(fmaf(s1[1] - u0, c_log2, kBias));
      l0 += (p00 + p01) + (p02 + p03);
      uint32_t pa[4], pl[4], t1a = 0, t3a = 0;
      pa[0] = pack2(T{}, p00, p01);
      pa[2] = pack2(T{}, p02, p03);
      const float2 h0 = unpack2(T{}, pa[0]), h2 = unpack2(T{}, pa[2]);
      pl[0] = pack2(T{}, p00 - h0.x, p01 - h0.y);
      pl[2] = pack2(T{}, p02 - h2.x, p03 - h2.y);
      if (kTwo) {
        const float p10 = ex2(fmaf(s0[2] - u1, c_log2, kBias)), p11 = ex2(fmaf(s0[3] - u1, c_log2, kBias));
        const float p12 = ex2(fmaf(s1[2] - u1, c_log2, kBias)), p13 = ex2(fmaf(s1[3] - u1, c_log2, kBias));
        l1 += (p10 + p11) + (p12 + p13);
        pa[1] = pack2(T{}, p10, p11);
        pa[3] = pack2(T{}, p12, p13);
        const float2 h1 = unpack2(T{}, pa[1]), h3 = unpack2(T{}, pa[3]);
        pl[1] = pack2(T{}, p10 - h1.x, p11 - h1.y);
        pl[3] = pack2(T{}, p12 - h3.x, p13 - h3.y);
        if (kThird) {
          const float2 e1 = unpack2(T{}, pl[1]), e3 = unpack2(T{}, pl[3]);
          t1a = pack2(T{}, p10 - h1.x - e1.x, p11 - h1.y - e1.y);
          t3a = pack2(T{}, p12 - h3.x - e3.x, p13 - h3.y - e3.y);
        }
      } else {
        pa[1] = pl[0];
        pa[3] = pl[2];
      }
      uint32_t pt[4] = {0u, 0u, 0u, 0u};
      if (kThird) {
        // what the two parts leave (2^-16) goes into a third
        const float2 e0 = unpack2(T{}, pl[0]), e2 = unpack2(T{}, pl[2]);
        pt[0] = pack2(T{}, p00 - h0.x - e0.x, p01 - h0.y - e0.y);
        pt[2] = pack2(T{}, p02 - h2.x - e2.x, p03 - h2.y - e2.y);
        if (kTwo) {
          pt[1] = t1a;
          pt[3] = t3a;
        }
        if (kFour && qr >= 4) {
          pa[0] = pt[0];
          pa[1] = 0u;
          pa[2] = pt[2];
          pa[3] = 0u;
        }
      }
      // ---- O += P V ----
      {
        const int row = (mi & 1) * 8 + rr;
        const uint32_t a = vt + row * R::row_bytes;
#pragma unroll
        for (int j = 0; j < kKSteps; ++j) {
          uint32_t r[4];
          ldsm4_t(a + (((2 * j + (mi >> 1)) ^ rr) << 4), r);
          float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
          float(&x)[4] = kRounded ? t0 : o[2 * j];
          float(&y)[4] = kRounded ? t1 : o[2 * j + 1];
          if (kThird && !kFour) {   // the smallest part first
            mma16816<T>(x, pt, r[0], r[1]);
            mma16816<T>(y, pt, r[2], r[3]);
          }
          if (kTwo) {
            mma16816<T>(x, pl, r[0], r[1]);
            mma16816<T>(y, pl, r[2], r[3]);
          }
          mma16816<T>(x, pa, r[0], r[1]);
          mma16816<T>(y, pa, r[2], r[3]);
          if (kRounded) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              add2(o[2 * j][e], o[2 * j][e + 1], t0[e], t0[e + 1]);
              add2(o[2 * j + 1][e], o[2 * j + 1][e + 1], t1[e], t1[e + 1]);
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();   // no copy in flight, no warp reads its ring: the space holds the warps' outputs now

    // ---- the four warps' results, added in warp order ----
    l0 += __shfl_xor_sync(~0u, l0, 1);
    l0 += __shfl_xor_sync(~0u, l0, 2);
    l1 += __shfl_xor_sync(~0u, l1, 1);
    l1 += __shfl_xor_sync(~0u, l1, 2);
    if (qc == 0) {
      red_m[warp][qr] = m0;
      red_l[warp][qr] = l0;
      red_m[warp][qr + 8] = m1;
      red_l[warp][qr + 8] = l1;
    }
    float* red = reinterpret_cast<float*>(smem);   // [warp][rows][D]
#pragma unroll
    for (int j = 0; j < 2 * kKSteps; ++j) {
      if (!kTwo) {
        o[j][0] += o[j][2];
        o[j][1] += o[j][3];
        if (kFour) {
          o[j][0] += __shfl_xor_sync(~0u, o[j][0], 16);
          o[j][1] += __shfl_xor_sync(~0u, o[j][1], 16);
        }
      }
      if (qr < rows)
        *reinterpret_cast<float2*>(red + (warp * kRowsM + qr) * D + j * 8 + 2 * qc) = make_float2(o[j][0], o[j][1]);
      if (kTwo && qr + 8 < rows)
        *reinterpret_cast<float2*>(red + (warp * kRowsM + qr + 8) * D + j * 8 + 2 * qc) =
            make_float2(o[j][2], o[j][3]);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == items;
    float* part = whole ? nullptr : part_slot(p, D, blockIdx.x, g > g0);
    for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
      const int row = i / (D / 4), c = (i % (D / 4)) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red_m[w][row]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = red_m[w][row];
        const float f = mw == m ? 1.f : ex2((mw - m) * c_log2);
        const float4 v = *reinterpret_cast<const float4*>(red + (w * kRowsM + row) * D + c);
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
        l += f * red_l[w][row];
      }
      if (!finite4(acc) && l == l) {   // infinities or NaN in V
        float4 odd = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i = t0 << p.item_shift; i < end; ++i) {
          int pos;
          const int blk = locate(i, pos);
          if (pos < 0) continue;
          const int64_t at = ((int64_t)blk * p.v_s0 + (int64_t)(pos % p.block_size) * p.v_s1 + c) * 2;
          const uint2 raw = *reinterpret_cast<const uint2*>(vbase + at);
          const float2 a = unpack2(T{}, raw.x), b = unpack2(T{}, raw.y);
          add_odd(odd, make_float4(a.x, a.y, b.x, b.y));
        }
        take_odd(acc, odd);
      }
      if (whole) {
        store_out<T>(p, b, head0 + row, c, acc, m, l);
      } else {
        *reinterpret_cast<float4*>(part + row * D + c) = acc;
        if (c == 0) {
          part[p.part_rows * D + row] = m;
          part[p.part_rows * (D + 1) + row] = l;
        }
      }
    }
    __syncthreads();   // the space is the rings' again

    g += t1 - t0;
    t0 = 0;
    if (g < g1 && ++unit == p.units) {
      unit = 0;
      do items = unit_items(p, ++b);
      while (items == 0 && b < p.n);
      if (b >= p.n) break;   // not reached: g < g1 <= total
    }
  }
}

// Adds the partials of the units that cross a border between shares. Block i: if the
// border after share i lies inside a unit, and share i is the unit's first, the unit's
// shares i .. j are added. A thread takes four channels of a row; the groups of
// rows * D / 4 threads take every kLanes-th share, four at a time in flight, and the
// groups' sums are added in order.
constexpr int kJoinThreads = 512;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const PagedAttnParams p, int grid) {
  constexpr int kCols = D / 4;
  constexpr int kAhead = 4;
  __shared__ float4 so[kJoinThreads];
  __shared__ float2 sml[kJoinThreads];
  const int width = p.part_rows * kCols, lanes = kJoinThreads / width;   // part_rows <= 16: width <= 512
  const auto count = [&](int b) { return unit_items(p, b) * p.units; };
  FlatItems<decltype(count)> all(count, p.n, threadIdx.x & 31);
  const int total = all.total;
  const int shares = min(grid, total);
  const int i0 = blockIdx.x;
  int u0 = 0, u1 = 0, b = 0, hk = 0, hg = 0;
  bool mine = false;
  if (i0 + 1 < shares) {
    const int border = share_begin(total, i0 + 1, shares);
    int first;
    all.place(border, b, first);
    const int items = unit_items(p, b);
    const int unit = (border - first) / items;
    u0 = first + unit * items;
    u1 = u0 + items;
    hk = unit / p.head_groups;
    hg = unit % p.head_groups;
    mine = u0 < border && share_begin(total, i0, shares) <= u0;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the partials are written
  if (!mine) return;
  // share of the unit's last item: the largest i with share_begin(i) <= u1 - 1
  const int i1 = (int)(((int64_t)u1 * shares + total - 1) / total) - 1;
  const int late = share_begin(total, i0, shares) < u0;   // the unit is not the first of share i0
  const int col = threadIdx.x % kCols, row = threadIdx.x / kCols % p.part_rows, grp = threadIdx.x / width;
  const bool in = grp < lanes && row < min(kRowsM, p.group - hg * kRowsM);
  const float c_log2 = p.scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int ib = in ? i0 + grp : i1 + 1; ib <= i1; ib += lanes * kAhead) {
    float pm[kAhead], pl[kAhead];
    float4 v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = ib + u * lanes;
      pm[u] = -INFINITY;
      pl[u] = 0.f;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i <= i1) {
        const float* part = part_slot(p, D, i, i == i0 && late);
        pm[u] = part[p.part_rows * D + row];
        pl[u] = part[p.part_rows * (D + 1) + row];
        v[u] = *reinterpret_cast<const float4*>(part + row * D + col * 4);
      }
    }
    float nm = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) nm = fmaxf(nm, pm[u]);
    const float fa = m == nm ? 1.f : ex2((m - nm) * c_log2);
    acc.x *= fa;
    acc.y *= fa;
    acc.z *= fa;
    acc.w *= fa;
    l *= fa;
    m = nm;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float f = pm[u] == m ? 1.f : ex2((pm[u] - m) * c_log2);
      acc.x += f * v[u].x;
      acc.y += f * v[u].y;
      acc.z += f * v[u].z;
      acc.w += f * v[u].w;
      l += f * pl[u];
    }
  }
  so[threadIdx.x] = acc;
  sml[threadIdx.x] = make_float2(m, l);
  __syncthreads();
  if (grp || !in) return;
  float M = m;
  for (int w = 1; w < lanes; ++w) M = fmaxf(M, sml[threadIdx.x + w * width].x);
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f;
  for (int w = 0; w < lanes; ++w) {
    const float2 ml = sml[threadIdx.x + w * width];
    const float4 v = so[threadIdx.x + w * width];
    const float f = ml.x == M ? 1.f : ex2((ml.x - M) * c_log2);
    acc.x += f * v.x;
    acc.y += f * v.y;
    acc.z += f * v.z;
    acc.w += f * v.w;
    l += f * ml.y;
  }
  if (!finite4(acc) && l == l) {
    float4 odd = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i = i0; i <= i1; ++i)
      add_odd(odd, *reinterpret_cast<const float4*>(part_slot(p, D, i, i == i0 && late) + row * D + col * 4));
    take_odd(acc, odd);
  }
  store_out<T>(p, b, hk * p.group + hg * kRowsM + row, col * 4, acc, M, l);
}

template <typename T, int D, bool kSparse, bool kF32>
const void* attn_fn(int group) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    if (group <= 4) return (const void*)paged_attn_kernel<T, D, 4, kSparse, kF32>;
  return group <= 8 ? (const void*)paged_attn_kernel<T, D, 8, kSparse, kF32>
                    : (const void*)paged_attn_kernel<T, D, 16, kSparse, kF32>;
}

template <typename T, int D>
int launch_typed(const PagedAttnParams& p, int num_sms, cudaStream_t stream) {
  const void* fn = p.pages ? p.m_out ? attn_fn<T, D, true, true>(p.group) : attn_fn<T, D, true, false>(p.group)
                   : p.m_out ? attn_fn<T, D, false, true>(p.group) : attn_fn<T, D, false, false>(p.group);
  const int smem = Ring<D>::bytes;
  if (const int st = allow_smem(fn, smem)) return st;
  PagedAttnParams q = p;
  q.item_shift = p.max_unit_tokens <= kWholeTokens ? kWholeShift : kTileShift;
  const auto most = [&] {
    return (int64_t)p.n * p.units * ((p.max_unit_tokens + ((int64_t)1 << q.item_shift) - 1) >> q.item_shift);
  };
  while (most() > 0x7fffffff && q.item_shift < 30) ++q.item_shift;   // 32-bit item numbers
  if (most() > 0x7fffffff) return STARKV_EINVAL;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>({2 * num_sms, kMaxShares, most()}));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_select;   // behind pick_kernel alone may the launch come early
  void* args[] = {&q};
  if (cudaLaunchKernelExC(&cfg, fn, args) != cudaSuccess) return STARKV_ECUDA;
  if (grid == 1 || p.max_unit_tokens <= kWholeTokens) return STARKV_OK;   // no unit is in two shares
  cfg.gridDim = dim3((unsigned)grid - 1);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  int g = grid;
  void* jargs[] = {&q, &g};
  if (cudaLaunchKernelExC(&cfg, (const void*)join_kernel<T, D>, jargs) != cudaSuccess) return STARKV_ECUDA;
  return STARKV_OK;
}

}  // namespace

size_t paged_attn_workspace_bytes(int rows, int head_dim, int max_tokens) {
  if (max_tokens <= kWholeTokens) return 0;   // every unit is one item
  return (size_t)2 * kMaxShares * part_floats(rows, head_dim) * sizeof(float);
}

int launch_paged_attn(const PagedAttnParams& p, int dtype, int head_dim, int num_sms, cudaStream_t stream) {
  if (dtype == STARKV_BF16)
    return head_dim == 64 ? launch_typed<__nv_bfloat16, 64>(p, num_sms, stream)
                          : launch_typed<__nv_bfloat16, 128>(p, num_sms, stream);
  return head_dim == 64 ? launch_typed<__half, 64>(p, num_sms, stream)
                        : launch_typed<__half, 128>(p, num_sms, stream);
}

}  // namespace starkv

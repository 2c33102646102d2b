// Equal division of a ragged batch's work: the items of all sequences are laid end to end
// and share i of `shares` takes items share_begin(i) .. share_begin(i + 1), whatever the
// mix of lengths. The launch keeps the batch's items below 2^31.
#pragma once

#include <stdint.h>

namespace starkv {

// First item of share i of `shares`.
__device__ __forceinline__ int share_begin(int total, int i, int shares) {
  return (int)((int64_t)total * i / shares);
}

// Items of a whole batch; count(b) is the number of sequence b's items, 0 <= b < n. One
// whole warp computes it; up to 32 sequences are read once.
template <class Count>
struct FlatItems {
  const Count& count;
  const int n, lane;
  int incl, mine;   // of the 32 sequences looked at last
  int total;

  __device__ FlatItems(const Count& count_, int n_, int lane_) : count(count_), n(n_), lane(lane_) {
    scan(0);
    total = __shfl_sync(~0u, incl, 31);
    if (n > 32) {
      int rest = 0;
      for (int b = lane + 32; b < n; b += 32) rest += count(b);
      total += (int)__reduce_add_sync(~0u, (unsigned)rest);
    }
  }
  __device__ void scan(int b0) {
    mine = b0 + lane < n ? count(b0 + lane) : 0;
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
  }
  // The sequence that holds item g < total and its first item; to be called once.
  __device__ void place(int g, int& seq, int& first) {
    int base = 0;
    for (int b0 = 0;;) {
      const uint32_t hit = __ballot_sync(~0u, base + incl > g);
      if (hit) {
        const int l = __ffs(hit) - 1;
        seq = b0 + l;
        first = base + __shfl_sync(~0u, incl - mine, l);
        return;
      }
      base += __shfl_sync(~0u, incl, 31);
      if ((b0 += 32) >= n) break;
      scan(b0);
    }
    seq = n;
    first = base;
  }
};

}  // namespace starkv

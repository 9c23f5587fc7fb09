// How the paged attention kernels share their work out, on the device and from the batch's
// numbers as they are in memory (so a captured call follows them when it is replayed).
//
// A unit is a (sequence, KV head) or a (sequence, KV head, query tile); its cost is the key tiles
// that it sees. All units' key tiles stand in one row, and CTA c of n takes tiles [cW/n, (c+1)W/n)
// of the W: every CTA the same number, whatever the lengths. A unit that crosses from one CTA to
// the next is cut there: each piece leaves (max, sum, unnormalised output) partials, and the last
// piece to arrive merges them in the order of the CTAs. A CTA has at most two cut units, the one
// that it enters in the middle (slot 2c) and the one that it leaves (slot 2c + 1), so the
// partials' memory depends on the grid alone. A unit's arrivals are counted at the CTA that
// starts it (counters[c]; the last piece sets it back to zero).
#pragma once

#include "fa_paged.h"
#include "fa_ptx.cuh"

namespace fa {

// CTA c's first tile of W shared among n. (A 64-bit division takes some hundred instructions, which
// short calls wait for: 32 bits where they do, n being at most 4096.)
__device__ __forceinline__ int64_t share_begin(int64_t w, int c, int n) {
  if (w < (1 << 20)) return int64_t(uint32_t(w) * uint32_t(c) / uint32_t(n));
  return int64_t((unsigned long long)(w) * (unsigned long long)(c) / (unsigned long long)(n));
}

// The CTA whose share holds tile t.
__device__ __forceinline__ int share_owner(int64_t w, int64_t t, int n) {
  if (w < (1 << 20)) return int(((uint32_t(t) + 1) * uint32_t(n) - 1) / uint32_t(w));
  return int((((unsigned long long)(t) + 1) * (unsigned long long)(n)-1) / (unsigned long long)(w));
}

// How many times `per` goes into t.
__device__ __forceinline__ int whole_times(int64_t t, int64_t per) {
  return t < (1 << 30) ? int(uint32_t(t) / uint32_t(per)) : int(t / per);
}

// Exclusive prefix sums over the CTA's threads of one value each, and the total (every thread);
// `scratch` holds a value per warp.
template <int kThreads>
__device__ __forceinline__ int64_t block_prefix(int64_t x, int64_t* scratch, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += y;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < warp) before += scratch[i];
    all += scratch[i];
  }
  __syncthreads();
  *total = all;
  return before + inc - x;
}

}  // namespace fa

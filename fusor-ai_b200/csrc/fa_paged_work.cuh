// How the paged attention kernels share their work out, on the device and from the batch's
// numbers as they are in memory (so a captured call follows them when it is replayed).
//
// A unit is a (sequence, KV head) or a (sequence, KV head, query tile); its cost is the key tiles
// that it sees. All units' key tiles stand in one row, and CTA c takes tiles [cQ, (c + 1)Q) of it, Q
// = ceil(all / CTAs): every CTA the same number (the last may have fewer), whatever the lengths. A
// unit that crosses from one CTA to the next is cut there: each piece leaves (max, sum,
// unnormalised output) partials, and the last piece to arrive merges them in the order of the CTAs.
// A CTA has at most two cut units, the one that it enters in the middle (slot 2c) and the one that
// it leaves (slot 2c + 1), so the partials' memory depends on the grid alone. A unit's arrivals are
// counted at the CTA that starts it (counters[c]; the last piece sets it back to zero).
#pragma once

#include "fa_paged.h"
#include "fa_ptx.cuh"

namespace fa {

// Tiles of a CTA's share: ceil(w / n). (A 64-bit division takes some hundred instructions, which
// short calls wait for: 32 bits where they do.)
__device__ __forceinline__ int64_t share_size(int64_t w, int n) {
  return w < (1 << 30) ? int64_t((uint32_t(w) + n - 1) / uint32_t(n)) : (w + n - 1) / n;
}

// The first and the last CTA that a unit of `cost` tiles from global tile unit0 on is shared among,
// asked by a CTA (of shares of q) that has tiles of it.
__device__ __forceinline__ void share_owners(int64_t q, int cta, int64_t unit0, int cost, int* c0,
                                             int* c1) {
  const int64_t begin = q * cta;
  const uint32_t q32 = uint32_t(min(q, int64_t(0x7fffffff)));  // (distances within a unit fit 31 bits)
  const uint32_t before = unit0 < begin ? uint32_t(begin - unit0) : 0u;
  *c0 = cta - int((before + q32 - 1) / q32);
  *c1 = cta + int(uint32_t(unit0 + cost - 1 - begin) / q32);
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

// Attention of a few packed rows over a paged cache: single tokens, and spans whose rows x query
// heads of a KV head fit in 16 columns (bound by the bytes of the pages: each is read once).
//
// The products run transposed on mma.sync, so that the keys fill the 16 rows and a KV head's packed
// rows (column c = row offset x group + query head) the 8 or 16 columns:
//   S^T (16 keys x columns) = K Q^T, then O^T (head_dim x columns) += V^T P^T.
// Each product's A operand comes straight from a page's rows: the order of the elements within
// the sums is free (Q is laid out to match, O is written back by the same order), so a thread's
// fragments are 16-byte vectors of its keys' rows. tcgen05 would want converted tiles written to
// shared memory and read again; at 16 columns the tensor pipe is idle either way, and what counts
// is instructions per byte:
//   8-bit keys go into m16n8k32 as they are; a query row is held in 15 bits as two 8-bit parts
//     (q = 128 hi + lo, scaled to its largest element), whose products are exact integers, so
//     that a score is off by at most half a step, 2^-15 of |q|max, of each element;
//   8-bit values become f16 integers in registers (exact, three instructions a pair: the bytes of
//     two keys side by side, 1024 + 128 put under them by one logical operation, subtracted), and
//     the probabilities take the values' scales: w = 2^(score + log2 scale - M) in f16, M the
//     running maximum of that exponent (the row's sum keeps the scores' own maximum), so that
//     the weights that matter are in f16's range whatever the scales;
//   bf16 keys and values as they are (values by transposing loads), probabilities in bf16.
// Scores, maxima, sums and outputs are f32. The maximum is lazy: moved when a score exceeds it by
// 2^8.
//
// A CTA has 4 warps, each with its own ring of stages of 32 (or 16) keys filled by cp.async (16
// consecutive keys lie in one page, so a stage holds contiguous blocks of keys, of values, and
// their scales): no barrier among the warps until a unit ends, and a warp loads ahead across
// units. Rows of a stage are swizzled by 16-byte chunks so that both products' reads are free of
// bank conflicts. Work is shared out as fa_paged_work.cuh says.
// Measured: 64 sequences of 512 to 8192 positions, 32/8 heads of 128: 165 us over bf16 pages (1.02
// GB, 6.2 TB/s: the rate of a copy), 118 us over 8-bit pages (578 MB, 4.9 TB/s: 56 % of the issue
// slots; its loads alone take 98 us). 131072 positions of one sequence, 16/8 heads, 8-bit pages: 61
// us. Three sequences of about 1000: 7.9 us, all latency (the plan, the pages, the merge).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_paged_work.cuh"

namespace fa {

constexpr int kTokWarps = 4;
constexpr int kTokThreads = kTokWarps * 32;

template <int D, bool Q8, int NT>
struct TokShape {
  static constexpr int kCols = 8 * NT;
  static constexpr int kElem = Q8 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kChunks = kRowBytes / 16;        // 16-byte chunks of a row
  static constexpr int kPer = 16 / kElem;               // elements of a chunk
  static constexpr int kBlock = 16 * kRowBytes;         // 16 keys (or values)
  static constexpr int kHalves = kRowBytes <= 128 ? 2 : 1;  // blocks of 16 keys in a stage
  static constexpr int kTile = 16 * kHalves * kTokWarps;    // keys of a CTA's tile
  static constexpr int kHalfBytes = 2 * kBlock + (Q8 ? 128 : 0);
  static constexpr int kStageBytes = kHalves * kHalfBytes;
  static constexpr int kStages = kRowBytes <= 64 ? 3 : 2;
  static constexpr int kSteps = D / 16;                 // m tiles of O (and 16-bit k steps of S)
  static constexpr int kRing = kTokWarps * kStages * kStageBytes;
  static constexpr int kMergeRow = D + 4;               // floats: O, then max and sum (16-byte rows)
  // At a unit's end each warp leaves its rows in the stage that it read last, if they fit there.
  static constexpr bool kInStage = kCols * kMergeRow * 4 <= kStageBytes;
  // resident CTAs per SM that the registers allow
  static constexpr int kCtas = D == 256 ? (NT == 1 ? 2 : 1) : (NT == 1 ? 3 : 2);
  // dynamic shared memory for batches of `cols` packed rows and `sequences` sequences
  static int smem(int cols, int sequences) {
    return kRing + (kInStage ? 0 : kTokWarps * cols * kMergeRow * 4) + sequences * 24 + 8;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 x 8 matrix of 16-bit elements transposed over the warp.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two signed bytes, at bits 0-7 and 16-23 of w, as f16: the byte plus 128 becomes the low bits of
// 1024 + (byte + 128), less 1152 (all exact). Bits 8-15 and 24-31 are ignored.
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t w) {
  const uint32_t x = (w & 0x00FF00FFu) ^ 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// m16n8k32 of signed bytes.
__device__ __forceinline__ void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices of 16-bit elements, transposed: lane l gives row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A walk over the CTA's share of the units' tiles: unit (s, h), its tiles [tile, tile_end) within
// this share, and the unit's own numbers. All of it is uniform over the CTA.
struct TokWalk {
  int64_t t, t_end;    // the global tile of `tile`, and the share's end
  int s, h;
  int tile, tile_end;  // of the unit's tiles
  int tiles;           // the unit's tiles
  int lo, hi;          // key positions that any of its rows sees
  int row0, n, first;
};

struct TokPlan {
  const int64_t* before;  // [sequences + 1]: tiles of the sequences before, of one KV head each
  const int4* spans;      // [sequences]: first row, rows, first position, first key seen
  int kvh;
};

// A sequence's part in the token kernel: its span, the first key that its rows see, and their
// tiles (0 if it is empty or the chunk kernel's, -1 if it is out of range).
template <int kTile>
__device__ __forceinline__ int token_tiles(const PagedAttendArgs& a, int s, int4* span) {
  PagedSpan sp;
  *span = make_int4(0, 0, 0, 0);
  if (!paged_span(a.spans, a.pool.page_shift, s, &sp)) return -1;
  if (sp.n == 0 || int64_t(sp.n) * a.group > a.token_cols) return 0;
  int lo, unused;
  paged_keys(a.kind, a.window, sp.first, sp.first + sp.n, &lo, &unused);
  *span = make_int4(sp.row0, sp.n, sp.first, lo);
  return (sp.first + sp.n + kTile - 1) / kTile - lo / kTile;
}

// Moves the walk to the unit that holds global tile w->t (w->s at or before it); false at the
// share's end.
__device__ __forceinline__ bool token_seek(const TokPlan& plan, TokWalk* w) {
  if (w->t >= w->t_end) return false;
  while (plan.before[w->s + 1] * plan.kvh <= w->t) ++w->s;
  const int4 sp = plan.spans[w->s];
  w->row0 = sp.x;
  w->n = sp.y;
  w->first = sp.z;
  w->lo = sp.w;
  w->hi = sp.z + sp.y;
  w->tiles = int(plan.before[w->s + 1] - plan.before[w->s]);
  const int64_t rest = w->t - plan.before[w->s] * plan.kvh;
  w->h = whole_times(rest, w->tiles);
  w->tile = int(rest - int64_t(w->h) * w->tiles);
  w->tile_end = int(min(int64_t(w->tiles), int64_t(w->tile) + (w->t_end - w->t)));
  return true;
}

// Elements 4 v .. 4 v + 3 of a packed row's output: o / l (a row that sees no key, its pages out of
// range, is zero).
template <int D>
__device__ __forceinline__ void token_write(const PagedAttendArgs& a, int row0, int h, int col, int v,
                                            float4 o, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  const int64_t at = int64_t(row0 + col / a.group) * a.out_stride +
                     int64_t(h * a.group + col % a.group) * D + v * 4;
  if (a.out_bf16) {
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    const uint2 w = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
    if (a.out_vec) {
      *reinterpret_cast<uint2*>(p) = w;
    } else {
      p[0] = uint16_t(w.x); p[1] = uint16_t(w.x >> 16);
      p[2] = uint16_t(w.y); p[3] = uint16_t(w.y >> 16);
    }
  } else {
    float* p = static_cast<float*>(a.out) + at;
    if (a.out_vec) *reinterpret_cast<float4*>(p) = o;
    else { p[0] = o.x; p[1] = o.y; p[2] = o.z; p[3] = o.w; }
  }
}

// The partials of a unit's pieces (of CTAs c0 ..) merged into the output, by the whole CTA of the
// piece that arrived last. Bound by trips to L2, one for each group of loads: of more than eight
// pieces four lanes share a vector of the output, each with a quarter of the pieces, and a piece's
// maximum is loaded beside its output (the sums are rescaled as the maximum grows), so that 8
// pieces, or 32, cost one trip; in an order that does not depend on who arrived last. Not inlined:
// the loop over the keys has its registers to itself.
template <int D>
__device__ __noinline__ void token_merge(const PagedAttendArgs& a, int row0, int h, int cols, int c0,
                                         int pieces) {
  constexpr int kVecs = D / 4, kGroup = 8;
  const int lanes = pieces > 8 ? 4 : 1;
  const int sub = threadIdx.x & (lanes - 1);
  for (int i = threadIdx.x / lanes; i < cols * kVecs; i += kTokThreads / lanes) {
    const int col = i / kVecs, v = i % kVecs;
    // piece j's row, in slot 2 (c0 + j), or 2 c0 + 1 for j = 0
    const int64_t at0 = int64_t(2 * c0) * kPagedTokenCols + col;
    const float* const o0 = a.part_o + at0 * D + 4 * v;
    const float* const ml0 = a.part_ml + at0 * 2;
    float mm = -INFINITY, ll = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int b = sub; b < pieces; b += lanes * kGroup) {
      float2 ml[kGroup];
      float4 x[kGroup];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        // (past the end the last piece's again, without a weight)
        const int j = min(b + lanes * k, pieces - 1);
        const int row = (j == 0 ? 1 : 2 * j) * kPagedTokenCols;
        ml[k] = __ldcg(reinterpret_cast<const float2*>(ml0 + row * 2));
        x[k] = __ldcg(reinterpret_cast<const float4*>(o0 + row * D));
      }
      float top = mm;
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        if (b + lanes * k >= pieces) ml[k] = make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[k].x);
      }
      const float e = mm == -INFINITY ? 1.0f : exp2_approx(mm - top);
      mm = top;
      ll *= e;
      acc = make_float4(acc.x * e, acc.y * e, acc.z * e, acc.w * e);
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        // a piece that saw no key has sum 0 (or NaN, which stays)
        const float f = ml[k].x == -INFINITY ? 0.0f : exp2_approx(ml[k].x - mm);
        ll += ml[k].x == -INFINITY ? ml[k].y : f * ml[k].y;
        acc.x = fmaf(f, x[k].x, acc.x); acc.y = fmaf(f, x[k].y, acc.y);
        acc.z = fmaf(f, x[k].z, acc.z); acc.w = fmaf(f, x[k].w, acc.w);
      }
    }
    if (lanes == 4) {  // (whole warps have the same items)
      __syncwarp();
      float top = mm;
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float f = mm == -INFINITY ? 1.0f : exp2_approx(mm - top);
      ll *= f;
      acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      if (lanes == 1) break;
      ll += __shfl_xor_sync(0xffffffffu, ll, off);
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, off);
      acc.y += __shfl_xor_sync(0xffffffffu, acc.y, off);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, off);
      acc.w += __shfl_xor_sync(0xffffffffu, acc.w, off);
    }
    if (sub == 0) token_write<D>(a, row0, h, col, v, acc, ll);
  }
}

template <int D, bool Q8, int NT>
__global__ void __launch_bounds__(kTokThreads, (TokShape<D, Q8, NT>::kCtas))
    paged_tokens_kernel(const __grid_constant__ PagedAttendArgs a) {
  using S = TokShape<D, Q8, NT>;
  constexpr int kRB = S::kRowBytes, kC = S::kChunks, kPer = S::kPer;
  constexpr int KH = S::kHalves, kTile = S::kTile;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t scratch[kTokWarps];
  __shared__ int arrived;
  const int mcols = a.merge_cols;  // packed rows that any sequence has
  int4* spans = reinterpret_cast<int4*>(
      smem + S::kRing + (S::kInStage ? 0 : kTokWarps * mcols * S::kMergeRow * 4));
  int64_t* before = reinterpret_cast<int64_t*>(spans + a.spans.sequences);

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  unsigned char* ring = smem + warp * (S::kStages * S::kStageBytes);

  pdl_wait();
  pdl_trigger();

  // ---- the plan: tiles before every sequence --------------------------------------------------
  const int nseq = a.spans.sequences, kvh = a.pool.kv_heads;
  {
    const int each = (nseq + kTokThreads - 1) / kTokThreads;
    const int s0 = min(nseq, int(threadIdx.x) * each), s1 = min(nseq, s0 + each);
    int64_t sum = 0;
    for (int s = s0; s < s1; ++s) {
      const int n = token_tiles<kTile>(a, s, &spans[s]);
      if (n < 0) atomicOr(a.err, kErrPagedSpan);
      sum += max(n, 0);
      before[s] = sum;  // inclusive within the thread's sequences, for now
    }
    int64_t total;
    const int64_t base = block_prefix<kTokThreads>(sum, scratch, &total);
    int64_t prev = base;
    for (int s = s0; s < s1; ++s) {
      const int64_t inc = base + before[s];
      before[s] = prev;
      prev = inc;
    }
    if (threadIdx.x == 0) before[nseq] = total;
    __syncthreads();
  }
  const TokPlan plan{before, spans, kvh};
  const int64_t work = before[nseq] * kvh;
  if (work == 0) return;
  const int64_t share = share_size(work, int(min(int64_t(gridDim.x), work)));  // a tile at least
  const int cta = blockIdx.x;
  if (share * cta >= work) return;

  TokWalk lw, cw;  // the loads' walk and the products' walk
  lw.t = cw.t = share * cta;
  lw.t_end = cw.t_end = min(work, share * (cta + 1));
  {
    int s0 = 0, s1 = nseq;  // the last s with before[s] * kvh <= t
    while (s1 - s0 > 1) {
      const int mid = (s0 + s1) / 2;
      if (before[mid] * kvh <= cw.t) s0 = mid; else s1 = mid;
    }
    lw.s = cw.s = s0;
  }

  // ---- loads: one stage at a time --------------------------------------------------------------
  const int shift = a.pool.page_shift;
  bool more = token_seek(plan, &lw);
  int next_page[KH];  // the pages of the next stage's 16s of keys (-1: none of them is seen)
  auto stage_pos = [&](const TokWalk& w) { return (w.lo / kTile + w.tile) * kTile + warp * (16 * KH); };
  auto fetch_pages = [&]() {
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      next_page[h] = -1;
      if (!more) continue;
      const int pos = stage_pos(lw) + 16 * h;
      if (pos < lw.hi && pos + 16 > lw.lo)
        next_page[h] = __ldg(a.spans.tables + int64_t(lw.s) * a.spans.table_stride + (pos >> shift));
    }
  };
  fetch_pages();
  uint32_t ring_live = 0;  // a bit per 16s: its keys are there (a page in range, some key seen)
  // chunk q = lane + 32 i of a block: its row and its place in the stage, by i's parity where the
  // swizzle's row bits change
  const int q_key = lane / kC, q_c = lane % kC;
  auto issue = [&](int stage) {
    if (!more) return;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      const int pos = stage_pos(lw) + 16 * h;
      const bool some = pos < lw.hi && pos + 16 > lw.lo;
      const bool live = some && paged_page_ok(next_page[h], a.pool.pages);
      if (some && !live && lane == 0) atomicOr(a.err, kErrPagedPage);
      const uint32_t bit = 1u << (stage * KH + h);
      ring_live = live ? ring_live | bit : ring_live & ~bit;
      if (!live) continue;
      const int64_t row = ((int64_t(next_page[h]) * kvh + lw.h) << shift) + (pos & ((1 << shift) - 1));
      const unsigned char* ks = a.pool.keys + row * kRB + lane * 16;
      const unsigned char* vs = a.pool.values + row * kRB + lane * 16;
      const uint32_t kd = smem_u32(ring + stage * S::kStageBytes + h * S::kHalfBytes), vd = kd + S::kBlock;
      const int64_t at = row + (lane & 15);
      const float* sc = lane < 16 ? a.pool.key_scales : a.pool.value_scales;
      auto copy = [&](bool all) {
#pragma unroll
        for (int i = 0; i < kC / 2; ++i) {
          const int key = q_key + i * (32 / kC);
          const int ck = kC >= 8 ? q_c ^ ((key & 1) << 2) : q_c;
          const int cv = kC < 8 ? q_c : Q8 ? q_c ^ (((key >> 1) & 3) << 1) : q_c ^ (key & 7);
          const uint32_t bytes = all || (pos + key >= lw.lo && pos + key < lw.hi) ? 16u : 0u;
          cp_async16(kd + key * kRB + ck * 16, ks + i * 512, bytes);
          cp_async16(vd + key * kRB + cv * 16, vs + i * 512, bytes);
        }
        if constexpr (Q8) {
          const int key = lane & 15;
          const uint32_t bytes = all || (pos + key >= lw.lo && pos + key < lw.hi) ? 4u : 0u;
          cp_async4(vd + S::kBlock + lane * 4, sc + at, bytes);
        }
      };
      // rows outside the keys seen (a page's stale end, or before the window) come as zeros
      if (pos >= lw.lo && pos + 16 <= lw.hi) copy(true);
      else copy(false);
    }
    ++lw.t;
    if (++lw.tile == lw.tile_end) more = token_seek(plan, &lw);
    fetch_pages();
  };
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    issue(i);
    cp_async_commit();
  }

  // ---- the products ---------------------------------------------------------------------------
  int stage = 0;
  while (token_seek(plan, &cw)) {
    // This lane's query column g (+ 8): its fragments. 8-bit pages: bytes of hi and lo for the
    // lane's chunks, two words for each product of 32 elements; bf16: pairs.
    constexpr int kFrags = Q8 ? D / 32 : S::kSteps;
    uint32_t qf[NT][kFrags][2], ql[NT][Q8 ? kFrags : 1][2];
    float qscale[NT][2];  // of this lane's score columns 2 t4, 2 t4 + 1
    int col_lo[NT][2], col_hi[NT][2];
    int lo_max = 0, hi_min = 0x7fffffff;  // keys that every column sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + g;
      const int r = col / a.group;
      const bool valid = r < cw.n;
      float x[S::kSteps][4];
      const int64_t at = int64_t(cw.row0 + r) * a.q_stride +
                         int64_t(cw.h * a.group + col % a.group) * D;
#pragma unroll
      for (int i = 0; i < kC / 4; ++i) {
        const int64_t e0 = at + (t4 + 4 * i) * kPer;
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
          float(&y)[4] = x[i * (kPer / 4) + j];
          y[0] = y[1] = y[2] = y[3] = 0.0f;
          if (!valid) continue;
          if (a.q_bf16) {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + e0 + 4 * j);
            y[0] = bf16_lo(w.x); y[1] = bf16_hi(w.x); y[2] = bf16_lo(w.y); y[3] = bf16_hi(w.y);
          } else {
            const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + e0 + 4 * j);
            y[0] = w.x; y[1] = w.y; y[2] = w.z; y[3] = w.w;
          }
        }
      }
      float down = 1.0f;
      if constexpr (Q8) {
        float top = 0.0f, total = 0.0f;  // (total: NaN if an element is)
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            top = fmaxf(top, fabsf(x[k][e]));
            total += x[k][e] * 0.0f;
          }
#pragma unroll
        for (int off = 1; off <= 2; off <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          total += __shfl_xor_sync(0xffffffffu, total, off);
        }
        // steps of top / 16256 (hi up to 127); elements below 1e-33 throughout are kept as zeros
        top = fmaxf(top, 1e-33f);
        const float up = 16256.0f / top;
        down = top / 16256.0f + total;  // a row with an infinity or a NaN scores NaN
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k) {
          uint32_t hw = 0, lw_ = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = __float2int_rn(fminf(fmaxf(x[k][e] * up, -16256.0f), 16256.0f));
            const int hi = (v + 64) >> 7, lo = v - (hi << 7);
            hw |= uint32_t(hi & 0xff) << (8 * e);
            lw_ |= uint32_t(lo & 0xff) << (8 * e);
          }
          qf[nt][k / 2][k & 1] = hw;
          ql[nt][k / 2][k & 1] = lw_;
        }
      } else {
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k) {
          qf[nt][k][0] = pack_bf16x2(x[k][0], x[k][1]);
          qf[nt][k][1] = pack_bf16x2(x[k][2], x[k][3]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int cc = nt * 8 + 2 * t4 + j, rr = cc / a.group;
        qscale[nt][j] = a.scale_log2 * __shfl_sync(0xffffffffu, down, (2 * t4 + j) * 4);
        col_lo[nt][j] = 0;
        col_hi[nt][j] = 0;  // a column without a row sees nothing
        if (rr < cw.n)
          paged_keys(a.kind, a.window, cw.first + rr, cw.hi, &col_lo[nt][j], &col_hi[nt][j]);
      }
    }
    {
      int l0, h0;
      paged_keys(a.kind, a.window, cw.first, cw.hi, &l0, &hi_min);
      paged_keys(a.kind, a.window, cw.first + cw.n - 1, cw.hi, &lo_max, &h0);
    }

    float o[S::kSteps][NT][4];
    float m[NT][2], l[NT][2];
    float mo[NT][2];  // 8-bit pages: the maximum of the weights' exponents (O is in its unit)
    bool poisoned[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = mo[nt][0] = mo[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
      poisoned[nt][0] = poisoned[nt][1] = false;
#pragma unroll
      for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][nt][e] = 0.0f;
    }

    for (; cw.tile < cw.tile_end; ++cw.tile, ++cw.t) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();
      const int fill = stage == 0 ? S::kStages - 1 : stage - 1;  // the stage read last time
      issue(fill);
      cp_async_commit();
      const unsigned char* base = ring + stage * S::kStageBytes;
      const uint32_t live = (ring_live >> (stage * KH)) & ((1u << KH) - 1);
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      if (live == 0) continue;  // uniform over the warp
      const int pos0 = stage_pos(cw);

      // S^T: keys g and g + 8 of each 16
      float s[KH][NT][4];  // e: key g + 8 (e / 2), column 2 t4 + e % 2
      bool whole[KH];
      bool grow = false;
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        const unsigned char* kb = base + h * S::kHalfBytes;
        const int pos = pos0 + 16 * h;
        whole[h] = pos >= lo_max && pos + 16 <= hi_min && ((live >> h) & 1u);
        float f[NT][4];
        if constexpr (Q8) {
          int ch[NT][4], cl[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) ch[nt][e] = cl[nt][e] = 0;
#pragma unroll
          for (int i = 0; i < kC / 4; ++i) {
            const int c = t4 + 4 * i, cs = kC >= 8 ? c ^ ((g & 1) << 2) : c;
            const uint4 ra = *reinterpret_cast<const uint4*>(kb + g * kRB + cs * 16);
            const uint4 rb = *reinterpret_cast<const uint4*>(kb + (g + 8) * kRB + cs * 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16832(ch[nt], ra.x, rb.x, ra.y, rb.y, qf[nt][2 * i][0], qf[nt][2 * i][1]);
              mma16832(cl[nt], ra.x, rb.x, ra.y, rb.y, ql[nt][2 * i][0], ql[nt][2 * i][1]);
              mma16832(ch[nt], ra.z, rb.z, ra.w, rb.w, qf[nt][2 * i + 1][0], qf[nt][2 * i + 1][1]);
              mma16832(cl[nt], ra.z, rb.z, ra.w, rb.w, ql[nt][2 * i + 1][0], ql[nt][2 * i + 1][1]);
            }
          }
          const float* sk = reinterpret_cast<const float*>(kb + 2 * S::kBlock);
          const float ks[2] = {sk[g], sk[g + 8]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[nt][e] = float(ch[nt][e] * 128 + cl[nt][e]) * (qscale[nt][e & 1] * ks[e >> 1]);
        } else {
          float sc[NT][2][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[nt][0][e] = sc[nt][1][e] = 0.0f;
#pragma unroll
          for (int i = 0; i < kC / 4; ++i) {
            const int c = t4 + 4 * i, cs = kC >= 8 ? c ^ ((g & 1) << 2) : c;
            const uint4 ra = *reinterpret_cast<const uint4*>(kb + g * kRB + cs * 16);
            const uint4 rb = *reinterpret_cast<const uint4*>(kb + (g + 8) * kRB + cs * 16);
            const uint32_t fa_[4] = {ra.x, rb.x, ra.y, rb.y}, fb_[4] = {ra.z, rb.z, ra.w, rb.w};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<false>(sc[nt][0], fa_, qf[nt][2 * i][0], qf[nt][2 * i][1]);
              mma16816<false>(sc[nt][1], fb_, qf[nt][2 * i + 1][0], qf[nt][2 * i + 1][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) f[nt][e] = (sc[nt][0][e] + sc[nt][1][e]) * qscale[nt][e & 1];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][nt][e] = f[nt][e];
        if (!whole[h]) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int p = pos + g + 8 * (e >> 1);
              if (!((live >> h) & 1u) || p < col_lo[nt][e & 1] || p >= col_hi[nt][e & 1])
                s[h][nt][e] = -INFINITY;
            }
        }
      }
      // the weights' exponents: over 8-bit pages with the values' scales
      float y[Q8 ? KH : 1][Q8 ? NT : 1][4];
      if constexpr (Q8) {
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          const float* sv = reinterpret_cast<const float*>(base + h * S::kHalfBytes + 2 * S::kBlock) + 16;
          const float lv[2] = {log2_approx(sv[g]), log2_approx(sv[g + 8])};  // (stale if not live)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              y[h][nt][e] = s[h][nt][e] + lv[e >> 1];
          if (!whole[h]) {  // (a scale that is not finite stays out of the columns that do not see it)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(s[h][nt][e] > -INFINITY)) y[h][nt][e] = s[h][nt][e];
          }
        }
      }
      auto top_of = [&](const auto& x, int nt, int j) {
        float top = fmaxf(x[0][nt][j], x[0][nt][2 + j]);
        if constexpr (KH == 2) top = fmaxf(top, fmaxf(x[1][nt][j], x[1][nt][2 + j]));
        return top;
      };
      auto moves = [](float top, float m) { return top > m + 8.0f || (m == -INFINITY && top > -INFINITY); };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          grow = grow || moves(top_of(s, nt, j), m[nt][j]);
          if constexpr (Q8) grow = grow || moves(top_of(y, nt, j), mo[nt][j]);
        }
      if (__any_sync(0xffffffffu, grow)) {
        // a maximum moves to its column's largest over the warp; what it was gets the ratio
        auto move = [&](float top, float& m) {
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          float alpha = 1.0f;
          if (top > m) {
            if (m > -INFINITY) alpha = exp2_approx(m - top);
            m = top;
          }
          return alpha;
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            alpha[j] = move(top_of(s, nt, j), m[nt][j]);
            l[nt][j] *= alpha[j];
            if constexpr (Q8) alpha[j] = move(top_of(y, nt, j), mo[nt][j]);
          }
#pragma unroll
          for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][nt][e] *= alpha[e & 1];
        }
      }
      uint32_t pf[KH][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float off[2], off_o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          off[j] = m[nt][j] == -INFINITY ? 0.0f : m[nt][j];
          off_o[j] = Q8 ? (mo[nt][j] == -INFINITY ? 0.0f : mo[nt][j]) - 6.0f : 0.0f;
        }
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_approx(s[h][nt][e] - off[e & 1]);
            l[nt][e & 1] += p;
            if constexpr (Q8) w[e] = exp2_approx(y[h][nt][e] - off_o[e & 1]);
            else w[e] = p;
          }
          pf[h][nt][0] = movmatrix(Q8 ? pack_f16(w[0], w[1]) : pack_bf16x2(w[0], w[1]));
          pf[h][nt][1] = movmatrix(Q8 ? pack_f16(w[2], w[3]) : pack_bf16x2(w[2], w[3]));
        }
      }

      // O^T
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        if (!((live >> h) & 1u)) continue;  // (stale bytes: not to be multiplied even by zero)
        const unsigned char* vb = base + h * S::kHalfBytes + S::kBlock;
        if constexpr (Q8) {
          // values of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
          constexpr int kPiece = kC >= 8 ? 16 : 8;  // bytes a lane takes of a row at a time
          constexpr int kPieces = kRB / (8 * kPiece), kWords = kPiece / 4;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            uint32_t wv[4][kWords];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int key = 2 * t4 + (q & 1) + 8 * (q >> 1);
              if constexpr (kPiece == 16) {
                const int c = (g + 8 * i) ^ (((key >> 1) & 3) << 1);
                const uint4 r = *reinterpret_cast<const uint4*>(vb + key * kRB + c * 16);
                wv[q][0] = r.x; wv[q][1] = r.y; wv[q][2] = r.z; wv[q][3] = r.w;
              } else {
                const uint2 r = *reinterpret_cast<const uint2*>(vb + key * kRB + g * 8);
                wv[q][0] = r.x; wv[q][1] = r.y;
              }
            }
#pragma unroll
            for (int x = 0; x < kWords; ++x)
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                // bytes 2 b and 2 b + 1 of word x: two elements, an m tile
                const uint32_t sel0 = b == 0 ? 0x0400u : 0x0602u, sel1 = b == 0 ? 0x0501u : 0x0703u;
                const uint32_t fr[4] = {bytes_to_f16(__byte_perm(wv[0][x], wv[1][x], sel0)),
                                        bytes_to_f16(__byte_perm(wv[0][x], wv[1][x], sel1)),
                                        bytes_to_f16(__byte_perm(wv[2][x], wv[3][x], sel0)),
                                        bytes_to_f16(__byte_perm(wv[2][x], wv[3][x], sel1))};
                const int mt = i * (kPiece / 2) + 2 * x + b;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<true>(o[mt][nt], fr, pf[h][nt][0], pf[h][nt][1]);
              }
          }
        } else {
          // lane: row lane % 8 of matrix lane / 8 (elements 0-7 and 8-15 of keys 0-7, then of 8-15)
          const int key = (lane & 7) + 8 * (lane >> 4), half = (lane >> 3) & 1;
          const uint32_t row = smem_u32(vb) + key * kRB;
          uint32_t bad = 0;  // which of the lane's four keys has a value that is not finite
#pragma unroll
          for (int mt = 0; mt < S::kSteps; ++mt) {
            uint32_t fr[4];
            ldmatrix4_trans(fr, row + (((2 * mt + half) ^ (key & 7)) * 16));
            if (!whole[h]) {
              // a value that is not finite would reach columns that do not see its key (0 x inf):
              // it is taken out here and every column that sees it marked below
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                if ((fr[x] & 0x7F80u) == 0x7F80u) { fr[x] &= 0xFFFF0000u; bad |= 1u << (x & 2); }
                if ((fr[x] & 0x7F800000u) == 0x7F800000u) { fr[x] &= 0xFFFFu; bad |= 2u << (x & 2); }
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<false>(o[mt][nt], fr, pf[h][nt][0], pf[h][nt][1]);
          }
          if (!whole[h]) {
            // the keys with such a value, over the warp: bit k for key k of the 16
            uint32_t keys = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if ((bad >> q) & 1u) keys |= 1u << (2 * t4 + (q & 1) + 8 * (q >> 1));
            keys = __reduce_or_sync(0xffffffffu, keys);
            for (uint32_t rest = keys; rest != 0; rest &= rest - 1) {
              const int p = pos0 + 16 * h + __ffs(rest) - 1;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  poisoned[nt][j] = poisoned[nt][j] || (p >= col_lo[nt][j] && p < col_hi[nt][j]);
            }
          }
        }
      }
    }

    // every warp's rows: in its stage read last (the same for all, as are the tiles)
    const int done = stage == 0 ? S::kStages - 1 : stage - 1;
    auto merge_of = [&](int w) {
      return reinterpret_cast<float*>(
          S::kInStage ? smem + w * (S::kStages * S::kStageBytes) + done * S::kStageBytes
                      : smem + S::kRing + w * (mcols * S::kMergeRow * 4));
    };
    __syncwarp();  // (the stage's last reads are done)

    // ---- the unit's (or piece's) end: the warps' parts merged -----------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
        if (poisoned[nt][j]) l[nt][j] = __int_as_float(0x7fffffff);
        const int col = nt * 8 + 2 * t4 + j;
        if (col >= mcols) continue;
        if constexpr (Q8) {
          // O to the sum's unit
          const float f = mo[nt][j] == -INFINITY || m[nt][j] == -INFINITY
                              ? 0.0f : exp2_approx(mo[nt][j] - m[nt][j] - 6.0f);
#pragma unroll
          for (int k = 0; k < S::kSteps; ++k) {
            o[k][nt][j] *= f;
            o[k][nt][2 + j] *= f;
          }
        }
        float* row = merge_of(warp) + col * S::kMergeRow;
        if (g == 0) { row[D] = m[nt][j]; row[D + 1] = l[nt][j]; }
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k) {
          if constexpr (Q8) {
            // m tile k: elements 2 (k % (kElems / 2)) + {0, 1} of the lane's piece k / (kElems / 2)
            constexpr int kElems = kC >= 8 ? 16 : 8;  // of a lane's piece of a row
            const int d = (g + 8 * (k / (kElems / 2))) * kElems + 2 * (k % (kElems / 2));
            *reinterpret_cast<float2*>(row + d) = make_float2(o[k][nt][j], o[k][nt][2 + j]);
          } else {
            row[16 * k + g] = o[k][nt][j];
            row[16 * k + g + 8] = o[k][nt][2 + j];
          }
        }
      }
    __syncthreads();
    const int64_t unit0 = plan.before[cw.s] * kvh + int64_t(cw.h) * cw.tiles;  // its first tile
    int c0, c1;
    share_owners(share, cta, unit0, cw.tiles, &c0, &c1);
    const int pieces = c1 - c0 + 1;
    const int cols = cw.n * a.group;
    constexpr int kVecs = D / 4;  // float4s of a column
    const int slot = 2 * cta + (cta == c0 ? 1 : 0);
    for (int i = threadIdx.x; i < cols * kVecs; i += kTokThreads) {
      const int col = i / kVecs, v = i % kVecs;
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < kTokWarps; ++w)
        mm = fmaxf(mm, merge_of(w)[col * S::kMergeRow + D]);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kTokWarps; ++w) {
        const float* row = merge_of(w) + col * S::kMergeRow;
        const float f = row[D] == -INFINITY ? 0.0f : exp2_approx(row[D] - mm);
        // a warp that saw no key has sum 0 (or NaN, which stays)
        ll += row[D] == -INFINITY ? row[D + 1] : f * row[D + 1];
        const float4 x = *reinterpret_cast<const float4*>(row + 4 * v);
        acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
      }
      if (pieces == 1) {
        // a row that sees no key (every page out of range) is zero
        token_write<D>(a, cw.row0, cw.h, col, v, acc, ll);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (int64_t(slot) * kPagedTokenCols + col) * D + 4 * v) = acc;
        if (v == 0)
          *reinterpret_cast<float2*>(a.part_ml + (int64_t(slot) * kPagedTokenCols + col) * 2) =
              make_float2(mm, ll);
      }
    }
    if (pieces > 1) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int before_me = atomicAdd(&a.counters[c0], 1);
        arrived = before_me == pieces - 1;
        if (arrived) a.counters[c0] = 0;
        __threadfence();  // (the other pieces' arrivals, before the whole CTA reads what they left)
      }
      __syncthreads();
      if (arrived) {
        token_merge<D>(a, cw.row0, cw.h, cols, c0, pieces);
      }
    }
    __syncthreads();  // the merge rows are free again
  }
}

}  // namespace fa

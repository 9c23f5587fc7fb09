// Attention of many rows over a paged cache on the tensor cores (tcgen05; bound by the products
// and the exponentials of long chunks, by the pages' bytes of short ones).
//
// A query tile is 128 packed rows of one KV head: 128 / group rows of the sequence times its
// `group` query heads (packed row p is row offset p / group, head p % group), so a page is read
// once for all the heads that share it. A unit is NQ query tiles (two in ping-pong up to head_dim
// 128; one at 256, whose output takes half of TMEM) and the key tiles that its rows see; units are
// shared out and cut as fa_paged_work.cuh says (causal chunks, ragged batches and single long
// rows all come out even).
//
// Warp roles:
//   softmax groups (4 warps for each query tile; thread = packed row = TMEM lane): Q rows into
//     shared memory, then per key tile the scores from TMEM, masked where the tile is on an edge,
//     online softmax with a lazy maximum, probabilities back to TMEM as bf16, and the output;
//   loaders (two warps for the keys and two for the values; four and four over 8-bit pages): the
//     pages' rows into the swizzled tiles that the products read. bf16 pages by cp.async straight
//     to their places; 8-bit pages through registers, a tile's bytes loaded while the one before
//     it is converted to f16;
//   one warp: TMEM and the MMA issue (one thread).
// 8-bit pages are dequantised to f16 (2^-11 of the value, an eighth of bf16's rounding) with each
// tile's scales divided by a power of two, 2^k for the keys and 2^v for the values, that takes the
// largest to [2^8, 2^9): none overflows. 2^k multiplies the tile's scores (with the softmax's scale),
// v is added to their base-2 exponents, so that the probabilities carry 2^v and the outputs of all
// tiles stay in one unit; the row's sum takes 2^-v back out. Where a tile's scales lie more than 2^8
// apart, each of its keys has a k, or a v, of its own: in the unit of a far larger one f16 would lose
// it (all of it from 2^-33 on), for rows too that do not see the large one or give it no weight.
// (Per-key multiplications of scores and probabilities in every tile would cost every softmax thread
// 64 16-byte shared loads a tile.) Probabilities are f16 too, up to 2^15 (the maximum is lazy by 2^8,
// and 2^7 are added for f16's small end). A word's bytes come out as 0, 2, 1, 3
// (two pairs without a byte permutation): Q's rows and the output's columns follow that order.
//
// A tile's scores are one product of 128 keys (of 64, the tensor core takes as long for each MMA:
// it waits for Q's rows out of shared memory; 0.75 against 0.57 ms for 2048 rows of 32/8 heads of
// 128 after 14336 positions of bf16 pages). The softmax and P.V go 64 keys at a time, so that P.V
// of the first half runs during the second half's exponentials: per tile the order is PV0, S0',
// PV1, S1' as in fmha2_kernel (fa_fmha2.cuh), one group's exponentials beside the other's
// products. One query tile (head_dim 256): tiles of 64 keys, two score buffers, S' before PV.
//
// Keys that no row of a unit sees come as zeros (a page's stale end may hold anything). On edge
// tiles, where some rows see a key and others do not, a value that is not finite would reach all
// of them (0 x inf): the loaders take it out and mark its key, and the rows that see the key get
// a NaN sum. Every wait is bounded (mbar_wait).
//
// Measured: 2048 rows after 14336 positions, 32/8 heads of 128 (515 GFLOP): 0.569 ms over bf16 pages
// (905 TFLOP/s, the softmax and the handshakes between the roles; one tile at a time on its way), 0.789
// ms over 8-bit pages (653 TFLOP/s: the conversion next to it; 54 % of the load/store data path, tensor
// pipe 31 %; 2.7 ms if every tile's scales lie far apart: such a tile's softmax is a rolled loop). Five
// chunks of 100 to 999 rows under a window of 1024, 8/2 heads of 256: 98 us, shares of about 12
// tiles a CTA whose fixed costs (plan 6-9 thousand cycles, queries 4-16, merge 20) weigh as much.
#pragma once

#include "fa_decode.cuh"
#include "fa_paged_tokens.cuh"
#include "fa_tc.cuh"

namespace fa {

template <int D, bool Q8>
struct ChunkShape {
  static constexpr int NQ = D == 256 ? 1 : 2;     // query tiles of a unit
  static constexpr int BM = 128;
  static constexpr int BN = D == 256 ? 64 : 128;  // keys of a tile (a stage)
  static constexpr int kSubs = BN / 64;           // blocks of 64 keys: the softmax's steps and P.V's
  static constexpr int kLoad = Q8 ? 128 : 64;     // loaders of the keys, and of the values
  static constexpr int kThreads = 2 * kLoad + NQ * 128 + 128;  // loaders, softmax, issuer
  // Two query tiles: the registers of the warpgroups, which add up to the launch's (16 or 20 warps
  // of 128 or 96): 2 x 88 + 2 x 112 + 80 = 5 x 96 and 128 + 2 x 144 + 96 = 4 x 128.
  static constexpr int kLoadRegs = Q8 ? 88 : 128, kSoftmaxRegs = Q8 ? 112 : 144, kIssueRegs = Q8 ? 80 : 96;
  static constexpr int kDBlocks = D / 64;         // 128-byte swizzled blocks of a row
  static constexpr int kKStages = 2;
  static constexpr int kVStages = 2;
  static constexpr int kQBytes = BM * D * 2;
  static constexpr int kTileBytes = BN * D * 2;   // of a converted (or bf16) K or V tile
  static constexpr int kAt_K = NQ * kQBytes;
  static constexpr int kAt_V = kAt_K + kKStages * kTileBytes;
  static constexpr int kAt_Bars = kAt_V + kVStages * kTileBytes;
  static constexpr size_t kSmemBytes = size_t(kAt_Bars) + 512 + 1024 /* alignment */;
  static constexpr int kO = 128;  // TMEM column of O, after 128 keys' scores or two of 64 keys'
  static_assert(kSmemBytes + 26 * 1024 <= 227 * 1024, "with the plan's static shared memory");
};

// One unit: rows q0 .. of sequence s, KV head h, and each query tile's key tiles.
struct ChunkUnit {
  int row0, n, first;    // the sequence's span
  int q0;                // row offset of query tile 0 within the span
  int tb[2], te[2];      // 64-key blocks that each query tile sees (empty: tb == te)
  int ub, ue;            // the key tiles that hold them
};

struct ChunkWalk {
  int64_t share;     // tiles of a CTA
  int64_t t, t_end;  // global tiles: the next piece's first, the share's end
  int64_t unit0;     // the unit's first global tile
  int s, h, qt, nq;  // sequence, KV head, unit of the sequence, units of the sequence
  int cta;
};

// Rows of a query tile.
__device__ __forceinline__ int chunk_rows(const PagedAttendArgs& a) { return a.tile_rows; }

// Units of sequence s (0 if it is empty, out of range or the token kernel's; -1 out of range).
template <int NQ>
__device__ __forceinline__ int chunk_units(const PagedAttendArgs& a, int s, PagedSpan* sp) {
  if (!paged_span(a.spans, a.pool.page_shift, s, sp)) return -1;
  if (sp->n == 0 || int64_t(sp->n) * a.group <= a.token_cols) return 0;
  const int rows = NQ * chunk_rows(a);
  return (sp->n + rows - 1) / rows;
}

template <int D, bool Q8>
__device__ __forceinline__ void chunk_unit(const PagedAttendArgs& a, const PagedSpan& sp, int qt,
                                           ChunkUnit* u) {
  using S = ChunkShape<D, Q8>;
  const int rows = chunk_rows(a);
  u->row0 = sp.row0;
  u->n = sp.n;
  u->first = sp.first;
  u->q0 = qt * S::NQ * rows;
  u->tb[1] = u->te[1] = 0;
  const int end = sp.first + sp.n;
#pragma unroll
  for (int i = 0; i < S::NQ; ++i) {
    const int r0 = u->q0 + i * rows, r1 = min(r0 + rows, sp.n);
    u->tb[i] = u->te[i] = 0;
    if (r0 >= sp.n) continue;
    int lo, hi, x;
    paged_keys(a.kind, a.window, sp.first + r0, end, &lo, &x);
    paged_keys(a.kind, a.window, sp.first + r1 - 1, end, &x, &hi);
    u->tb[i] = lo / 64;
    u->te[i] = (hi + 63) / 64;
  }
  // later rows see later keys, without a gap
  u->ub = u->tb[0] / S::kSubs;
  u->ue = (max(u->te[0], u->te[1]) + S::kSubs - 1) / S::kSubs;
}

// Tiles of a whole unit.
template <int D, bool Q8>
__device__ __noinline__ int chunk_cost(const PagedAttendArgs& a, const PagedSpan& sp, int qt) {
  ChunkUnit u;
  chunk_unit<D, Q8>(a, sp, qt, &u);
  return u.ue - u.ub;
}

struct ChunkPiece {
  ChunkUnit u;
  int h;
  int begin, end;  // key tiles of this piece
  int c0, c1;      // the first and last CTA that the unit is shared among
};

// The next piece of the CTA's share, or false at its end. spans: every sequence's row0, rows (0 if
// none are this kernel's) and first position.
template <int D, bool Q8>
__device__ __forceinline__ bool chunk_next(const PagedAttendArgs& a, const int3* spans, ChunkWalk* w,
                                           ChunkPiece* p) {
  if (w->t >= w->t_end) return false;
  while (w->qt >= w->nq) {
    w->qt = 0;
    if (w->nq > 0 && ++w->h < a.pool.kv_heads) continue;
    w->h = 0;
    ++w->s;
    const int rows = ChunkShape<D, Q8>::NQ * chunk_rows(a);
    w->nq = (spans[w->s].y + rows - 1) / rows;
  }
  const PagedSpan sp{spans[w->s].x, spans[w->s].y, spans[w->s].z};
  chunk_unit<D, Q8>(a, sp, w->qt, &p->u);
  p->h = w->h;
  const int cost = p->u.ue - p->u.ub;
  share_owners(w->share, w->cta, w->unit0, cost, &p->c0, &p->c1);
  p->begin = p->u.ub + int(w->t - w->unit0);
  p->end = int(min(int64_t(p->u.ue), p->begin + (w->t_end - w->t)));
  w->t += p->end - p->begin;
  w->unit0 += cost;
  ++w->qt;
  return true;
}

// A warp's 32 query rows of query tile i (packed rows 32 wq ..) into the swizzled tile at dst, zeros
// for those that are none: a row on D / 8 lanes, 8 or 16 loads of a lane in flight. Over 8-bit pages
// f16, a row scaled by a power of two to its range (and back by down[row]), its elements in the
// converted keys' order.
template <int D, bool Q8, bool BF16>
__device__ __forceinline__ void chunk_queries(const PagedAttendArgs& a, const ChunkPiece& pc, int i, int wq,
                                           unsigned char* dst, float* down) {
  constexpr int kCh = D / 8, kRows = 32 / kCh;
  constexpr int kBatch = BF16 && !Q8 && kCh >= 16 ? 16 : 8, kVecs = BF16 ? 1 : 2;
  const int lane = threadIdx.x & 31, ch = lane % kCh;
  const int rows = chunk_rows(a), left = min(rows, pc.u.n - pc.u.q0 - i * rows);
  const uint32_t magic = (65536 + a.group - 1) / a.group;  // row / group for rows below 128
  const int64_t base = int64_t(pc.u.row0 + pc.u.q0 + i * rows) * a.q_stride +
                       int64_t(pc.h * a.group) * D + ch * 8;
  constexpr int kBytes = BF16 ? 2 : 4;
#pragma unroll 1
  for (int b = 0; b < kCh; b += kBatch) {
    uint4 raw[kBatch][kVecs];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
#pragma unroll
      for (int y = 0; y < kVecs; ++y) raw[k][y] = make_uint4(0, 0, 0, 0);
      const int row = wq * 32 + (b + k) * kRows + lane / kCh;  // packed
      const int rr = int(row * magic >> 16), rh = row - rr * a.group;
      if (rr >= left) continue;
      const unsigned char* q = static_cast<const unsigned char*>(a.q) + (base + rr * a.q_stride + rh * D) * kBytes;
#pragma unroll
      for (int y = 0; y < kVecs; ++y) raw[k][y] = *reinterpret_cast<const uint4*>(q + 16 * y);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int row = wq * 32 + (b + k) * kRows + lane / kCh;
      const uint4 u = raw[k][0], v = raw[k][kVecs - 1];
      uint4 w = u;
      if constexpr (Q8 || !BF16) {
        float x[8];
        if constexpr (BF16) {
          x[0] = bf16_lo(u.x); x[1] = bf16_hi(u.x); x[2] = bf16_lo(u.y); x[3] = bf16_hi(u.y);
          x[4] = bf16_lo(u.z); x[5] = bf16_hi(u.z); x[6] = bf16_lo(u.w); x[7] = bf16_hi(u.w);
        } else {
          x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y);
          x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
          x[4] = __uint_as_float(v.x); x[5] = __uint_as_float(v.y);
          x[6] = __uint_as_float(v.z); x[7] = __uint_as_float(v.w);
        }
        if constexpr (Q8) {
          float top = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
          for (int off = kCh / 2; off >= 1; off >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const int e = min(max(int(__float_as_uint(top) >> 23), 1), 253);
          const float up = __uint_as_float(uint32_t(254 - e) << 23);
          if (ch == 0) down[row] = __uint_as_float(uint32_t(e) << 23);
          w = make_uint4(pack_f16(x[0] * up, x[2] * up), pack_f16(x[1] * up, x[3] * up),
                         pack_f16(x[4] * up, x[6] * up), pack_f16(x[5] * up, x[7] * up));
        } else {
          w = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                         pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        }
      }
      *reinterpret_cast<uint4*>(dst + (ch / 8) * (128 * 128) + row * 128 + (((ch % 8) ^ (row & 7)) * 16)) = w;
    }
  }
}

// 32 elements of a packed row's output, from element `at` of `out` on.
__device__ __forceinline__ void chunk_write(void* out, int64_t at, int bf16, int vec, const float (&x)[32]) {
  if (bf16) {
    uint16_t* dst = static_cast<uint16_t*>(out) + at;
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
    if (vec) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<uint4*>(dst)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) dst[e] = uint16_t(w[e / 2] >> (16 * (e & 1)));
    }
  } else {
    float* dst = static_cast<float*>(out) + at;
    if (vec) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        reinterpret_cast<float4*>(dst)[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) dst[e] = x[e];
    }
  }
}

template <int D, bool Q8>
__global__ void __launch_bounds__((ChunkShape<D, Q8>::kThreads), 1)
    paged_chunk_kernel(const __grid_constant__ PagedAttendArgs a) {
  using S = ChunkShape<D, Q8>;
  constexpr int NQ = S::NQ, BM = S::BM, BN = S::BN;
  constexpr uint32_t kFmt = Q8 ? 0u : 1u;  // f16 or bf16
  constexpr uint32_t kIdescQK = tc::instr_desc(kFmt, false, BN, BM);
  constexpr uint32_t kIdescPV = tc::instr_desc(kFmt, true, D, BM);
  constexpr int kTileCols = 256;  // TMEM columns of a query tile (two of them)

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ int64_t before[kMaxPagedSequences + 1];
  __shared__ int64_t scratch[S::kThreads / 32];
  // each warp's walk and piece live in shared memory: the softmax needs its registers for a row
  // of scores
  __shared__ ChunkWalk walks[S::kThreads / 32];
  __shared__ ChunkPiece pieces[S::kThreads / 32];
  __shared__ uint32_t poison[2][BN / 32];  // by V stage: keys with a value that is not finite
  // by tile % 4 (a tile's keys may arrive while a softmax group is still at the tile two before
  // it, never three: its scores wait for that group's products): a bit per 16 keys whose page is
  // out of range, and 8-bit pages' 2^k, v and 2^-v (2^k or 2^-v negative: each key has its own k or v)
  __shared__ uint32_t absent[4];
  __shared__ float k_units[4];
  __shared__ float2 v_units[4];
  __shared__ signed char own_k[4][Q8 ? BN : 1], own_v[4][Q8 ? BN : 1];
  __shared__ float q_down[Q8 ? NQ * 128 : 1];  // 8-bit pages: what a query row was scaled by, back
  __shared__ int3 spans[kMaxPagedSequences];   // row0, rows (0: none of this kernel's), first position
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = smem;
  unsigned char* sK = smem + S::kAt_K;
  unsigned char* sV = smem + S::kAt_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kAt_Bars);
  uint64_t* q_full = bars;                     // [2]: by query tile, once a piece it is part of
  uint64_t* k_full = bars + 2;                 // [2]
  uint64_t* k_empty = k_full + 2;              // [2]
  uint64_t* v_full = k_empty + 2;              // [2]
  uint64_t* v_empty = v_full + 2;              // [2]
  uint64_t* s_full = v_empty + 2;              // [2]: by query tile, or by score buffer
  uint64_t* p_full = s_full + 2;               // [4]: by query tile and block of the tile, or by
                                               // score buffer
  uint64_t* o_done = p_full + 4;               // [2]: each P.V
  uint64_t* o_final = o_done + 2;              // [2]: a piece's last P.V
  uint64_t* v_told = o_final + 2;              // [4]: by tile % 4, 8-bit pages' v_units, own_v
  uint64_t* drained = v_told + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kSoftmax0 = 2 * S::kLoad / 32, kMmaWarp = kSoftmax0 + NQ * 4;  // the first warps load

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&k_full[i], S::kLoad);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], S::kLoad);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 2);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_final[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&v_told[i], 1);
    mbar_init(drained, 1);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, 512);

  pdl_wait();
  pdl_trigger();

  // ---- the plan: tiles before every sequence, and this CTA's start ------------------------------
  const int nseq = a.spans.sequences, kvh = a.pool.kv_heads;
  for (int s = warp; s < nseq; s += S::kThreads / 32) {
    PagedSpan sp;
    const int units = chunk_units<NQ>(a, s, &sp);
    if (units < 0 && lane == 0) atomicOr(a.err, kErrPagedSpan);
    int64_t sum = 0;
    for (int qt = lane; qt < units; qt += 32) sum += chunk_cost<D, Q8>(a, sp, qt);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      before[s] = sum;
      spans[s] = make_int3(sp.row0, units > 0 ? sp.n : 0, sp.first);
    }
  }
  __syncthreads();
  {
    constexpr int kEach = (kMaxPagedSequences + S::kThreads - 1) / S::kThreads;
    const int s0 = min(nseq, int(threadIdx.x) * kEach), s1 = min(nseq, s0 + kEach);
    int64_t sum = 0;
    for (int s = s0; s < s1; ++s) sum += before[s];
    int64_t total;
    int64_t at = block_prefix<S::kThreads>(sum, scratch, &total);
    for (int s = s0; s < s1; ++s) {
      const int64_t x = before[s];
      before[s] = at;
      at += x;
    }
    if (threadIdx.x == 0) before[nseq] = total;
  }
  __syncthreads();
  const int64_t work = before[nseq] * kvh;
  // at least two tiles a CTA: a piece's partials cost about as much as a tile
  const int64_t share = share_size(work, int(min(int64_t(gridDim.x), (work + 1) / 2)) + (work == 0));
  const int cta = blockIdx.x;
  const bool idle = share * cta >= work;
  if (!idle && warp == 0) {
    ChunkWalk w;
    w.share = share;
    w.cta = cta;
    w.t = share * cta;
    w.t_end = min(work, w.t + share);
    int s0 = 0, s1 = nseq;  // the last s with before[s] * kvh <= t
    while (s1 - s0 > 1) {
      const int mid = (s0 + s1) / 2;
      if (before[mid] * kvh <= w.t) s0 = mid; else s1 = mid;
    }
    w.s = s0;
    const PagedSpan sp{spans[s0].x, spans[s0].y, spans[s0].z};
    const int unit_rows = NQ * chunk_rows(a);
    w.nq = (sp.n + unit_rows - 1) / unit_rows;
    const int64_t per = before[s0 + 1] - before[s0];
    const int64_t rest = w.t - before[s0] * kvh;
    w.h = whole_times(rest, per);
    int64_t off = rest - int64_t(w.h) * per;  // tiles into the head
    w.qt = 0;
    for (;;) {  // 32 units at a time
      const int64_t c = w.qt + lane < w.nq ? chunk_cost<D, Q8>(a, sp, w.qt + lane) : 0;
      int64_t inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, inc > off);
      if (past != 0 || w.qt + 32 >= w.nq) {
        const int at = past != 0 ? __ffs(past) - 1 : 31;
        off -= __shfl_sync(0xffffffffu, inc - c, at);
        w.qt += at;
        break;
      }
      off -= __shfl_sync(0xffffffffu, inc, 31);
      w.qt += 32;
    }
    w.unit0 = w.t - off;
    if (lane < S::kThreads / 32) walks[lane] = w;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (!idle) {
    const ChunkWalk& walk = walks[warp];
    const ChunkPiece& pc = pieces[warp];
    // The warp's next piece (the whole warp, except the MMA issuer's one thread). A shuffle orders no
    // memory: the barriers keep lane 0's writes after the others' reads of the piece before, and
    // before their reads of this one.
    auto next_piece = [&]() {
      __syncwarp();
      int more = 0;
      if (lane == 0) more = chunk_next<D, Q8>(a, spans, &walks[warp], &pieces[warp]);
      __syncwarp();
      return __shfl_sync(0xffffffffu, more, 0) != 0;
    };
    if (warp >= kMmaWarp) {
      // ---- MMA issuer ------------------------------------------------------------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kIssueRegs));
      if (warp == kMmaWarp && lane == 0) {
        const uint64_t q_desc = tc::smem_desc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t k_desc = tc::smem_desc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t v_desc = tc::smem_desc(smem_u32(sV), BN * 128, 1024, tc::kSwizzle128B);
        uint32_t tile = 0;        // K (and V) tiles consumed so far
        uint32_t queries[2] = {0, 0};  // pieces that each query tile was part of
        uint32_t pv[2][2] = {{0, 0}, {0, 0}};  // P.V products by block of a tile and query tile
        uint32_t sb = 0;                       // score products
        bool ok = true;
        while (ok && chunk_next<D, Q8>(a, spans, &walks[warp], &pieces[warp])) {
          const int n_tiles = pc.end - pc.begin, n = n_tiles * S::kSubs;  // 64-key blocks
          const int at0 = pc.begin * S::kSubs;
          bool first[2] = {true, true};
          const int b0 = pc.u.tb[0] - at0, e0 = pc.u.te[0] - at0;
          const int b1 = pc.u.tb[1] - at0, e1 = pc.u.te[1] - at0;
          auto part = [&](int i, int u) { return i == 0 ? u >= b0 && u < e0 : u >= b1 && u < e1; };
          // scores of tile L (score buffer sb & 1 where there are two)
          auto issue_s = [&](int i, int L) {
            const uint64_t qd = q_desc + uint64_t(i * S::kQBytes >> 4);
            const uint64_t kd = k_desc + uint64_t((tile + L) % S::kKStages) * uint64_t(S::kTileBytes >> 4);
            const uint32_t b = NQ == 2 ? uint32_t(i) : sb & 1;
            const uint32_t dst = tmem + (NQ == 2 ? uint32_t(i * kTileCols) : b * 64);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const int db = k / 4, koff = (k % 4) * 32;
              tc::mma_ss<false>(dst, qd + uint64_t((db * BM * 128 + koff) >> 4),
                                kd + uint64_t((db * BN * 128 + koff) >> 4), kIdescQK, k > 0 ? 1u : 0u);
            }
            tc::commit(&s_full[b]);
            // (and this thread's own arrival, which passes on what the loaders wrote for the softmax;
            // the tile's values may still be on their way, their units come before them)
            if constexpr (Q8) ok = ok && mbar_wait(&v_told[(tile + L) & 3], ((tile + L) >> 2) & 1, a.err);
            mbar_arrive(&s_full[b]);
            ++sb;
          };
          // block h of tile L: its probabilities are in columns 32 h of the scores' 128, or at the
          // start of its score buffer
          auto issue_pv = [&](int i, int L, int h) {
            const uint32_t vt = tile + L;
            const uint32_t pb = NQ == 2 ? uint32_t(2 * i + h) : vt & 1;
            if (!mbar_wait(&p_full[pb], NQ == 2 ? pv[h][i] & 1 : (vt >> 1) & 1, a.err)) return false;
            ++pv[h][i];
            if (!mbar_wait(&v_full[vt % S::kVStages], (vt / S::kVStages) & 1, a.err)) return false;
            tc::fence_after_sync();
            const uint32_t p_tmem = tmem + (NQ == 2 ? uint32_t(i * kTileCols + h * 32) : pb * 64);
            const uint32_t o_tmem = tmem + i * kTileCols + S::kO;
            const uint64_t vd = v_desc + uint64_t(vt % S::kVStages) * uint64_t(S::kTileBytes >> 4) +
                                uint64_t(h * (64 * 128) >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc::mma_ts<false>(o_tmem, p_tmem + k * 8, vd + uint64_t((k * 16 * 128) >> 4), kIdescPV,
                                (!first[i] || k > 0) ? 1u : 0u);
            tc::commit(&o_done[i]);
            first[i] = false;
            return true;
          };
          auto wait_k = [&](int L) {
            const uint32_t kt = tile + L;
            if (!mbar_wait(&k_full[kt % S::kKStages], (kt / S::kKStages) & 1, a.err)) return false;
            tc::fence_after_sync();
            return true;
          };
          auto part_tile = [&](int i, int L) {
            const int u0 = L * S::kSubs, u1 = u0 + S::kSubs;
            return i == 0 ? u1 > b0 && u0 < e0 : u1 > b1 && u0 < e1;
          };
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if ((i == 0 ? min(n, e0) <= max(0, b0) : min(n, e1) <= max(0, b1))) continue;
            ok = ok && mbar_wait(&q_full[i], queries[i] & 1, a.err);
            ++queries[i];
          }
          ok = ok && wait_k(0);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (part_tile(i, 0)) issue_s(i, 0);
          tc::commit(&k_empty[tile % S::kKStages]);
          for (int L = 0; ok && L < n_tiles; ++L) {
            const bool next = L + 1 < n_tiles;
            if constexpr (NQ == 1) {
              // the next scores go to the other buffer before this tile's P.V
              ok = !next || wait_k(L + 1);
              if (ok && next) issue_s(0, L + 1);
            }
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
#pragma unroll
              for (int h = 0; h < S::kSubs; ++h)
                if (ok && part(i, L * S::kSubs + h)) ok = issue_pv(i, L, h);
              if constexpr (NQ == 2) {
                if (ok && next && i == 0) ok = wait_k(L + 1);
                if (ok && next && part_tile(i, L + 1)) issue_s(i, L + 1);
              }
            }
            if (!ok) break;
            if (next) tc::commit(&k_empty[(tile + L + 1) % S::kKStages]);
            tc::commit(&v_empty[(tile + L) % S::kVStages]);
          }
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (!first[i]) tc::commit(&o_final[i]);
          tile += uint32_t(n_tiles);
        }
        // every MMA this thread issued has completed before the CTA may free TMEM
        tc::commit(drained);
        mbar_wait(drained, 0, a.err);
      }
    } else if (warp < kSoftmax0) {
      // ---- loaders: the first half brings the keys, the other the values ----------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kLoadRegs));
      const bool is_v = warp >= S::kLoad / 32;
      const int tid = threadIdx.x & (S::kLoad - 1);
      constexpr int kRB = D * (Q8 ? 1 : 2), kCR = kRB / 16;  // a page row's bytes and chunks
      constexpr int kPass = S::kLoad / kCR;                  // rows of one pass of the threads (bf16)
      constexpr int kSub = 16 / kPass, kGroups = BN / 16;    // passes of 16 keys, 16s of a tile
      const int shift = a.pool.page_shift;
      const int chunk = tid % kCR, prow = tid / kCR;
      const unsigned char* pool = is_v ? a.pool.values : a.pool.keys;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      unsigned char* tiles = is_v ? sV : sK;
      uint32_t tile = 0;
      bool ok = true, more = next_piece();
      // one key tile's numbers: its first position, the keys that rows of the unit see, and lane
      // i's page of keys 16 i .. 16 i + 15 (-1: none seen; -2: out of range, a bit of `gone`)
      int pos = 0, lo = 0, hi = 0, page = -1;
      uint32_t gone = 0;
      bool edge = false;
      int ahead = -1, ahead_at = -1;  // the table's entry for the lane of the tile after the last
      auto look = [&](int at) {
        const ChunkUnit& u = pc.u;
        const int last = min(u.q0 + NQ * chunk_rows(a), u.n) - 1, end = u.first + u.n;
        int lo_all, hi_all;
        paged_keys(a.kind, a.window, u.first + u.q0, end, &lo, &hi_all);
        paged_keys(a.kind, a.window, u.first + last, end, &lo_all, &hi);
        pos = at * BN;
        edge = pos < lo_all || pos + BN > hi_all;
        page = -1;
        const int p = pos + lane * 16;
        const int* table = a.spans.tables + int64_t(walk.s) * a.spans.table_stride;
        const int read = ahead_at == at ? ahead : -3;
        // the next tile's entries are fetched now (within the piece: its own sequence's)
        ahead_at = at + 1 < pc.end ? at + 1 : -1;
        const int pn = p + BN;
        ahead = -1;
        if (ahead_at >= 0 && lane < kGroups && pn < hi && pn + 16 > lo) ahead = __ldg(table + (pn >> shift));
        if (lane < kGroups && p < hi && p + 16 > lo) {
          page = read != -3 ? read : __ldg(table + (p >> shift));
          if (!paged_page_ok(page, a.pool.pages)) {
            atomicOr(a.err, kErrPagedPage);
            page = -2;
          }
        }
        gone = __ballot_sync(0xffffffffu, page == -2);
      };
      // Row `row` of 16 keys from position p0 is seen by some row of the unit.
      auto seen = [&](int p0, int row) { return p0 + row >= lo && p0 + row < hi; };
      // A stage's products are done (its marks are cleared). The value loaders decide as one, so
      // that a wait that gave up cannot leave the others at their barrier; the key loaders need
      // none.
      auto vacant = [&](int st, uint32_t parity) {
        const bool there = mbar_wait(&empty[st], parity, a.err);
        if (!is_v) return __all_sync(0xffffffffu, there) != 0;
        if (there && tid < BN / 32) poison[st][tid] = 0;
        return !named_sync_or(1, S::kLoad, !there);
      };
      auto stage_of = [&]() { return int(tile % (is_v ? S::kVStages : S::kKStages)); };
      auto phase_of = [&]() { return ((tile / (is_v ? S::kVStages : S::kKStages)) & 1) ^ 1; };
      if constexpr (!Q8) {
        while (more && ok) {
          const int begin = pc.begin, end = pc.end;
          for (int at = begin; at < end; ++at, ++tile) {
            look(at);
            const int st = stage_of();
            if (!vacant(st, phase_of())) { ok = false; break; }
            const uint32_t dst = smem_u32(tiles) + st * S::kTileBytes + (chunk / 8) * (BN * 128);
#pragma unroll 2
            for (int gr = 0; gr < kGroups; ++gr) {
              const int pg = __shfl_sync(0xffffffffu, page, gr), p0 = pos + gr * 16;
              const int64_t row0 = ((int64_t(max(pg, 0)) * kvh + pc.h) << shift) + (p0 & ((1 << shift) - 1));
              const unsigned char* src = pool + (row0 + prow) * kRB + chunk * 16;
#pragma unroll
              for (int j = 0; j < kSub; ++j) {
                const int row = gr * 16 + prow + j * kPass;
                const bool there = pg >= 0 && seen(p0, prow + j * kPass);
                cp_async16(dst + row * 128 + (((chunk % 8) ^ (row & 7)) * 16), src + j * kPass * kRB,
                           there ? 16u : 0u);
              }
            }
            cp_async_commit();
            cp_async_wait<0>();
            if (is_v && edge) {
              // what is not finite taken out, its key marked
#pragma unroll 1
              for (int i = 0; i < kGroups * kSub; ++i) {
                const int row = prow + i * kPass;
                uint4* p = reinterpret_cast<uint4*>(tiles + st * S::kTileBytes + (chunk / 8) * (BN * 128) +
                                                    row * 128 + (((chunk % 8) ^ (row & 7)) * 16));
                const uint4 v = *p;
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
                bool bad = false;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  if ((w[x] & 0x7F80u) == 0x7F80u) { w[x] &= 0xFFFF0000u; bad = true; }
                  if ((w[x] & 0x7F800000u) == 0x7F800000u) { w[x] &= 0xFFFFu; bad = true; }
                }
                if (bad) {
                  *p = make_uint4(w[0], w[1], w[2], w[3]);
                  atomicOr(&poison[st][row >> 5], 1u << (row & 31));
                }
              }
            }
            if (!is_v && tid == 0) absent[tile & 3] = gone;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full[st]);
          }
          if (ok) more = next_piece();
        }
      } else {
        // A tile's bytes wait in registers, loaded while the tile before it is converted. A warp
        // takes 8 rows x 64 bytes at a time (lane: row lane % 8, chunk lane / 8), so that its
        // 16-byte stores into the swizzled rows meet no bank twice.
        constexpr int kWide = kCR / 4;              // 64-byte columns of a row: 1, 2 or 4
        constexpr int kItems = BN / 8 * kWide / 4;  // of a warp
        constexpr int kKeys = BN / 32;
        const int w4 = warp & 3, r8 = lane & 7, c4 = lane >> 3;
        uint4 raw[kItems];
        float sc[kKeys];  // scales of keys lane, lane + 32, ...
        // item k of the warp: rows 8 rg .. 8 rg + 7, chunks 4 cg .. 4 cg + 3
        auto rg_of = [&](int k) { return kWide == 1 ? 4 * k + w4 : kWide == 2 ? 2 * k + (w4 >> 1) : k; };
        const int cg = kWide == 1 ? 0 : kWide == 2 ? w4 & 1 : w4;
        auto row_of = [&](int gr) {
          const int pg = __shfl_sync(0xffffffffu, page, gr);
          return ((int64_t(max(pg, 0)) * kvh + pc.h) << shift) + ((pos + gr * 16) & ((1 << shift) - 1));
        };
        // (rows that are not seen get a zero scale: what their bytes are, or page 0's in their
        // place, does not matter)
        auto load = [&](int k) {
          raw[k] = __ldg(reinterpret_cast<const uint4*>(
              pool + (row_of(rg_of(k) >> 1) + (rg_of(k) & 1) * 8 + r8) * kRB + (cg * 4 + c4) * 16));
        };
        const float* scales = is_v ? a.pool.value_scales : a.pool.key_scales;
        auto load_scales = [&]() {
#pragma unroll
          for (int x = 0; x < kKeys; ++x) {
            const int row = lane + 32 * x, p = pos + row;
            const int pg = __shfl_sync(0xffffffffu, page, row >> 4);
            const bool there = pg >= 0 && p >= lo && p < hi;
            const int64_t at = ((int64_t(max(pg, 0)) * kvh + pc.h) << shift) + (p & ((1 << shift) - 1));
            const float v = __ldg(scales + at);
            sc[x] = there ? v : 0.0f;
          }
        };
        // The exponent that takes a scale to [2^8, 2^9) (127 of it stay in f16), or 2^least for
        // smaller ones. A row's sum is kept in the unit of its largest values, so units must not lie
        // further apart than f32 reaches: from the values' least, 2^-40, they do not for scales up to
        // 2^70 (and a value is off by at most 2^-58 more).
        const int least = is_v ? -40 : -118;
        auto exponent = [&](uint32_t bits) { return min(max(int(bits >> 23) - 135, least), 112); };
        auto finite_bits = [](float x) {
          return fabsf(x) <= 3.402823466e38f ? __float_as_uint(fabsf(x)) : 0u;
        };
        // Whether a scale in the unit of its tile, that is not zero, lies more than 2^8 below the
        // largest. f16 would then lose what rows are made of that do not see the largest, or give it
        // no weight: every key gets its own unit.
        auto far_below = [](float y) { return fabsf(y) < 1.0f && y != 0.0f; };
        auto power = [](int e) { return __uint_as_float(uint32_t(127 + e) << 23); };
        int at = pc.begin, end = pc.end;
        if (more) {
          look(at);
#pragma unroll
          for (int k = 0; k < kItems; ++k) load(k);
          load_scales();
        }
        while (more) {
          const int st = stage_of();
          const bool was_edge = edge;
          const uint32_t was_gone = gone;
          uint32_t top = 0;
#pragma unroll
          for (int x = 0; x < kKeys; ++x) top = max(top, finite_bits(sc[x]));
          const int e = exponent(__reduce_max_sync(0xffffffffu, top));
          // this tile's scales as f16 pairs
          const float down = power(-e);
          __half2 hs[kKeys];
          uint32_t bad = 0;  // keys lane + 32 x whose value scale is not finite
          bool own = false;
#pragma unroll
          for (int x = 0; x < kKeys; ++x) {
            const bool drop = is_v && was_edge && !(fabsf(sc[x]) <= 3.402823466e38f);
            bad |= uint32_t(drop) << x;
            const float y = drop ? 0.0f : sc[x] * down;
            own = own || far_below(y);
            hs[x] = __float2half2_rn(y);
          }
          own = __any_sync(0xffffffffu, own);
          // (the tile four before this one, whose place the units take, is done with: its products
          // came before those that made room for the last tile)
          if (own) {
#pragma unroll
            for (int x = 0; x < kKeys; ++x) {
              const int mine = exponent(finite_bits(sc[x]));
              if ((warp & 3) == 0) (is_v ? own_v : own_k)[tile & 3][lane + 32 * x] = (signed char)(mine);
              if (!((bad >> x) & 1u)) hs[x] = __float2half2_rn(sc[x] * power(-mine));
            }
          }
          if (is_v && warp == 4) {
            if (lane == 0) v_units[tile & 3] = make_float2(float(e), own ? -power(-e) : power(-e));
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_told[tile & 3]);
          }
          // the tile after this one, of this piece or the next
          if (++at == end) {
            more = next_piece();
            at = pc.begin;
            end = pc.end;
          }
          if (more) {
            look(at);
            load_scales();
          }
          if (!vacant(st, phase_of())) { ok = false; break; }
          unsigned char* dst = tiles + st * S::kTileBytes;
          const int c0 = (cg * 4 + c4) * 2;
          dst += (c0 / 8) * (BN * 128) + r8 * 128;
          const int to0 = ((c0 % 8) ^ r8) * 16, to1 = ((c0 % 8 + 1) ^ r8) * 16;
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            constexpr int kPer = kWide == 1 ? 1 : kWide == 2 ? 2 : 4;  // items of 32 rows
            const __half2 h = __shfl_sync(0xffffffffu, hs[k / kPer], (rg_of(k) * 8 + r8) & 31);
            const uint4 v = raw[k];
            load(k);  // (this tile's again after the last: no branch around the loads)
            auto half = [&](uint32_t w) {
              const uint32_t y = bytes_to_f16(w);
              const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&y), h);
              return *reinterpret_cast<const uint32_t*>(&r);
            };
            unsigned char* p = dst + rg_of(k) * 1024;
            *reinterpret_cast<uint4*>(p + to0) =
                make_uint4(half(v.x), half(v.x >> 8), half(v.y), half(v.y >> 8));
            *reinterpret_cast<uint4*>(p + to1) =
                make_uint4(half(v.z), half(v.z >> 8), half(v.w), half(v.w >> 8));
          }
          if (is_v && was_edge && warp == 4) {
#pragma unroll
            for (int x = 0; x < kKeys; ++x)
              if ((bad >> x) & 1u) atomicOr(&poison[st][x], 1u << lane);
          }
          if (!is_v && tid == 0) {
            absent[tile & 3] = was_gone;
            k_units[tile & 3] = own ? -power(e) : power(e);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&full[st]);
          ++tile;
        }
      }
    } else {
      // ---- softmax and output of query tile i ------------------------------------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
      const int i = NQ == 2 ? (warp - kSoftmax0) >> 2 : 0;
      const int wq = warp & 3;             // the TMEM lane quarter that this warp may access
      const int p = wq * 32 + lane;        // packed row
      const int rows = chunk_rows(a);
      const int pr = p / a.group, ph = p % a.group;
      const uint32_t lane_base = tmem + (NQ == 2 ? i * kTileCols : 0) + (uint32_t(wq * 32) << 16);
      const uint32_t o_base = lane_base + S::kO;
      uint32_t sc = 0;     // this query tile's blocks so far
      uint32_t st = 0;     // and score products
      uint32_t finals = 0; // pieces that it took part in
      uint32_t tile = 0;   // K (and V) tiles so far
      bool ok = true;
      while (ok && next_piece()) {
        const int n_tiles = pc.end - pc.begin;
        const int n = n_tiles * S::kSubs;  // 64-key blocks
        const int my_b = pc.u.tb[i] - pc.begin * S::kSubs, my_e = pc.u.te[i] - pc.begin * S::kSubs;
        const int kp0 = pc.begin * BN;  // the piece's first key
        const int r = pc.u.q0 + i * rows + pr;  // row of the span
        const bool valid = pr < rows && r < pc.u.n;
        float scale = a.scale_log2;
        if (min(n, my_e) > max(0, my_b)) {
          unsigned char* dst = sQ + i * S::kQBytes;
          if (a.q_bf16) chunk_queries<D, Q8, true>(a, pc, i, wq, dst, q_down + (Q8 ? i * 128 : 0));
          else chunk_queries<D, Q8, false>(a, pc, i, wq, dst, q_down + (Q8 ? i * 128 : 0));
          __syncwarp();
          if constexpr (Q8) scale *= q_down[i * 128 + p];
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&q_full[i]);
        }
        Runs runs{0, 0, 0, 0};
        if (valid) {
          int lo, hi;
          paged_keys(a.kind, a.window, pc.u.first + r, pc.u.first + pc.u.n, &lo, &hi);
          runs.b0 = lo;
          runs.n0 = hi - lo;
        }
        int lo_all, hi_all;  // keys that every row of the unit sees
        {
          int x;
          const int end = pc.u.first + pc.u.n;
          paged_keys(a.kind, a.window, pc.u.first + pc.u.q0, end, &x, &hi_all);
          paged_keys(a.kind, a.window,
                     pc.u.first + min(pc.u.q0 + NQ * rows, pc.u.n) - 1, end, &lo_all, &x);
        }
        float m_used = -INFINITY, l_sum = 0.0f;
        bool poisoned = false;
        int c = 0;  // blocks of this piece so far
        const int u_end = min(n, my_e);
        for (int u = max(0, my_b); u < u_end; ++u) {
          const int L = u / S::kSubs;
          const int kp = kp0 + u * 64;
          const int h = u % S::kSubs;
          const uint32_t buf = (tile + L) & 1;  // one query tile: the score buffer
          const uint32_t s_base = lane_base + (NQ == 2 ? uint32_t(h) * 64 : buf * 64);
          const uint32_t p_base = lane_base + (NQ == 2 ? uint32_t(h) * 32 : buf * 64);
          // A block's end: the keys that the loaders marked, O to the maximum's new unit, and word to
          // the issuer. (Once in each of the two paths below: where they join, the common one takes
          // 30 us longer of 790 for 2048 rows after 14336 positions.)
          auto finish = [&](float alpha) __attribute__((always_inline)) {
            if (kp0 + L * BN < lo_all || kp0 + (L + 1) * BN > hi_all) {
              // an edge tile (of the unit, as the loaders see it): keys that they marked
              const uint32_t vt = tile + L;
              const bool v_there = mbar_wait(&v_full[vt % S::kVStages], (vt / S::kVStages) & 1, a.err);
              if (!__all_sync(0xffffffffu, v_there)) return ok = false;
              const volatile uint32_t* marks = poison[vt % S::kVStages];
#pragma unroll
              for (int w = 0; w < 2; ++w)
                if (marks[h * 2 + w] & run_word(runs.b0, runs.n0, kp, w)) poisoned = true;
            }
            if (__any_sync(0xffffffffu, alpha != 1.0f) && c > 0) {
              // O holds the products of this piece's earlier tiles, the last of which may still run
              if (!__all_sync(0xffffffffu, mbar_wait(&o_done[i], (sc - 1) & 1, a.err))) return ok = false;
              tc::fence_after_sync();
#pragma unroll 1
              for (int cc = 0; cc < D / 32; ++cc) {
                uint32_t o[32];
                tc::tmem_ld32_wait(o_base + cc * 32, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tc::tmem_st32(o_base + cc * 32, o);
                tc::tmem_wait_st();
              }
            }
            tc::tmem_wait_st();
            tc::fence_before_sync();
            mbar_arrive(&p_full[NQ == 2 ? uint32_t(2 * i + h) : buf]);
            ++c;
            ++sc;
            return true;
          };
          if (h == 0 || c == 0) {
            // every decision before a whole-warp tcgen05 instruction is made warp-uniform
            const bool there = NQ == 2 ? mbar_wait(&s_full[i], st & 1, a.err)
                                       : mbar_wait(&s_full[buf], ((tile + L) >> 1) & 1, a.err);
            if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
            ++st;
            tc::fence_after_sync();
          }
          const uint32_t gone = *const_cast<const volatile uint32_t*>(&absent[(tile + L) & 3]);
          float alpha = 1.0f;
          float k_unit = 1.0f;
          float2 v_unit = make_float2(0.0f, 1.0f);
          if constexpr (Q8) {
            k_unit = k_units[(tile + L) & 3];
            v_unit = v_units[(tile + L) & 3];
          }
          uint32_t sreg[64];
          tc::tmem_ld64_wait(s_base, sreg);
          if (Q8 && (k_unit < 0.0f || v_unit.y < 0.0f)) {  // (the same for all)
            // Keys with units of their own: what follows below, 32 keys at a time and twice over (the
            // maximum first), the scores as base-2 exponents with each key's v in them.
            const signed char* ks = &own_k[(tile + L) & 3][h * 64];
            const signed char* vs = &own_v[(tile + L) & 3][h * 64];
            float top = -INFINITY, sum = 0.0f, less = 0.0f;
#pragma unroll 1
            for (int step = 0; step < 4; ++step) {
              const int k0 = (step & 1) * 32;
              uint32_t r[32];
              tc::tmem_ld32_wait(s_base + k0, r);
              const uint32_t off = gone >> (h * 4 + k0 / 16);
              const uint32_t in = run_word(runs.b0, runs.n0, kp + k0, 0) &
                                  ~((off & 1u ? 0xFFFFu : 0u) | (off & 2u ? 0xFFFF0000u : 0u));
              if (step == 2) {
                if (top > m_used + 8.0f || (m_used == -INFINITY && top > -INFINITY)) {
                  if (m_used > -INFINITY) alpha = exp2_approx(m_used - top);
                  m_used = top;
                }
                less = 7.0f - (m_used == -INFINITY ? 0.0f : m_used);
              }
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float unit = k_unit < 0.0f ? __uint_as_float(uint32_t(127 + ks[k0 + x]) << 23) : k_unit;
                const float v = v_unit.y < 0.0f ? float(vs[k0 + x]) : v_unit.x;
                float y = fmaf(__uint_as_float(r[x]), fmaxf(scale * unit, 1.175494351e-38f), v);
                if (!((in >> x) & 1u)) y = -INFINITY;
                if (step < 2) top = fmaxf(top, y);
                else sum += exp2_approx(y + (less - v));  // (each key's 2^-v taken back out)
                r[x] = __float_as_uint(exp2_approx(y + less));
              }
              if (step < 2) continue;
              uint32_t w[16];
#pragma unroll
              for (int x = 0; x < 16; ++x) w[x] = pack_f16(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1]));
              tc::tmem_st16(p_base + k0 / 2, w);
            }
            l_sum = l_sum * alpha + sum;
            if (!finish(alpha)) break;
            continue;
          }
          // the tile's units: its scores' scale, what its exponents and its sum take besides
          float scale_t = scale, up_t = 0.0f, down_t = 1.0f;
          if constexpr (Q8) {
            // (not 0, for a masked score times it would be a NaN)
            scale_t = fmaxf(scale * k_unit, 1.175494351e-38f);
            up_t = v_unit.x;
            down_t = v_unit.y;
          }
          float* s = reinterpret_cast<float*>(sreg);
          const bool all_in = !valid || (kp >= runs.b0 && kp + 64 <= runs.b0 + runs.n0);
          if (!all_in || gone != 0) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t off = gone >> (h * 4 + w * 2);
              const uint32_t bits = run_word(runs.b0, runs.n0, kp, w) &
                                    ~((off & 1u ? 0xFFFFu : 0u) | (off & 2u ? 0xFFFF0000u : 0u));
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (!((bits >> x) & 1u)) s[32 * w + x] = -INFINITY;
            }
          }
          float mx0 = s[0], mx1 = s[1], mx2 = s[2], mx3 = s[3];
#pragma unroll
          for (int x = 4; x < 60; x += 8) {
            mx0 = fmax3(mx0, s[x], s[x + 1]);
            mx1 = fmax3(mx1, s[x + 2], s[x + 3]);
            mx2 = fmax3(mx2, s[x + 4], s[x + 5]);
            mx3 = fmax3(mx3, s[x + 6], s[x + 7]);
          }
          mx0 = fmax3(mx0, s[60], s[61]);
          mx1 = fmax3(mx1, s[62], s[63]);
          const float m_tile = fmaf(fmax3(mx0, mx1, fmaxf(mx2, mx3)), scale_t, up_t);
          if (m_tile > m_used + 8.0f || (m_used == -INFINITY && m_tile > -INFINITY)) {
            if (m_used > -INFINITY) alpha = exp2_approx(m_used - m_tile);
            m_used = m_tile;
          }
          const float ms = m_used == -INFINITY ? 0.0f : m_used;
          const float off = Q8 ? up_t - ms + 7.0f : -ms;
          const float2 scale2 = make_float2(scale_t, scale_t), neg2 = make_float2(off, off);
          float2 sum2a = make_float2(0.0f, 0.0f), sum2b = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int x = 0; x < 64; x += 4) {
            const float2 x0 = __ffma2_rn(make_float2(s[x], s[x + 1]), scale2, neg2);
            const float2 x1 = __ffma2_rn(make_float2(s[x + 2], s[x + 3]), scale2, neg2);
            const float2 p0 = make_float2(exp2_approx(x0.x), exp2_approx(x0.y));
            const float2 p1 = make_float2(exp2_approx(x1.x), exp2_approx(x1.y));
            sum2a = __fadd2_rn(sum2a, p0);
            sum2b = __fadd2_rn(sum2b, p1);
            sreg[x / 2] = Q8 ? pack_f16(p0.x, p0.y) : tc::pack_bf16(p0.x, p0.y);
            sreg[x / 2 + 1] = Q8 ? pack_f16(p1.x, p1.y) : tc::pack_bf16(p1.x, p1.y);
          }
          tc::tmem_st32(p_base, *reinterpret_cast<const uint32_t(*)[32]>(&sreg[0]));
          l_sum = l_sum * alpha + ((sum2a.x + sum2a.y) + (sum2b.x + sum2b.y)) * down_t;
          if (!finish(alpha)) break;
        }
        if (!ok) break;
        tile += uint32_t(n_tiles);
        bool have = c > 0;
        if (have) {
          if (!__all_sync(0xffffffffu, mbar_wait(&o_final[i], finals & 1, a.err))) { ok = false; break; }
          ++finals;
          tc::fence_after_sync();
        }
        if (poisoned) l_sum = __int_as_float(0x7fffffff);
        const int c0 = pc.c0, c1 = pc.c1;
        const int64_t orow = int64_t(pc.u.row0 + r) * a.out_stride + int64_t(pc.h * a.group + ph) * D;
        // O to the output, or (a piece of a unit) to the partials; then, by the last piece to
        // arrive, the partials merged to the output: one loop over O's columns for all three.
        // Partials lie by float4s of 128 packed rows (a warp's stores are contiguous).
        auto slot_of = [&](int x) { return int64_t(2 * x + (x == c0 ? 1 : 0)) * NQ + i; };
        const int64_t slot = slot_of(cta);
        int mode = c0 == c1 ? 0 : 1;  // 2: merge
        float mm = -INFINITY;
        for (;;) {
          const float inv = l_sum == 0.0f ? 0.0f : 1.0f / l_sum;
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            float* x = reinterpret_cast<float*>(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
            if (mode < 2) {
              if (!have) break;
              tc::tmem_ld32_wait(o_base + cc * 32, o);
              if constexpr (Q8) {
                // the elements' order
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const uint32_t y = o[e + 1];
                  o[e + 1] = o[e + 2];
                  o[e + 2] = y;
                }
              }
            } else {
#pragma unroll 1
              for (int z = c0; z <= c1; ++z) {
                const float mx = __ldcg(a.part_ml + (slot_of(z) * 128 + p) * 2);
                const float* src = a.part_o + ((slot_of(z) * (D / 4) + cc * 8) * 128 + p) * 4;
                float4 v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __ldcg(reinterpret_cast<const float4*>(src + e * 512));
                // (no key of that piece is seen: its O is not there)
                if (mx == -INFINITY) continue;
                const float f = exp2_approx(mx - mm);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  x[4 * e] = fmaf(f, v[e].x, x[4 * e]);
                  x[4 * e + 1] = fmaf(f, v[e].y, x[4 * e + 1]);
                  x[4 * e + 2] = fmaf(f, v[e].z, x[4 * e + 2]);
                  x[4 * e + 3] = fmaf(f, v[e].w, x[4 * e + 3]);
                }
              }
            }
            if (mode == 1) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(a.part_o + ((slot * (D / 4) + cc * 8 + e) * 128 + p) * 4) =
                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else if (valid) {
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] *= inv;
              chunk_write(a.out, orow + cc * 32, a.out_bf16, a.out_vec, *reinterpret_cast<const float(*)[32]>(x));
            }
          }
          if (mode != 1) break;
          *reinterpret_cast<float2*>(a.part_ml + (slot * 128 + p) * 2) =
              make_float2(have ? m_used : -INFINITY, l_sum);
          // each warp's rows count their pieces on their own counter: no barrier among the warps
          __threadfence();
          __syncwarp();
          int last = 0;
          if (lane == 0) {
            int* counter = a.counters + c0 * (NQ * 4) + i * 4 + wq;
            last = atomicAdd(counter, 1) == c1 - c0;
            if (last) *counter = 0;
          }
          if (__shfl_sync(0xffffffffu, last, 0) == 0) break;
          // (lane 0 saw the other pieces' arrivals; the whole warp reads what they left)
          __threadfence();
          __syncwarp();
          l_sum = 0.0f;
#pragma unroll 4
          for (int z = c0; z <= c1; ++z) mm = fmaxf(mm, __ldcg(a.part_ml + (slot_of(z) * 128 + p) * 2));
#pragma unroll 4
          for (int z = c0; z <= c1; ++z) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + (slot_of(z) * 128 + p) * 2));
            l_sum += ml.x == -INFINITY ? ml.y : ml.y * exp2_approx(ml.x - mm);
          }
          mode = 2;
        }
        tc::fence_before_sync();
      }
    }
  }

  // ---- teardown: every TMEM user is done before the owner frees it -------------------------------
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace fa

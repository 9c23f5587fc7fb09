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
//   loaders (4 warps): the pages' rows into the swizzled tiles that the products read. bf16 pages
//     by cp.async straight to their places; 8-bit pages by cp.async into a raw buffer, then
//     converted by the thread that fetched them: keys to f16 and values to bf16 integers (both
//     exact), two pairs a word without a byte permutation: a word's bytes come out as 0, 2, 1, 3,
//     and Q's rows (keys) and the output's columns (values) follow that order;
//   one warp: TMEM and the MMA issue (one thread).
// 8-bit pages: a key's scale multiplies its score before the maximum, a value's scale its
// probability before that is rounded to bf16; a query row is scaled by a power of two to f16's
// range. Two tiles: as fmha2_kernel (fa_fmha2.cuh) the order per key tile is PV0, S0', PV1, S1',
// so that one group's exponentials overlap the other's products. One tile: two score buffers,
// S' is issued before PV.
//
// Keys that no row of a unit sees come as zeros (a page's stale end may hold anything). On edge
// tiles, where some rows see a key and others do not, a value that is not finite would reach all
// of them (0 x inf): the loaders take it out and mark its key, and the rows that see the key get
// a NaN sum. Every wait is bounded (mbar_wait).
#pragma once

#include "fa_decode.cuh"
#include "fa_paged_tokens.cuh"
#include "fa_tc.cuh"

namespace fa {

template <int D, bool Q8>
struct ChunkShape {
  static constexpr int NQ = D == 256 ? 1 : 2;     // query tiles of a unit
  static constexpr int BM = 128;
  static constexpr int BN = D == 256 ? 64 : 128;  // keys of a tile
  static constexpr int kThreads = NQ == 2 ? 512 : 384;
  static constexpr int kDBlocks = D / 64;         // 128-byte swizzled blocks of a row
  static constexpr int kKStages = 2;
  static constexpr int kVStages = Q8 && D >= 128 ? 1 : 2;  // what shared memory holds
  static constexpr int kQBytes = BM * D * 2;
  static constexpr int kTileBytes = BN * D * 2;   // of a converted (or bf16) K or V tile
  static constexpr int kRawBytes = Q8 ? BN * D : 0;
  // scales of keys and of values, of four tiles: a tile's keys may arrive while a softmax group is
  // still at the tile two before it, never three (its scores wait for that group's products)
  static constexpr int kScaleBytes = Q8 ? 4 * 2 * BN * 4 : 0;
  static constexpr int kAt_K = NQ * kQBytes;
  static constexpr int kAt_V = kAt_K + kKStages * kTileBytes;
  static constexpr int kAt_Raw = kAt_V + kVStages * kTileBytes;
  static constexpr int kAt_Scales = kAt_Raw + 2 * kRawBytes;
  static constexpr int kAt_Bars = kAt_Scales + kScaleBytes;
  static constexpr size_t kSmemBytes = size_t(kAt_Bars) + 512 + 1024 /* alignment */;
  static constexpr int kO = 128;  // TMEM column of O, after S (or the two S of 64 keys)
  static_assert(kSmemBytes + 16 * 1024 <= 227 * 1024, "with the plan's static shared memory");
};

// One unit: rows q0 .. of sequence s, KV head h, and each query tile's key tiles.
struct ChunkUnit {
  int row0, n, first;    // the sequence's span
  int q0;                // row offset of query tile 0 within the span
  int tb[2], te[2];      // key tiles of each query tile (empty: tb == te)
  int ub, ue;            // their union
};

struct ChunkWalk {
  int64_t t, t_end;  // global tiles: the next piece's first, the share's end
  int64_t unit0;     // the unit's first global tile
  int s, h, qt, nq;  // sequence, KV head, unit of the sequence, units of the sequence
};

// Rows of a query tile.
__device__ __forceinline__ int chunk_rows(const PagedAttendArgs& a) { return 128 / a.group; }

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
    u->tb[i] = lo / S::BN;
    u->te[i] = (hi + S::BN - 1) / S::BN;
  }
  u->ub = u->tb[0];
  u->ue = max(u->te[0], u->te[1]);  // later rows see later keys
}

// Tiles of a whole unit.
template <int D, bool Q8>
__device__ __forceinline__ int chunk_cost(const PagedAttendArgs& a, const PagedSpan& sp, int qt) {
  ChunkUnit u;
  chunk_unit<D, Q8>(a, sp, qt, &u);
  return u.ue - u.ub;
}

struct ChunkPiece {
  ChunkUnit u;
  int h;
  int begin, end;  // key tiles of this piece
  int64_t unit0;
  int cost;        // the whole unit's tiles
};

// The next piece of the CTA's share, or false at its end.
template <int D, bool Q8>
__device__ __forceinline__ bool chunk_next(const PagedAttendArgs& a, ChunkWalk* w, ChunkPiece* p) {
  if (w->t >= w->t_end) return false;
  PagedSpan sp;
  while (w->qt >= w->nq) {
    w->qt = 0;
    if (w->nq > 0 && ++w->h < a.pool.kv_heads) continue;
    w->h = 0;
    ++w->s;
    w->nq = chunk_units<ChunkShape<D, Q8>::NQ>(a, w->s, &sp);
  }
  paged_span(a.spans, a.pool.page_shift, w->s, &sp);
  chunk_unit<D, Q8>(a, sp, w->qt, &p->u);
  p->h = w->h;
  p->cost = p->u.ue - p->u.ub;
  p->unit0 = w->unit0;
  p->begin = p->u.ub + int(w->t - w->unit0);
  p->end = int(min(int64_t(p->u.ue), p->begin + (w->t_end - w->t)));
  w->t += p->end - p->begin;
  w->unit0 += p->cost;
  ++w->qt;
  return true;
}

template <int D, bool Q8>
__global__ void __launch_bounds__((ChunkShape<D, Q8>::kThreads), 1)
    paged_chunk_kernel(const __grid_constant__ PagedAttendArgs a) {
  using S = ChunkShape<D, Q8>;
  constexpr int NQ = S::NQ, BM = S::BM, BN = S::BN;
  constexpr uint32_t kFmtS = Q8 ? 0u : 1u;  // f16 or bf16
  constexpr uint32_t kIdescQK = tc::instr_desc(kFmtS, false, BN, BM);
  constexpr uint32_t kIdescPV = tc::instr_desc(1u, true, D, BM);
  constexpr int kTileCols = 256;  // TMEM columns of a query tile (two of them)

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ int64_t before[kMaxPagedSequences + 1];
  __shared__ int64_t scratch[S::kThreads / 32];
  __shared__ ChunkWalk start;
  __shared__ uint32_t poison[2][BN / 32];  // by V stage: keys with a value that is not finite
  __shared__ uint32_t absent[4];  // by tile % 4: a bit per 16 keys whose page is out of range
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = smem;
  unsigned char* sK = smem + S::kAt_K;
  unsigned char* sV = smem + S::kAt_V;
  float* scales = reinterpret_cast<float*>(smem + S::kAt_Scales);  // [tile % 4][K, V][BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kAt_Bars);
  uint64_t* q_full = bars;                     // [2]: by query tile, once a piece it is part of
  uint64_t* k_full = bars + 2;                 // [2]
  uint64_t* k_empty = k_full + 2;              // [2]
  uint64_t* v_full = k_empty + 2;              // [2]
  uint64_t* v_empty = v_full + 2;              // [2]
  uint64_t* s_full = v_empty + 2;              // [2]: by query tile, or by score buffer
  uint64_t* p_full = s_full + 2;               // [2]: by query tile
  uint64_t* o_done = p_full + 2;               // [2]: each P.V
  uint64_t* o_final = o_done + 2;              // [2]: a piece's last P.V
  uint64_t* drained = o_final + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kLoader0 = NQ * 4, kMmaWarp = kLoader0 + 4;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_final[i], 1);
    }
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
    if (lane == 0) before[s] = sum;
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
  const int ctas = int(min(int64_t(gridDim.x), (work + 1) / 2));
  const int cta = blockIdx.x;
  const bool idle = cta >= ctas;
  if (!idle && warp == 0) {
    ChunkWalk w;
    w.t = share_begin(work, cta, ctas);
    w.t_end = share_begin(work, cta + 1, ctas);
    int s0 = 0, s1 = nseq;  // the last s with before[s] * kvh <= t
    while (s1 - s0 > 1) {
      const int mid = (s0 + s1) / 2;
      if (before[mid] * kvh <= w.t) s0 = mid; else s1 = mid;
    }
    w.s = s0;
    PagedSpan sp;
    w.nq = chunk_units<NQ>(a, s0, &sp);
    const int64_t per = before[s0 + 1] - before[s0];
    const int64_t rest = w.t - before[s0] * kvh;
    w.h = int(rest / per);
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
    if (lane == 0) start = w;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (!idle) {
    ChunkWalk walk = start;
    ChunkPiece pc;
    if (warp >= kMmaWarp) {
      // ---- MMA issuer ------------------------------------------------------------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
      if (warp == kMmaWarp && lane == 0) {
        const uint64_t q_desc = tc::smem_desc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t k_desc = tc::smem_desc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t v_desc = tc::smem_desc(smem_u32(sV), BN * 128, 1024, tc::kSwizzle128B);
        uint32_t tile = 0;        // K (and V) tiles consumed so far
        uint32_t queries[2] = {0, 0};  // pieces that each query tile was part of
        uint32_t pv[2] = {0, 0};  // P.V products of each query tile so far
        uint32_t sb = 0;          // one query tile: score products so far
        bool ok = true;
        while (ok && chunk_next<D, Q8>(a, &walk, &pc)) {
          const int n_tiles = pc.end - pc.begin;
          bool first[2] = {true, true};
          auto part = [&](int i, int L) {
            return pc.begin + L >= pc.u.tb[i] && pc.begin + L < pc.u.te[i];
          };
          auto issue_s = [&](int i, int L) {
            const uint64_t qd = q_desc + uint64_t(i * S::kQBytes >> 4);
            const uint64_t kd = k_desc + uint64_t((tile + L) % S::kKStages) * uint64_t(S::kTileBytes >> 4);
            const int b = NQ == 2 ? i : int(sb & 1);
            const uint32_t dst = tmem + (NQ == 2 ? i * kTileCols : b * BN);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const int db = k / 4, koff = (k % 4) * 32;
              tc::mma_ss<false>(dst, qd + uint64_t((db * BM * 128 + koff) >> 4),
                                kd + uint64_t((db * BN * 128 + koff) >> 4), kIdescQK, k > 0 ? 1u : 0u);
            }
            tc::commit(&s_full[b]);
            ++sb;
          };
          auto issue_pv = [&](int i, int L) {
            if (!mbar_wait(&p_full[i], pv[i] & 1, a.err)) return false;
            const uint32_t vt = tile + L;
            if (!mbar_wait(&v_full[vt % S::kVStages], (vt / S::kVStages) & 1, a.err)) return false;
            tc::fence_after_sync();
            const uint32_t p_tmem = tmem + (NQ == 2 ? i * kTileCols : int(pv[i] & 1) * BN);
            const uint32_t o_tmem = tmem + (NQ == 2 ? i * kTileCols : 0) + S::kO;
            const uint64_t vd = v_desc + uint64_t(vt % S::kVStages) * uint64_t(S::kTileBytes >> 4);
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              tc::mma_ts<false>(o_tmem, p_tmem + k * 8, vd + uint64_t((k * 16 * 128) >> 4), kIdescPV,
                                (!first[i] || k > 0) ? 1u : 0u);
            tc::commit(&o_done[i]);
            first[i] = false;
            ++pv[i];
            return true;
          };
          auto wait_k = [&](int L) {
            const uint32_t kt = tile + L;
            if (!mbar_wait(&k_full[kt % S::kKStages], (kt / S::kKStages) & 1, a.err)) return false;
            tc::fence_after_sync();
            return true;
          };
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if (min(pc.end, pc.u.te[i]) <= max(pc.begin, pc.u.tb[i])) continue;
            ok = ok && mbar_wait(&q_full[i], queries[i] & 1, a.err);
            ++queries[i];
          }
          if (!ok) break;
          ok = wait_k(0);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (part(i, 0)) issue_s(i, 0);
          tc::commit(&k_empty[tile % S::kKStages]);
          for (int L = 0; ok && L < n_tiles; ++L) {
            const bool next = L + 1 < n_tiles;
            if (next && !wait_k(L + 1)) { ok = false; break; }
            if constexpr (NQ == 2) {
              if (part(0, L) && !issue_pv(0, L)) { ok = false; break; }
              if (next && part(0, L + 1)) issue_s(0, L + 1);
              if (part(1, L) && !issue_pv(1, L)) { ok = false; break; }
              if (next && part(1, L + 1)) issue_s(1, L + 1);
            } else {
              if (next) issue_s(0, L + 1);
              if (!issue_pv(0, L)) { ok = false; break; }
            }
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
    } else if (warp >= kLoader0) {
      // ---- loaders ---------------------------------------------------------------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      const int tid = threadIdx.x - kLoader0 * 32;
      constexpr int kRB = D * (Q8 ? 1 : 2), kCR = kRB / 16;  // a page row's bytes and chunks
      constexpr int kPass = 128 / kCR;                       // rows of one pass of the threads
      constexpr int kPasses = BN / kPass;
      const int shift = a.pool.page_shift;
      const int chunk = tid % kCR, prow = tid / kCR;
      uint32_t tile = 0;
      bool ok = true, more = chunk_next<D, Q8>(a, &walk, &pc);
      // one key tile's numbers: its first position, the keys that rows of the unit see, and lane
      // i's page of keys 16 i .. 16 i + 15 (-1: none seen; -2: out of range, a bit of `absent`)
      struct Tile {
        int pos, lo, hi, lo_all, hi_all, h, page;
        uint32_t absent;
      };
      auto look = [&](int at, Tile* t) {
        const ChunkUnit& u = pc.u;
        const int last = min(u.q0 + NQ * chunk_rows(a), u.n) - 1;
        const int end = u.first + u.n;
        paged_keys(a.kind, a.window, u.first + u.q0, end, &t->lo, &t->hi_all);
        paged_keys(a.kind, a.window, u.first + last, end, &t->lo_all, &t->hi);
        t->pos = at * BN;
        t->h = pc.h;
        t->page = -1;
        const int p = t->pos + lane * 16;
        if (lane < BN / 16 && p < t->hi && p + 16 > t->lo) {
          // the span's table row: found by its sequence
          t->page = __ldg(a.spans.tables + int64_t(walk.s) * a.spans.table_stride + (p >> shift));
          if (!paged_page_ok(t->page, a.pool.pages)) {
            atomicOr(a.err, kErrPagedPage);
            t->page = -2;
          }
        }
        t->absent = __ballot_sync(0xffffffffu, t->page == -2);
      };
      // the thread's chunks of the tile's key (or value) rows, as one group of copies
      auto fetch = [&](const Tile& t, const unsigned char* base, uint32_t dst) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          const int row = prow + i * kPass;
          const int page = __shfl_sync(0xffffffffu, t.page, row >> 4);
          const int p = t.pos + row;
          const bool there = page >= 0 && p >= t.lo && p < t.hi;
          const int64_t at = ((int64_t(max(page, 0)) * kvh + t.h) << shift) + (p & ((1 << shift) - 1));
          const uint32_t to = Q8 ? uint32_t((tid + i * 128) * 16)
                                 : uint32_t((chunk / 8) * (BN * 128) + row * 128 +
                                            (((chunk % 8) ^ (row & 7)) * 16));
          cp_async16(dst + to, base + (there ? at * kRB + chunk * 16 : 0), there ? 16u : 0u);
        }
        cp_async_commit();
      };
      // a value tile on an edge: what is not finite taken out, its key marked
      auto scrub_bf16 = [&](unsigned char* dst, int stage) {
#pragma unroll 1
        for (int i = 0; i < kPasses; ++i) {
          const int row = prow + i * kPass;
          uint4* p = reinterpret_cast<uint4*>(dst + (chunk / 8) * (BN * 128) + row * 128 +
                                              (((chunk % 8) ^ (row & 7)) * 16));
          uint4 v = *p;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool bad = false;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if ((w[x] & 0x7F80u) == 0x7F80u) { w[x] &= 0xFFFF0000u; bad = true; }
            if ((w[x] & 0x7F800000u) == 0x7F800000u) { w[x] &= 0xFFFFu; bad = true; }
          }
          if (bad) {
            *p = make_uint4(w[0], w[1], w[2], w[3]);
            atomicOr(&poison[stage][row >> 5], 1u << (row & 31));
          }
        }
      };
      auto publish = [&](uint64_t* bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bar);
      };
      // A stage's products are done (its marks are cleared): decided by all loaders as one, so that
      // a wait that gave up cannot leave the others at this barrier.
      auto vacant = [&](uint64_t* bar, uint32_t parity, int marks = -1) {
        const bool there = mbar_wait(bar, parity, a.err);
        if (there && marks >= 0 && tid < BN / 32) poison[marks][tid] = 0;
        return !named_sync_or(1, 128, !there);
      };
      auto edge = [&](const Tile& t) { return t.pos < t.lo_all || t.pos + BN > t.hi_all; };

      if constexpr (!Q8) {
        // slots K0, V0, K1, V1, ...: each published when the next one's copies are on their way
        uint64_t* pending = nullptr;
        unsigned char* pending_v = nullptr;  // a V tile on an edge, to be scrubbed
        int pending_stage = 0;
        auto finish = [&]() {
          if (pending == nullptr) return;
          if (pending_v != nullptr) scrub_bf16(pending_v, pending_stage);
          publish(pending);
        };
        Tile t;
        if (more) look(pc.begin, &t);
        while (more && ok) {
          for (int at = pc.begin; at < pc.end; ++at, ++tile) {
            const int ks = tile % S::kKStages, vs = tile % S::kVStages;
            if (!vacant(&k_empty[ks], ((tile / S::kKStages) & 1) ^ 1)) { ok = false; break; }
            fetch(t, a.pool.keys, smem_u32(sK) + ks * S::kTileBytes);
            if (tid == 0) absent[tile & 3] = t.absent;
            cp_async_wait<1>();
            finish();
            pending = &k_full[ks];
            pending_v = nullptr;
            if (!vacant(&v_empty[vs], ((tile / S::kVStages) & 1) ^ 1, vs)) { ok = false; break; }
            fetch(t, a.pool.values, smem_u32(sV) + vs * S::kTileBytes);
            const bool e = edge(t);
            if (at + 1 < pc.end) look(at + 1, &t);
            cp_async_wait<1>();
            finish();
            pending = &v_full[vs];
            pending_v = e ? sV + vs * S::kTileBytes : nullptr;
            pending_stage = vs;
          }
          if (!ok) break;
          more = chunk_next<D, Q8>(a, &walk, &pc);
          if (more) look(pc.begin, &t);
        }
        cp_async_wait<0>();
        if (ok) finish();
      } else {
        unsigned char* raw = smem + S::kAt_Raw;  // a key tile, then a value tile
        // a tile's copies are under way while the one before it is converted
        Tile t, next;
        float ksc = 0.0f, vsc = 0.0f;  // thread i: key i's scales of tile t
        auto begin_tile = [&](const Tile& x, float* k, float* v) {
          *k = *v = 0.0f;
          const int page = __shfl_sync(0xffffffffu, x.page, (tid & (BN - 1)) >> 4);
          const int p = x.pos + (tid & (BN - 1));
          if (page >= 0 && p >= x.lo && p < x.hi) {
            const int64_t at = ((int64_t(page) * kvh + x.h) << shift) + (p & ((1 << shift) - 1));
            *k = __ldcg(a.pool.key_scales + at);
            *v = __ldcg(a.pool.value_scales + at);
          }
        };
        if (more) {
          look(pc.begin, &t);
          fetch(t, a.pool.keys, smem_u32(raw));
          fetch(t, a.pool.values, smem_u32(raw) + S::kRawBytes);
          begin_tile(t, &ksc, &vsc);
        }
        while (more && ok) {
          for (int at = pc.begin; at < pc.end;) {
            const int ks = tile % S::kKStages, vs = tile % S::kVStages;
            const bool e = edge(t);
            // the tile after this one, of this piece or the next
            ++at;
            bool have = true;
            if (at == pc.end) {
              have = more = chunk_next<D, Q8>(a, &walk, &pc);
              at = pc.begin;
            }
            if (have) look(at, &next);
            float nk = 0.0f, nv = 0.0f;
            if (have) begin_tile(next, &nk, &nv);
            // keys
            if (!vacant(&k_empty[ks], ((tile / S::kKStages) & 1) ^ 1)) { ok = false; break; }
            cp_async_wait<1>();
            {
              unsigned char* dst = sK + ks * S::kTileBytes;
#pragma unroll
              for (int i = 0; i < kPasses; ++i) {
                const int row = prow + i * kPass;
                const uint4 v = *reinterpret_cast<const uint4*>(raw + (tid + i * 128) * 16);
                const int c0 = chunk * 2;
                unsigned char* p = dst + (c0 / 8) * (BN * 128) + row * 128;
                *reinterpret_cast<uint4*>(p + ((c0 % 8) ^ (row & 7)) * 16) =
                    make_uint4(bytes_to_f16(v.x), bytes_to_f16(v.x >> 8), bytes_to_f16(v.y),
                               bytes_to_f16(v.y >> 8));
                *reinterpret_cast<uint4*>(p + ((c0 % 8 + 1) ^ (row & 7)) * 16) =
                    make_uint4(bytes_to_f16(v.z), bytes_to_f16(v.z >> 8), bytes_to_f16(v.w),
                               bytes_to_f16(v.w >> 8));
              }
            }
            if (tid < BN) scales[(tile & 3) * 2 * BN + tid] = ksc;
            if (tid == 0) absent[tile & 3] = t.absent;
            publish(&k_full[ks]);
            if (have) fetch(next, a.pool.keys, smem_u32(raw)); else cp_async_commit();
            // values
            if (!vacant(&v_empty[vs], ((tile / S::kVStages) & 1) ^ 1, vs)) { ok = false; break; }
            cp_async_wait<1>();
            {
              unsigned char* dst = sV + vs * S::kTileBytes;
#pragma unroll
              for (int i = 0; i < kPasses; ++i) {
                const int row = prow + i * kPass;
                const uint4 v = *reinterpret_cast<const uint4*>(raw + S::kRawBytes + (tid + i * 128) * 16);
                const int c0 = chunk * 2;
                unsigned char* p = dst + (c0 / 8) * (BN * 128) + row * 128;
                *reinterpret_cast<uint4*>(p + ((c0 % 8) ^ (row & 7)) * 16) =
                    make_uint4(bytes_to_bf16(v.x), bytes_to_bf16(v.x >> 8), bytes_to_bf16(v.y),
                               bytes_to_bf16(v.y >> 8));
                *reinterpret_cast<uint4*>(p + ((c0 % 8 + 1) ^ (row & 7)) * 16) =
                    make_uint4(bytes_to_bf16(v.z), bytes_to_bf16(v.z >> 8), bytes_to_bf16(v.w),
                               bytes_to_bf16(v.w >> 8));
              }
            }
            if (tid < BN) {
              if (e && !(fabsf(vsc) <= 3.402823466e38f)) {
                vsc = 0.0f;
                atomicOr(&poison[vs][tid >> 5], 1u << (tid & 31));
              }
              scales[(tile & 3) * 2 * BN + BN + tid] = vsc;
            }
            publish(&v_full[vs]);
            if (have) fetch(next, a.pool.values, smem_u32(raw) + S::kRawBytes); else cp_async_commit();
            ++tile;
            t = next;
            ksc = nk;
            vsc = nv;
            if (!have) break;
          }
        }
        cp_async_wait<0>();
      }
    } else {
      // ---- softmax and output of query tile i ------------------------------------------------
      if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
      const int i = NQ == 2 ? warp >> 2 : 0;
      const int wq = warp & 3;             // the TMEM lane quarter that this warp may access
      const int p = wq * 32 + lane;        // packed row
      const int rows = chunk_rows(a);
      const int pr = p / a.group, ph = p % a.group;
      const uint32_t lane_base = tmem + (NQ == 2 ? i * kTileCols : 0) + (uint32_t(wq * 32) << 16);
      const uint32_t o_base = lane_base + S::kO;
      uint32_t sc = 0;     // this query tile's score tiles so far
      uint32_t finals = 0; // pieces that it took part in
      uint32_t tile = 0;   // K (and V) tiles so far
      bool ok = true;
      while (ok && chunk_next<D, Q8>(a, &walk, &pc)) {
        const int n_tiles = pc.end - pc.begin;
        const int r = pc.u.q0 + i * rows + pr;  // row of the span
        const bool valid = pr < rows && r < pc.u.n;
        float scale = a.scale_log2;
        if (min(pc.end, pc.u.te[i]) > max(pc.begin, pc.u.tb[i])) {
          // the packed row's query, zeros for a row that is none; over 8-bit pages f16, scaled by
          // a power of two, its elements in the converted keys' order
          const int64_t at = int64_t(pc.u.row0 + r) * a.q_stride + int64_t(pc.h * a.group + ph) * D;
          unsigned char* dst = sQ + i * S::kQBytes + p * 128;
          auto load8 = [&](int c, float (&x)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            if (!valid) return;
            if (a.q_bf16) {
              const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + at + c * 8;
              if (a.q_vec) {
                const uint4 w = *reinterpret_cast<const uint4*>(q);
                x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
                x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z); x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __bfloat162float(q[e]);
              }
            } else {
              const float* q = static_cast<const float*>(a.q) + at + c * 8;
              if (a.q_vec) {
                const float4 u = reinterpret_cast<const float4*>(q)[0];
                const float4 v = reinterpret_cast<const float4*>(q)[1];
                x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
                x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = q[e];
              }
            }
          };
          float up = 1.0f;
          if constexpr (Q8) {
            float top = 0.0f;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              float x[8];
              load8(c, x);
#pragma unroll
              for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
            }
            const int e = min(max(int(__float_as_uint(top) >> 23), 1), 253);
            up = __uint_as_float(uint32_t(254 - e) << 23);
            scale *= __uint_as_float(uint32_t(e) << 23);
          }
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            float x[8];
            load8(c, x);
            uint4 w;
            if constexpr (Q8)
              w = make_uint4(pack_f16(x[0] * up, x[2] * up), pack_f16(x[1] * up, x[3] * up),
                             pack_f16(x[4] * up, x[6] * up), pack_f16(x[5] * up, x[7] * up));
            else
              w = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                             pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
            *reinterpret_cast<uint4*>(dst + (c / 8) * (BM * 128) + ((c % 8) ^ (p & 7)) * 16) = w;
          }
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
        int c = 0;  // score tiles of this piece so far
        for (int L = 0; L < n_tiles; ++L) {
          const int at = pc.begin + L;
          if (at < pc.u.tb[i] || at >= pc.u.te[i]) continue;
          const int kp = at * BN;
          const uint32_t s_base = lane_base + (NQ == 2 ? 0 : int(sc & 1) * BN);
          // every decision before a whole-warp tcgen05 instruction is made warp-uniform
          const bool there = NQ == 2 ? mbar_wait(&s_full[i], sc & 1, a.err)
                                     : mbar_wait(&s_full[sc & 1], (sc >> 1) & 1, a.err);
          if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
          tc::fence_after_sync();
          uint32_t sreg[BN];
#pragma unroll
          for (int x = 0; x < BN / 64; ++x)
            tc::tmem_ld64_wait(s_base + x * 64, *reinterpret_cast<uint32_t(*)[64]>(&sreg[x * 64]));
          float* s = reinterpret_cast<float*>(sreg);
          const float* sc_k = scales + ((tile + L) & 3) * 2 * BN;
          if constexpr (Q8) {
#pragma unroll
            for (int x = 0; x < BN; x += 4) {
              const float4 k = *reinterpret_cast<const float4*>(sc_k + x);
              s[x] *= k.x; s[x + 1] *= k.y; s[x + 2] *= k.z; s[x + 3] *= k.w;
            }
          }
          const bool all_in = !valid || (kp >= runs.b0 && kp + BN <= runs.b0 + runs.n0);
          if (!all_in) mask_scores<BN>(runs, kp, s);
          const uint32_t gone = *const_cast<const volatile uint32_t*>(&absent[(tile + L) & 3]);
          if (gone != 0) {
#pragma unroll
            for (int x = 0; x < BN; ++x)
              if ((gone >> (x >> 4)) & 1u) s[x] = -INFINITY;
          }
          float mx0 = fmax3(s[0], s[1], s[2]), mx1 = fmax3(s[3], s[4], s[5]);
          float mx2 = fmax3(s[6], s[7], s[8]), mx3 = fmax3(s[9], s[10], s[11]);
#pragma unroll
          for (int x = 12; x < BN - 4; x += 8) {
            mx0 = fmax3(mx0, s[x], s[x + 1]);
            mx1 = fmax3(mx1, s[x + 2], s[x + 3]);
            mx2 = fmax3(mx2, s[x + 4], s[x + 5]);
            mx3 = fmax3(mx3, s[x + 6], s[x + 7]);
          }
          mx0 = fmax3(mx0, s[BN - 4], s[BN - 3]);
          mx1 = fmax3(mx1, s[BN - 2], s[BN - 1]);
          const float m_tile = fmax3(mx0, mx1, fmaxf(mx2, mx3)) * scale;
          float alpha = 1.0f;
          if (m_tile > m_used + 8.0f || (m_used == -INFINITY && m_tile > -INFINITY)) {
            if (m_used > -INFINITY) alpha = exp2_approx(m_used - m_tile);
            m_used = m_tile;
          }
          const float ms = m_used == -INFINITY ? 0.0f : m_used;
          const float2 scale2 = make_float2(scale, scale), neg2 = make_float2(-ms, -ms);
          float2 sum2a = make_float2(0.0f, 0.0f), sum2b = make_float2(0.0f, 0.0f);
          const float* sc_v = sc_k + BN;
          if constexpr (Q8) {
            // the values' scales are there with the values
            const uint32_t vt = tile + L;
            const bool v_there = mbar_wait(&v_full[vt % S::kVStages], (vt / S::kVStages) & 1, a.err);
            if (!__all_sync(0xffffffffu, v_there)) { ok = false; break; }
          }
#pragma unroll
          for (int x = 0; x < BN; x += 4) {
            const float2 x0 = __ffma2_rn(make_float2(s[x], s[x + 1]), scale2, neg2);
            const float2 x1 = __ffma2_rn(make_float2(s[x + 2], s[x + 3]), scale2, neg2);
            float2 p0 = make_float2(exp2_approx(x0.x), exp2_approx(x0.y));
            float2 p1 = make_float2(exp2_approx(x1.x), exp2_approx(x1.y));
            sum2a = __fadd2_rn(sum2a, p0);
            sum2b = __fadd2_rn(sum2b, p1);
            if constexpr (Q8) {
              const float4 v = *reinterpret_cast<const float4*>(sc_v + x);
              p0 = __fmul2_rn(p0, make_float2(v.x, v.y));
              p1 = __fmul2_rn(p1, make_float2(v.z, v.w));
            }
            sreg[x / 2] = tc::pack_bf16(p0.x, p0.y);
            sreg[x / 2 + 1] = tc::pack_bf16(p1.x, p1.y);
          }
#pragma unroll
          for (int x = 0; x < BN / 64; ++x)
            tc::tmem_st32(s_base + x * 32, *reinterpret_cast<const uint32_t(*)[32]>(&sreg[x * 32]));
          l_sum = l_sum * alpha + ((sum2a.x + sum2a.y) + (sum2b.x + sum2b.y));
          if (kp < lo_all || kp + BN > hi_all) {
            // an edge tile (of the unit, as the loaders see it): keys that they marked
            const uint32_t vt = tile + L;
            const bool v_there = mbar_wait(&v_full[vt % S::kVStages], (vt / S::kVStages) & 1, a.err);
            if (!__all_sync(0xffffffffu, v_there)) { ok = false; break; }
            const volatile uint32_t* marks = poison[vt % S::kVStages];
#pragma unroll
            for (int w = 0; w < BN / 32; ++w)
              if (marks[w] & run_word(runs.b0, runs.n0, kp, w)) poisoned = true;
          }
          if (__any_sync(0xffffffffu, alpha != 1.0f) && c > 0) {
            // O holds the products of this piece's earlier tiles, the last of which may still run
            if (!__all_sync(0xffffffffu, mbar_wait(&o_done[i], (sc - 1) & 1, a.err))) { ok = false; break; }
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
          mbar_arrive(&p_full[i]);
          ++c;
          ++sc;
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
        const int c0 = share_owner(work, pc.unit0, ctas);
        const int c1 = share_owner(work, pc.unit0 + pc.cost - 1, ctas);
        const int64_t orow = int64_t(pc.u.row0 + r) * a.out_stride + int64_t(pc.h * a.group + ph) * D;
        // 32 columns of O in the elements' order
        auto order = [&](uint32_t (&o)[32]) {
          if constexpr (Q8) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              const uint32_t y = o[x + 1];
              o[x + 1] = o[x + 2];
              o[x + 2] = y;
            }
          }
        };
        auto write_out = [&](int cc, const float (&x)[32], float inv) {
          if (a.out_bf16) {
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + orow + cc * 32;
            if (a.out_vec) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<uint4*>(dst)[e] =
                    make_uint4(pack_bf16x2(x[8 * e] * inv, x[8 * e + 1] * inv),
                               pack_bf16x2(x[8 * e + 2] * inv, x[8 * e + 3] * inv),
                               pack_bf16x2(x[8 * e + 4] * inv, x[8 * e + 5] * inv),
                               pack_bf16x2(x[8 * e + 6] * inv, x[8 * e + 7] * inv));
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) dst[e] = __float2bfloat16_rn(x[e] * inv);
            }
          } else {
            float* dst = static_cast<float*>(a.out) + orow + cc * 32;
            if (a.out_vec) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                reinterpret_cast<float4*>(dst)[e] = make_float4(
                    x[4 * e] * inv, x[4 * e + 1] * inv, x[4 * e + 2] * inv, x[4 * e + 3] * inv);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) dst[e] = x[e] * inv;
            }
          }
        };
        if (c0 == c1) {
          const float inv = l_sum == 0.0f ? 0.0f : 1.0f / l_sum;
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            if (have) tc::tmem_ld32_wait(o_base + cc * 32, o);
            else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            order(o);
            if (valid) write_out(cc, *reinterpret_cast<const float(*)[32]>(&o), inv);
          }
        } else {
          // a piece: partials by float4s of 128 packed rows (a warp's stores are contiguous)
          const int64_t slot = (int64_t(2 * cta + (cta == c0 ? 1 : 0)) * NQ + i);
          if (have) {
#pragma unroll 1
            for (int cc = 0; cc < D / 32; ++cc) {
              uint32_t o[32];
              tc::tmem_ld32_wait(o_base + cc * 32, o);
              order(o);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(a.part_o + ((slot * (D / 4) + cc * 8 + e) * 128 + p) * 4) =
                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
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
          if (__shfl_sync(0xffffffffu, last, 0) != 0) {
            __threadfence();
            auto slot_of = [&](int x) { return int64_t(2 * x + (x == c0 ? 1 : 0)) * NQ + i; };
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll 4
            for (int x = c0; x <= c1; ++x)
              mm = fmaxf(mm, __ldcg(a.part_ml + (slot_of(x) * 128 + p) * 2));
#pragma unroll 4
            for (int x = c0; x <= c1; ++x) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + (slot_of(x) * 128 + p) * 2));
              ll += ml.x == -INFINITY ? ml.y : ml.y * exp2_approx(ml.x - mm);
            }
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll 1
            for (int cc = 0; cc < D / 32; ++cc) {
              float acc[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) acc[e] = 0.0f;
#pragma unroll 1
              for (int x = c0; x <= c1; ++x) {
                const float mx = __ldcg(a.part_ml + (slot_of(x) * 128 + p) * 2);
                if (mx == -INFINITY) continue;  // no key of that piece is seen: its O is not there
                const float f = exp2_approx(mx - mm);
                const float* src = a.part_o + ((slot_of(x) * (D / 4) + cc * 8) * 128 + p) * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float4 v = __ldcg(reinterpret_cast<const float4*>(src + e * 512));
                  acc[4 * e] = fmaf(f, v.x, acc[4 * e]);
                  acc[4 * e + 1] = fmaf(f, v.y, acc[4 * e + 1]);
                  acc[4 * e + 2] = fmaf(f, v.z, acc[4 * e + 2]);
                  acc[4 * e + 3] = fmaf(f, v.w, acc[4 * e + 3]);
                }
              }
              if (valid) write_out(cc, acc, inv);
            }
          }
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

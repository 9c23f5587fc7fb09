// Rows into pages and back: head norm, RoPE and the 8-bit quantisation of a call's keys and
// values as they are written (PagedWriteArgs), and the rows read back out (PagedReadArgs).
//
// 8-bit pages: with a = max|x_e| over a head's elements, scale = a / 127 and q_e = round(x_e *
// (127 / a)) to the nearest even, in f32: |x_e - q_e scale| <= scale / 2. A head below 2^-100
// everywhere is kept as zeros (127 / a must not overflow), and one with an infinity or a NaN as
// a NaN scale (it reads back as NaN throughout, and attends as NaN where it is seen).
#include <cuda_bf16.h>

#include <type_traits>

#include "fa_paged.h"
#include "fa_ptx.cuh"

namespace fa {

namespace {

constexpr int kRowWarps = 4;

// Row r's place: its page and slot. kNoRow if no sequence holds the row (rows before the first
// sequence's and past the last's are padding) or its span is out of range, kNoPage if its page is;
// what is out of range is set in the error word. One warp; two trips to memory (three
// for more than 32 sequences): the row's sequence s is the number of sequences that end at or
// before it (row_starts rises, or the span check refuses what is found), and each lane has its
// sequence's span at hand when s is known.
constexpr int kNoRow = 0, kNoPage = 1, kPlaced = 2;

__device__ __forceinline__ int place_of(const PagedSpans& b, const PagedPool& pool, int r,
                                        int lane, int* page, int* slot, unsigned* err) {
  int base = 0;
  if (b.sequences > 32) {
    const int at = (lane + 1) * 32;  // the end of block `lane` of 32 sequences
    const bool past = at <= b.sequences && b.row_starts[at] <= r;
    base = 32 * __popc(__ballot_sync(0xffffffffu, past));
  }
  const int mine = base + lane;
  int r0 = 0, r1 = 0x7fffffff, first = 0;
  if (mine < b.sequences) {
    r0 = b.row_starts[mine];
    r1 = b.row_starts[mine + 1];
    first = b.firsts[mine];
  }
  const int in = __popc(__ballot_sync(0xffffffffu, mine < b.sequences && r1 <= r));
  const int s = base + in;
  if (s >= b.sequences) return kNoRow;
  r0 = __shfl_sync(0xffffffffu, r0, in & 31);
  r1 = __shfl_sync(0xffffffffu, r1, in & 31);
  first = __shfl_sync(0xffffffffu, first, in & 31);
  PagedSpan span;
  const bool ok = in < 32 && paged_span_of(b, pool.page_shift, r0, r1, first, &span);
  if (!ok || r < span.row0 || r >= span.row0 + span.n) {
    if (lane == 0 && !(ok && s == 0 && r < span.row0)) atomicOr(err, kErrPagedSpan);
    return kNoRow;
  }
  const int pos = span.first + (r - span.row0);
  *page = b.tables[int64_t(s) * b.table_stride + (pos >> pool.page_shift)];
  *slot = pos & ((1 << pool.page_shift) - 1);
  if (!paged_page_ok(*page, pool.pages)) {
    if (lane == 0) atomicOr(err, kErrPagedPage);
    return kNoPage;
  }
  return kPlaced;
}

// Four consecutive elements: one load where the row is aligned for it.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, T* x) {
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(p));
    else *reinterpret_cast<uint2*>(x) = __ldcs(reinterpret_cast<const uint2*>(p));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p[e];
  }
}

template <int E>
__device__ __forceinline__ void store_elems(void* base, int64_t at, bool bf16, bool vec,
                                            const float (&x)[E]) {
  if (bf16) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + at;
    if (vec) {
      alignas(16) __nv_bfloat162 raw[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) raw[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      if constexpr (E == 2) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(raw);
      else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(raw);
      else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(raw);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = __float2bfloat16_rn(x[e]);
    }
  } else {
    float* p = static_cast<float*>(base) + at;
    if (vec) {
      if constexpr (E == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
      else {
#pragma unroll
        for (int e = 0; e < E / 4; ++e)
          reinterpret_cast<float4*>(p)[e] =
              make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = x[e];
    }
  }
}

// Two words' low bytes, then two more's, as one word.
__device__ __forceinline__ uint32_t pack_bytes(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One CTA per row. A head's elements lie eight to a lane on D / 8 lanes, four of each half (the
// partners of RoPE by halves are in one lane, and those of interleaved RoPE too), so that a warp
// takes 32 / (D / 8) heads of one kind (queries, keys, values) at a time (a step); it takes every
// kRowWarps-th step, the first one's loads issued before the row's place is looked up and each next
// one's before the last is worked on. The row's cosines and sines are loaded once for all of a
// warp's heads. Arithmetic of the rotation: each product rounded, then the difference or sum
// (ops.rs:77-95).
// Bound by issued instructions (80 % of the cycles of a long call) with memory close behind, so each
// kind has a loop of its own, and calls whose arrays are all 16-byte aligned have a kernel without
// the element-wise accesses (Vec): 8500 rows of 32/8 heads of 128 (bf16 rows, 8-bit pages, 196 MB)
// take 42 us (4.7 TB/s), 51 us in one loop of all kinds that tests the alignment; 2800 f32 rows of
// 8/2 heads of 256 with head norms into bf16 pages 16 us; the keys and values alone, as they are, of
// 8500 rows 20 us. The arithmetic is one f32 at a time, and 40 registers (12 CTAs an SM) spill 12 to 48
// bytes of stores in every instantiation.
template <typename T, int D, bool Vec>
__global__ void __launch_bounds__(kRowWarps * 32, 12)
    paged_write_kernel(const __grid_constant__ PagedWriteArgs a) {
  constexpr int LH = D / 8, HW = 32 / LH;  // lanes of a head, heads of a step
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % LH, which = lane / LH;
  const int lo = sub * 4;  // this lane's elements lo .. lo + 3 and D / 2 + lo ..
  const int r = blockIdx.x;
  const int kvh = a.pool.kv_heads;
  const int q_steps = a.q_out == nullptr ? 0 : (a.heads + HW - 1) / HW, kv_steps = (kvh + HW - 1) / HW;
  const int steps = q_steps + 2 * kv_steps;
  alignas(16) T raw[8];
  auto load = [&](const void* base, int64_t row, int64_t head, int heads, int t) {
    const int h = t * HW + which;
    if (h >= heads) return;  // (the lane keeps what it had)
    const T* p = static_cast<const T*>(base) + r * row + h * head + lo;
    load4(p, Vec, raw);
    load4(p + D / 2, Vec, raw + 4);
  };
  auto load_any = [&](int t) {
    if (t < q_steps) load(a.q, a.q_stride, D, a.heads, t);
    else if (t < q_steps + kv_steps) load(a.k, a.k_stride, a.k_head_stride, kvh, t - q_steps);
    else if (t < steps) load(a.v, a.v_stride, a.v_head_stride, kvh, t - q_steps - kv_steps);
  };
#pragma unroll
  for (int e = 0; e < 8; ++e) raw[e] = T(0.0f);
  load_any(warp);
  alignas(16) float c[4], s[4];
  if (a.rope != 0) {
    // by halves: the elements' own; interleaved: of pairs lo / 2, lo / 2 + 1, and those of D / 2 + lo
    const float* cs = a.angles + int64_t(r) * D;
    if (a.rope == 1) {
      load4(cs + lo, Vec, c);
      load4(cs + D / 2 + lo, Vec, s);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int pair = (e & 1) + lo / 2 + (e >> 1) * (D / 4);
        c[e] = cs[pair];
        s[e] = cs[D / 2 + pair];
      }
    }
  }
  int page, slot;
  const int place = place_of(a.spans, a.pool, r, lane, &page, &slot, a.err);  // the warp's, as one
  if (place == kNoRow) return;
  const int64_t row0 = ((int64_t(page) * kvh) << a.pool.page_shift) + slot;  // KV head 0's
  // The steps of one kind: 0 queries, 1 keys, 2 values; `begin` of them all to `end`.
  int t = warp;
  auto section = [&](auto kind_c, int begin, int end) {
    constexpr int kind = decltype(kind_c)::value;
    const int heads = kind == 0 ? a.heads : kvh;
    for (; t < end; t += kRowWarps) {
      const int h = (t - begin) * HW + which;
      const bool live = h < heads;
      float x[8];  // elements lo .. lo + 3, D / 2 + lo ..
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = float(raw[e]);
      if (kind == 0 && t + kRowWarps < end) load(a.q, a.q_stride, D, heads, t + kRowWarps);
      else load_any(t + kRowWarps);
      if constexpr (kind < 2) {
        const float* weight = kind == 0 ? a.q_norm : a.k_norm;
        if (weight != nullptr) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int off = LH / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
          const float inverse = 1.0f / sqrtf(ss / float(D) + a.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = __fmul_rn(__fmul_rn(x[e], inverse), weight[(e >> 2) * (D / 2) + lo + (e & 3)]);
        }
        auto turn = [&](float& x0, float& x1, int i) {
          const float y0 = x0, y1 = x1;
          x0 = __fsub_rn(__fmul_rn(y0, c[i]), __fmul_rn(y1, s[i]));
          x1 = __fadd_rn(__fmul_rn(y1, c[i]), __fmul_rn(y0, s[i]));
        };
        if (a.rope == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) turn(x[e], x[4 + e], e);
        } else if (a.rope == 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) turn(x[2 * e], x[2 * e + 1], e);
        }
      }
      const float(&x0)[4] = *reinterpret_cast<const float(*)[4]>(&x[0]);
      const float(&x1)[4] = *reinterpret_cast<const float(*)[4]>(&x[4]);
      if constexpr (kind == 0) {
        if (live) {
          const int64_t at = r * a.q_out_stride + h * D + lo;
          store_elems<4>(a.q_out, at, a.q_out_bf16 != 0, Vec, x0);
          store_elems<4>(a.q_out, at + D / 2, a.q_out_bf16 != 0, Vec, x1);
        }
      } else {
        const int64_t row = row0 + (int64_t(h) << a.pool.page_shift);
        unsigned char* base = kind == 1 ? a.pool.keys : a.pool.values;
        if (!a.pool.q8) {
          if (live) {
            store_elems<4>(base, row * D + lo, true, true, x0);
            store_elems<4>(base, row * D + D / 2 + lo, true, true, x1);
          }
          continue;
        }
        // the largest |x|, as integers (they rise with the floats; an infinity or a NaN is above all)
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
        for (int off = LH / 2; off >= 1; off >>= 1)
          bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, off));
        const float top = __uint_as_float(bits);
        const bool finite = bits < 0x7f800000u;
        const bool some = finite && top >= 7.888609052e-31f;  // 2^-100
        const float inverse = some ? __fdiv_rn(127.0f, top) : 0.0f;
        // x (127 / top) is within +-127 but for two roundings, and so rounds to -127 .. 127; what is
        // not finite times 0 converts to 0
        int n[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] = __float2int_rn(__fmul_rn(x[e], inverse));
        if (!live) continue;
        unsigned char* to = base + row * D + lo;
        *reinterpret_cast<uint32_t*>(to) = pack_bytes(n[0], n[1], n[2], n[3]);
        *reinterpret_cast<uint32_t*>(to + D / 2) = pack_bytes(n[4], n[5], n[6], n[7]);
        if (sub == 0)
          (kind == 1 ? a.pool.key_scales : a.pool.value_scales)[row] =
              !finite ? __int_as_float(0x7fffffff) : some ? __fdiv_rn(top, 127.0f) : 0.0f;
      }
    }
  };
  section(std::integral_constant<int, 0>{}, 0, q_steps);
  if (place == kNoPage) return;  // (the row's query is rotated all the same: it attends)
  section(std::integral_constant<int, 1>{}, q_steps, q_steps + kv_steps);
  section(std::integral_constant<int, 2>{}, q_steps + kv_steps, steps);
}

// A warp takes two rows: their places, then 16 bytes of them a lane at a time, eight such loads in
// flight (two vectors of keys and of values of each row). 125 thousand positions of 8 KV heads of 128
// to bf16 rows take 159 us out of bf16 pages (1029 MB, 6.5 TB/s: the rate of a copy) and 161 us out
// of 8-bit pages (780 MB, 4.8 TB/s: a lane stores 32 bytes in two vectors, so that each store
// instruction of a warp writes half of every sector that it touches; so do bf16 pages to f32 rows,
// at 5.7 TB/s).
constexpr int kReadWarps = 8, kReadRows = 2 * kReadWarps;

template <bool Q8, int D>
__global__ void __launch_bounds__(kReadWarps * 32)
    paged_read_kernel(const __grid_constant__ PagedReadArgs a) {
  constexpr int kElems = Q8 ? 16 : 8;          // of a 16-byte vector
  constexpr int kPerHead = D / kElems;         // vectors of a head
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = blockIdx.x * kReadRows + warp;
  int64_t place[2];  // (page, slot)'s row of KV head 0, or -1
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + i * kReadWarps;
    int page = 0, slot = 0;
    const bool ok = r < a.spans.rows &&
                    place_of(a.spans, a.pool, r, lane, &page, &slot, a.err) == kPlaced;
    place[i] = ok ? ((int64_t(page) * a.pool.kv_heads) << a.pool.page_shift) + slot : -1;
  }
  const int vectors = a.pool.kv_heads * kPerHead;
  for (int x0 = lane; x0 < vectors; x0 += 64) {
    uint4 raw[2][2][2];   // [row][vector][keys, values]
    float scale[2][2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int x = x0 + 32 * j;
        if (place[i] < 0 || x >= vectors) continue;
        const int64_t at = place[i] + (int64_t(x / kPerHead) << a.pool.page_shift);
        raw[i][j][0] = __ldcs(reinterpret_cast<const uint4*>(a.pool.keys) + at * kPerHead + x % kPerHead);
        raw[i][j][1] = __ldcs(reinterpret_cast<const uint4*>(a.pool.values) + at * kPerHead + x % kPerHead);
        if constexpr (Q8) {
          scale[i][j][0] = a.pool.key_scales[at];
          scale[i][j][1] = a.pool.value_scales[at];
        }
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int x = x0 + 32 * j;
        if (place[i] < 0 || x >= vectors) continue;
        const int64_t r = r0 + i * kReadWarps;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          void* out = kv ? a.v : a.k;
          const int64_t to = r * (kv ? a.v_stride : a.k_stride) +
                             int64_t(x / kPerHead) * (kv ? a.v_head_stride : a.k_head_stride) +
                             (x % kPerHead) * kElems;
          const uint4 w4 = raw[i][j][kv];
          if constexpr (Q8) {
            const signed char* q = reinterpret_cast<const signed char*>(&w4);
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = float(q[e]) * scale[i][j][kv];
            store_elems<8>(out, to, a.out_bf16 != 0, a.vec != 0, *reinterpret_cast<const float(*)[8]>(&y[0]));
            store_elems<8>(out, to + 8, a.out_bf16 != 0, a.vec != 0, *reinterpret_cast<const float(*)[8]>(&y[8]));
          } else {
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = bf16_lo(w[e]);
              y[2 * e + 1] = bf16_hi(w[e]);
            }
            store_elems<8>(out, to, a.out_bf16 != 0, a.vec != 0, y);
          }
        }
      }
  }
}

// A plain stream-ordered launch that the kernel before it may overlap (it waits for it).
template <typename Args>
cudaError_t launch(void (*kernel)(Args), int grid, int block, const Args& args,
                   cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(block));
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

}  // namespace

cudaError_t launch_paged_write(const PagedWriteArgs& a, cudaStream_t stream) {
  if (a.spans.rows == 0) return cudaSuccess;
  const int d = a.pool.head_dim;
  // (of every array that is there, each 16-byte aligned; else element by element)
  const bool vec = a.vec != 0 && (a.rope != 1 || a.angles_vec != 0) && (a.q_out == nullptr || a.q_out_vec != 0);
  auto go = [&](auto t, auto dim) {
    using T = decltype(t);
    constexpr int D = decltype(dim)::value;
    return launch(vec ? paged_write_kernel<T, D, true> : paged_write_kernel<T, D, false>, a.spans.rows,
                  kRowWarps * 32, a, stream);
  };
  auto dims = [&](auto t) {
    if (d == 64) return go(t, std::integral_constant<int, 64>{});
    if (d == 128) return go(t, std::integral_constant<int, 128>{});
    if (d == 256) return go(t, std::integral_constant<int, 256>{});
    return cudaErrorInvalidValue;
  };
  return a.in_bf16 ? dims(__nv_bfloat16(0.0f)) : dims(0.0f);
}

cudaError_t launch_paged_read(const PagedReadArgs& a, cudaStream_t stream) {
  if (a.spans.rows == 0) return cudaSuccess;
  auto go = [&](void (*k)(PagedReadArgs)) {
    return launch(k, (a.spans.rows + kReadRows - 1) / kReadRows, kReadWarps * 32, a, stream);
  };
  switch (a.pool.head_dim) {
    case 64: return go(a.pool.q8 ? paged_read_kernel<true, 64> : paged_read_kernel<false, 64>);
    case 128: return go(a.pool.q8 ? paged_read_kernel<true, 128> : paged_read_kernel<false, 128>);
    case 256: return go(a.pool.q8 ? paged_read_kernel<true, 256> : paged_read_kernel<false, 256>);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace fa

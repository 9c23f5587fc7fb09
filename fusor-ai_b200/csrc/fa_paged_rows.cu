// Rows into pages and back: head norm, RoPE and the 8-bit quantisation of a call's keys and
// values as they are written (PagedWriteArgs), and the rows read back out (PagedReadArgs).
//
// 8-bit pages: with a = max|x_e| over a head's elements, scale = a / 127 and q_e = round(x_e *
// (127 / a)) to the nearest even, in f32: |x_e - q_e scale| <= scale / 2. A head below 2^-100
// everywhere is kept as zeros (127 / a must not overflow), and one with an infinity or a NaN as
// a NaN scale (it reads back as NaN throughout, and attends as NaN where it is seen).
#include <cuda_bf16.h>

#include "fa_paged.h"
#include "fa_ptx.cuh"

namespace fa {

namespace {

constexpr int kRowWarps = 4;

// Row r's place: its page and slot, or false (with the error word set) if the batch's numbers are
// out of range. Rows past the last sequence's are left alone. One warp; two trips to memory (three
// for more than 32 sequences): the row's sequence s is the number of sequences that end at or
// before it (row_starts rises, or the span check refuses what is found), and each lane has its
// sequence's span at hand when s is known.
__device__ __forceinline__ bool place_of(const PagedSpans& b, const PagedPool& pool, int r,
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
  if (s >= b.sequences) return false;
  r0 = __shfl_sync(0xffffffffu, r0, in & 31);
  r1 = __shfl_sync(0xffffffffu, r1, in & 31);
  first = __shfl_sync(0xffffffffu, first, in & 31);
  PagedSpan span;
  const bool ok = in < 32 && paged_span_of(b, pool.page_shift, r0, r1, first, &span);
  if (!ok || r < span.row0 || r >= span.row0 + span.n) {
    if (lane == 0) atomicOr(err, kErrPagedSpan);
    return false;
  }
  const int pos = span.first + (r - span.row0);
  *page = b.tables[int64_t(s) * b.table_stride + (pos >> pool.page_shift)];
  *slot = pos & ((1 << pool.page_shift) - 1);
  if (!paged_page_ok(*page, pool.pages)) {
    if (lane == 0) atomicOr(err, kErrPagedPage);
    return false;
  }
  return true;
}

// E consecutive elements as f32: one vector load where the row is aligned for it.
template <typename T, int E>
__device__ __forceinline__ void load_elems(const T* p, bool vec, float (&x)[E]) {
  if (vec) {
    constexpr int B = E * int(sizeof(T));
    alignas(16) T raw[E];
    if constexpr (B == 4) *reinterpret_cast<uint32_t*>(raw) = __ldcs(reinterpret_cast<const unsigned int*>(p));
    else if constexpr (B == 8) *reinterpret_cast<uint2*>(raw) = __ldcs(reinterpret_cast<const uint2*>(p));
    else {
#pragma unroll
      for (int i = 0; i < B / 16; ++i)
        reinterpret_cast<uint4*>(raw)[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = float(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = float(p[e]);
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

// One CTA per row. A head's elements lie eight to a lane on D / 8 lanes, so that a warp takes 32 / (D
// / 8) heads at a time (a step); it takes every kRowWarps-th step, U at a time so that their loads
// are in flight together, the first of them while the row's place is looked up. RoPE by halves
// finds the partner of an element half a head's lanes away, interleaved RoPE within the lane; the
// row's cosines and sines are loaded once for all of a warp's heads. Every lane takes part in the
// shuffles, whatever its head is (a step may hold heads of two kinds). Arithmetic of the rotation:
// each product rounded, then the difference or sum (ops.rs:77-95).
// Bound by memory, next by instructions: with four elements a lane, a head to a warp, 10 thousand
// rows of 32/8 heads of 128 (bf16 rows, 8-bit pages, 231 MB) took 77 us.
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32)
    paged_write_kernel(const __grid_constant__ PagedWriteArgs a) {
  constexpr int E = 8, LH = D / E, HW = 32 / LH;  // lanes of a head, heads of a step
  constexpr int U = D == 256 ? 4 : 3;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % LH;
  const int r = blockIdx.x;
  const int kvh = a.pool.kv_heads;
  const int units = a.heads + 2 * kvh;
  float xs[U][E];
  auto skipped = [&](int u) { return u >= units || (u < a.heads && a.q_out == nullptr); };
  auto load = [&](int u0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = u0 + i * (kRowWarps * HW) + lane / LH;
#pragma unroll
      for (int e = 0; e < E; ++e) xs[i][e] = 0.0f;
      if (skipped(u)) continue;
      const T* p;
      if (u < a.heads)
        p = static_cast<const T*>(a.q) + int64_t(r) * a.q_stride + int64_t(u) * D;
      else if (u < a.heads + kvh)
        p = static_cast<const T*>(a.k) + int64_t(r) * a.k_stride + int64_t(u - a.heads) * a.k_head_stride;
      else
        p = static_cast<const T*>(a.v) + int64_t(r) * a.v_stride +
            int64_t(u - a.heads - kvh) * a.v_head_stride;
      load_elems<T, E>(p + sub * E, a.vec != 0, xs[i]);
    }
  };
  load(warp * HW);
  float c[E], s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) c[e] = s[e] = 0.0f;
  if (a.rope == 1) {
    const float* cs = a.angles + int64_t(r) * D + (sub % (LH / 2)) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) { c[e] = cs[e]; s[e] = cs[D / 2 + e]; }
  } else if (a.rope == 2) {
    const float* cs = a.angles + int64_t(r) * D + sub * (E / 2);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) { c[e] = cs[e]; s[e] = cs[D / 2 + e]; }
  }
  int page, slot;
  if (!place_of(a.spans, a.pool, r, lane, &page, &slot, a.err)) return;  // the warp's, as one
  for (int u0 = warp * HW; u0 < units; u0 += U * kRowWarps * HW) {
    if (u0 != warp * HW) load(u0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int step = u0 + i * (kRowWarps * HW);  // the step's first head
      if (step >= units) break;
      const int u = step + lane / LH;
      const bool skip = skipped(u);
      const bool is_query = u < a.heads, is_key = !is_query && u < a.heads + kvh;
      float(&x)[E] = xs[i];
      if (step < a.heads + kvh) {  // (some head of the step is turned)
        const float* weight = is_query ? a.q_norm : is_key ? a.k_norm : nullptr;
        if (a.q_norm != nullptr || a.k_norm != nullptr) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int off = LH / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
          if (weight != nullptr) {
            const float inverse = 1.0f / sqrtf(ss / float(D) + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], inverse), weight[sub * E + e]);
          }
        }
        if (a.rope == 1) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float o = __shfl_xor_sync(0xffffffffu, x[e], LH / 2);
            const float xc = __fmul_rn(x[e], c[e]), os = __fmul_rn(o, s[e]);
            if (is_query || is_key) x[e] = sub < LH / 2 ? __fsub_rn(xc, os) : __fadd_rn(xc, os);
          }
        } else if (a.rope == 2 && (is_query || is_key)) {
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            const float y0 = x[2 * e], y1 = x[2 * e + 1];
            x[2 * e] = __fsub_rn(__fmul_rn(y0, c[e]), __fmul_rn(y1, s[e]));
            x[2 * e + 1] = __fadd_rn(__fmul_rn(y1, c[e]), __fmul_rn(y0, s[e]));
          }
        }
      }
      if (is_query && !skip)
        store_elems<E>(a.q_out, int64_t(r) * a.q_out_stride + int64_t(u) * D + sub * E,
                       a.q_out_bf16 != 0, a.q_out_vec != 0, x);
      if (step + HW <= a.heads) continue;  // all of the step's heads are queries
      const int kv = is_key ? u - a.heads : u - a.heads - kvh;
      const int64_t row = ((int64_t(page) * kvh + kv) << a.pool.page_shift) + slot;
      unsigned char* base = is_key ? a.pool.keys : a.pool.values;
      if (!a.pool.q8) {
        if (!is_query && !skip) store_elems<E>(base, row * D + sub * E, true, true, x);
        continue;
      }
      float top = 0.0f, total = 0.0f;  // (total: NaN if an element is not finite)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        top = fmaxf(top, fabsf(x[e]));
        total = fmaf(x[e], 0.0f, total);
      }
#pragma unroll
      for (int off = LH / 2; off >= 1; off >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        total += __shfl_xor_sync(0xffffffffu, total, off);
      }
      const bool finite = total == 0.0f;
      const bool live = finite && top >= 7.888609052e-31f;  // 2^-100
      const float inverse = live ? __fdiv_rn(127.0f, top) : 0.0f;
      const float scale = !finite ? __int_as_float(0x7fffffff) : live ? __fdiv_rn(top, 127.0f) : 0.0f;
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = finite ? __fmul_rn(x[e], inverse) : 0.0f;  // within +-127 but for a rounding
        w[e / 4] |= uint32_t(max(-127, min(127, __float2int_rn(y))) & 0xff) << (8 * (e % 4));
      }
      if (is_query || skip) continue;
      *reinterpret_cast<uint2*>(base + row * D + sub * E) = make_uint2(w[0], w[1]);
      if (sub == 0) (is_key ? a.pool.key_scales : a.pool.value_scales)[row] = scale;
    }
  }
}

// A warp takes two rows: their places, then 16 bytes of them a lane at a time, eight such loads in
// flight (two vectors of keys and of values of each row). Bound by memory.
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
    const bool ok = r < a.spans.rows && place_of(a.spans, a.pool, r, lane, &page, &slot, a.err);
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
  auto go = [&](void (*k)(PagedWriteArgs)) {
    return launch(k, a.spans.rows, kRowWarps * 32, a, stream);
  };
  if (a.in_bf16) {
    if (d == 64) return go(paged_write_kernel<__nv_bfloat16, 64>);
    if (d == 128) return go(paged_write_kernel<__nv_bfloat16, 128>);
    if (d == 256) return go(paged_write_kernel<__nv_bfloat16, 256>);
  } else {
    if (d == 64) return go(paged_write_kernel<float, 64>);
    if (d == 128) return go(paged_write_kernel<float, 128>);
    if (d == 256) return go(paged_write_kernel<float, 256>);
  }
  return cudaErrorInvalidValue;
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

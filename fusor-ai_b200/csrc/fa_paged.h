// The paged cache's kernels as the C ABI sees them (plain data), and the checks of a batch's
// spans that host and device share.
//
// Pages of `page_size` positions (a power of two, so that a position splits into page and slot
// by shifts, and at least 16, so that 16 consecutive positions from a multiple of 16 lie in one
// page) hold every KV head's rows: [layer][page][KV head][slot][head_dim]. 8-bit pages hold
// integers in -127..127 and one f32 scale per (position, KV head): [layer][page][KV head][slot].
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __CUDACC__
#define FA_HD __host__ __device__ __forceinline__
#else
#define FA_HD inline
#endif

namespace fa {

constexpr int kMaxPagedSequences = 1024;
constexpr int kMinPageSize = 16, kMaxPageSize = 4096;

// Bits of the device error word (beside kErrTimeout): a span or a page id out of range.
constexpr unsigned kErrPagedSpan = 2u;
constexpr unsigned kErrPagedPage = 4u;

// One layer of a paged cache.
struct PagedPool {
  unsigned char* keys;    // this layer's pages
  unsigned char* values;
  float* key_scales;      // 8-bit pages: this layer's scales
  float* value_scales;
  int pages, page_shift, kv_heads, head_dim;
  int q8;                 // 8-bit pages (else bf16)
};

// A ragged batch: sequence s's rows are row_starts[s] .. row_starts[s + 1] of the call's arrays,
// at consecutive positions from firsts[s]; its position p lies in page tables[s * table_stride +
// p / page_size].
struct PagedSpans {
  int sequences, rows, max_rows, table_width;
  int64_t table_stride;
  const int* row_starts;
  const int* firsts;
  const int* tables;
};

struct PagedSpan {
  int row0, n, first;
};

// The span of rows r0 .. r1 from position `first` on, or false if it is out of range: rows that are
// not within the call's or run backwards, more rows than max_rows, a negative position or positions
// past its table. Nothing of such a sequence is read or written.
FA_HD bool paged_span_of(const PagedSpans& b, int page_shift, int r0, int r1, int first,
                         PagedSpan* out) {
  out->row0 = r0;
  out->n = 0;
  out->first = first;
  if (r0 < 0 || r1 < r0 || r1 > b.rows || r1 - r0 > b.max_rows || first < 0) return false;
  if (int64_t(first) + (r1 - r0) > (int64_t(b.table_width) << page_shift)) return false;
  if (int64_t(first) + (r1 - r0) > 0x7fffff00) return false;  // positions stay 32-bit integers
  out->n = r1 - r0;
  return true;
}

// Sequence s's span.
FA_HD bool paged_span(const PagedSpans& b, int page_shift, int s, PagedSpan* out) {
  return paged_span_of(b, page_shift, b.row_starts[s], b.row_starts[s + 1], b.firsts[s], out);
}

// Whether a page id names a page of the pool.
FA_HD bool paged_page_ok(int page, int pages) { return page >= 0 && page < pages; }

// The keys a query at `position` sees, [lo, hi), in a sequence of `end` positions (Mask::keys,
// transformer.rs:116-128, the masks of one run): causal, window or full.
FA_HD void paged_keys(int kind, int window, int position, int end, int* lo, int* hi) {
  *hi = kind == 2 ? end : position + 1;
  *lo = kind == 1 && position + 1 > window ? position + 1 - window : 0;
}

// Rows written into pages: the attention input (queries rotated into q_out, keys rotated and
// values kept), or plain key and value rows (heads = 0).
struct PagedWriteArgs {
  PagedPool pool;
  PagedSpans spans;
  int heads;             // query heads (0: none)
  int rope;              // 0 none, 1 by halves, 2 interleaved
  int in_bf16;           // element type of q, k, v (and of q_out)
  int q_out_bf16;
  const void* q;         // row r, head h at q + r * q_stride + h * head_dim
  const void* k;         // row r, head h at k + r * k_stride + h * k_head_stride
  const void* v;
  int64_t q_stride, k_stride, k_head_stride, v_stride, v_head_stride;
  int vec;               // every head's row starts on a 16-byte boundary
  const float* angles;   // row r at angles + r * head_dim: cosines then sines
  int angles_vec;        // 16-byte aligned
  const float* q_norm;
  const float* k_norm;
  float eps;
  void* q_out;           // row r, head h at q_out + r * q_out_stride + h * head_dim (or null)
  int64_t q_out_stride;
  int q_out_vec;
  unsigned* err;
};
cudaError_t launch_paged_write(const PagedWriteArgs& args, cudaStream_t stream);

// Rows of pages read back: row r, head h to out + r * stride + h * head_stride.
struct PagedReadArgs {
  PagedPool pool;
  PagedSpans spans;
  int out_bf16;
  int vec;  // 16-byte aligned rows
  void* k;
  void* v;
  int64_t k_stride, k_head_stride, v_stride, v_head_stride;
  unsigned* err;
};
cudaError_t launch_paged_read(const PagedReadArgs& args, cudaStream_t stream);

// Attention over the pages. Sequences of few packed rows (rows x query heads of a KV head) run
// on the token kernel (fa_paged_tokens.cuh), the others on the chunk kernel (fa_paged_chunk.cuh);
// each skips the other's. The token kernel takes what fits its two products of 8 columns. Measured
// on both sides (64 sequences of 512 to 8192 positions, token kernel against chunk kernel, us):
// 32/8 heads of 128, 1 / 2 / 4 rows: 119 / 122 / 201 against 470 over 8-bit pages, 166 / 171 / 209
// against 348 over bf16 ones; 14/2 heads of 64, 2 rows: 51 against 105 and 43 against 87; 8/2 heads
// of 256, 2 / 4 rows: 76 / 161 against 236 and 109 / 162 against 158 (the one tie). Five rows of 32/8
// heads, past its columns, take the chunk kernel's 474 and 350.
constexpr int kPagedTokenCols = 16;

struct PagedAttendArgs {
  PagedPool pool;
  PagedSpans spans;
  int heads, group;      // query heads; query heads of a KV head
  int kind, window;      // mask: 0 causal, 1 window, 2 full
  int token_cols;        // packed rows up to which a sequence runs on the token kernel
  int merge_cols;        // token kernel: the most packed rows that a sequence of it can have
  int tile_rows;         // rows of a chunk's query tile: 128 / group
  int q_bf16, out_bf16, out_vec;
  const void* q;         // row r, head h at q + r * q_stride + h * head_dim; 16-byte aligned rows
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  float scale_log2;      // log2(e) / sqrt(head_dim)
  float* part_o;         // split units' partials: two slots for each CTA
  float* part_ml;
  int* counters;         // one per CTA, zero between launches
  unsigned* err;
};

// Partial floats (outputs, then max and sum pairs) and counters that a launch needs at most.
void paged_tokens_workspace(int head_dim, int sms, int64_t* o_floats, int64_t* ml_floats,
                            int* counters);
cudaError_t launch_paged_tokens(const PagedAttendArgs& args, int sms, cudaStream_t stream);

void paged_chunk_workspace(int head_dim, int sms, int64_t* o_floats, int64_t* ml_floats,
                           int* counters);
cudaError_t launch_paged_chunk(const PagedAttendArgs& args, int sms, cudaStream_t stream);

}  // namespace fa

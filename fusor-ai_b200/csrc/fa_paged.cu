// The C ABI's paged cache (include/fa_attn.h): argument checks, the workspace's layout and the
// launches. The batch's numbers stay in device memory; the host picks kernels by max_rows alone.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <new>
#include <vector>

#include "fa_attn.h"
#include "fa_host.h"
#include "fa_launch.cuh"
#include "fa_paged.h"

namespace {

using fa::host::cuda_fail;
using fa::host::fail;

#define FA_TRY(call)              \
  do {                            \
    if (int rc_ = (call)) return rc_; \
  } while (0)

// Restores the caller's current device on scope exit.
struct OnDevice {
  int prev = -1;
  explicit OnDevice(int device) {
    if (cudaGetDevice(&prev) == cudaSuccess && prev != device) cudaSetDevice(device);
    else prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_shape(const fa_paged_cache* c) {
  if (c == nullptr) return fail(FA_ERR_ARG, "null paged cache");
  if (c->layers < 1 || c->heads < 1 || c->kv_heads < 1 || c->pages < 1)
    return fail(FA_ERR_ARG, "%d layers, %d heads, %d KV heads, %d pages", c->layers, c->heads,
                c->kv_heads, c->pages);
  if (c->heads % c->kv_heads)
    return fail(FA_ERR_SHAPE, "%d heads over %d KV heads", c->heads, c->kv_heads);
  if (c->heads / c->kv_heads > 128)
    return fail(FA_ERR_UNSUPPORTED, "%d query heads to a KV head; at most 128", c->heads / c->kv_heads);
  if (c->kv_heads > 1024) return fail(FA_ERR_UNSUPPORTED, "%d KV heads; at most 1024", c->kv_heads);
  if (c->dtype == FA_F32) return fail(FA_ERR_UNSUPPORTED, "pages of f32: bf16 and 8-bit pages here");
  if (c->dtype != FA_BF16 && c->dtype != FA_Q8) return fail(FA_ERR_ARG, "page dtype %d", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(FA_ERR_UNSUPPORTED, "pages of head_dim %d: 64, 128 and 256 here", c->head_dim);
  if (c->page_size < fa::kMinPageSize || c->page_size > fa::kMaxPageSize ||
      (c->page_size & (c->page_size - 1)))
    return fail(FA_ERR_ARG, "page_size %d: a power of two from %d to %d", c->page_size,
                fa::kMinPageSize, fa::kMaxPageSize);
  return FA_OK;
}

int page_shift(const fa_paged_cache* c) {
  int s = 0;
  while ((1 << s) < c->page_size) ++s;
  return s;
}

int check_spans(const fa_paged_batch* b) {
  if (b == nullptr) return fail(FA_ERR_ARG, "null batch");
  if (b->sequences < 0 || b->rows < 0 || b->max_rows < 0 || b->table_width < 0)
    return fail(FA_ERR_ARG, "a negative count: %d sequences, %d rows, max_rows %d, table_width %d",
                b->sequences, b->rows, b->max_rows, b->table_width);
  if (b->rows > (1 << 28)) return fail(FA_ERR_ARG, "%d rows; at most %d", b->rows, 1 << 28);
  if (b->sequences > fa::kMaxPagedSequences)
    return fail(FA_ERR_ARG, "%d sequences; at most %d", b->sequences, fa::kMaxPagedSequences);
  if (b->table_stride < b->table_width)
    return fail(FA_ERR_ARG, "table_stride %lld for tables of %d pages", (long long)b->table_stride,
                b->table_width);
  if (b->sequences > 0 && (b->row_starts == nullptr || b->firsts == nullptr || b->tables == nullptr))
    return fail(FA_ERR_ARG, "null row_starts, firsts or tables");
  return FA_OK;
}

int check_mask(const fa_paged_batch* b) {
  if (b->mask == FA_MASK_GROUPS) return fail(FA_ERR_UNSUPPORTED, "a Groups mask over pages");
  if (b->mask != FA_MASK_CAUSAL && b->mask != FA_MASK_WINDOW && b->mask != FA_MASK_FULL)
    return fail(FA_ERR_ARG, "mask kind %d", b->mask);
  if (b->mask == FA_MASK_WINDOW && b->window < 1) return fail(FA_ERR_ARG, "window %d", b->window);
  return FA_OK;
}

int check_rows_dtype(int dtype, const char* what) {
  if (dtype != FA_F32 && dtype != FA_BF16) return fail(FA_ERR_ARG, "%s dtype %d", what, dtype);
  return FA_OK;
}

// What every device call checks: the cache's shape and arrays, the layer, the batch.
int check_call(const fa_paged_cache* c, int layer, const fa_paged_batch* b) {
  FA_TRY(check_shape(c));
  if (layer < 0 || layer >= c->layers)
    return fail(FA_ERR_SHAPE, "layer %d of a %d-layer cache", layer, c->layers);
  if (c->keys == nullptr || c->values == nullptr) return fail(FA_ERR_ARG, "null pages");
  if (c->dtype == FA_Q8 && (c->key_scales == nullptr || c->value_scales == nullptr))
    return fail(FA_ERR_ARG, "8-bit pages without scales");
  if (!aligned(c->keys, 16) || !aligned(c->values, 16))
    return fail(FA_ERR_ARG, "pages must start on 16-byte boundaries");
  if (!aligned(c->key_scales, 4) || !aligned(c->value_scales, 4))
    return fail(FA_ERR_ARG, "scales must start on 4-byte boundaries");
  FA_TRY(check_spans(b));
  if (!aligned(b->row_starts, 4) || !aligned(b->firsts, 4) || !aligned(b->tables, 4))
    return fail(FA_ERR_ARG, "row_starts, firsts and tables must start on 4-byte boundaries");
  return FA_OK;
}

int check_pointers(const fa_paged_cache* c, const fa_paged_batch* b) {
  const int dev = c->device;
  FA_TRY(fa::host::pointer_on(c->keys, dev, "keys"));
  FA_TRY(fa::host::pointer_on(c->values, dev, "values"));
  FA_TRY(fa::host::pointer_on(c->dtype == FA_Q8 ? c->key_scales : nullptr, dev, "key_scales"));
  FA_TRY(fa::host::pointer_on(c->dtype == FA_Q8 ? c->value_scales : nullptr, dev, "value_scales"));
  FA_TRY(fa::host::pointer_on(b->row_starts, dev, "row_starts"));
  FA_TRY(fa::host::pointer_on(b->firsts, dev, "firsts"));
  FA_TRY(fa::host::pointer_on(b->tables, dev, "tables"));
  return FA_OK;
}

fa::PagedPool pool_of(const fa_paged_cache* c, int layer) {
  fa::PagedPool p{};
  const int64_t rows = int64_t(c->pages) * c->kv_heads * c->page_size;  // of a layer
  const int64_t bytes = rows * c->head_dim * (c->dtype == FA_Q8 ? 1 : 2);
  p.keys = static_cast<unsigned char*>(c->keys) + layer * bytes;
  p.values = static_cast<unsigned char*>(c->values) + layer * bytes;
  if (c->dtype == FA_Q8) {
    p.key_scales = c->key_scales + layer * rows;
    p.value_scales = c->value_scales + layer * rows;
  }
  p.pages = c->pages;
  p.page_shift = page_shift(c);
  p.kv_heads = c->kv_heads;
  p.head_dim = c->head_dim;
  p.q8 = c->dtype == FA_Q8;
  return p;
}

fa::PagedSpans spans_of(const fa_paged_batch* b) {
  return {b->sequences, b->rows, b->max_rows, b->table_width, b->table_stride,
          b->row_starts, b->firsts, b->tables};
}

// Whether rows `strides` elements apart (all of them) can be read `bytes` at a time.
bool vectors(const void* p, std::initializer_list<int64_t> strides, int elem, int bytes) {
  if (!aligned(p, bytes)) return false;
  for (int64_t s : strides)
    if ((s * elem) % bytes) return false;
  return true;
}

// ---- the workspace: counters (zeroed by the caller), partials, then a call's queries ------------

struct Workspace {
  int64_t ml_at, o_at, q_at, bytes;
  int chunk_counters;  // index of the chunk kernel's first counter
};

Workspace workspace_of(const fa_paged_cache* c, int rows, int max_rows, int sms) {
  int64_t o = 0, ml = 0;
  int counters = 0;
  fa::paged_tokens_workspace(c->head_dim, sms, &o, &ml, &counters);
  Workspace w{};
  w.chunk_counters = counters;
  if (int64_t(max_rows) * (c->heads / c->kv_heads) > fa::kPagedTokenCols) {
    int64_t o2 = 0, ml2 = 0;
    int n2 = 0;
    fa::paged_chunk_workspace(c->head_dim, sms, &o2, &ml2, &n2);
    o = std::max(o, o2);
    ml = std::max(ml, ml2);
  }
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  w.ml_at = FA_PAGED_COUNTER_BYTES;
  w.o_at = w.ml_at + up(ml * 4);
  w.q_at = w.o_at + up(o * 4);
  w.bytes = w.q_at + up(int64_t(rows) * c->heads * c->head_dim * 4);
  return w;
}

int check_workspace(const fa_paged_cache* c, const fa_paged_batch* b, int sms, Workspace* w) {
  *w = workspace_of(c, b->rows, b->max_rows, sms);
  if (b->workspace == nullptr) return fail(FA_ERR_ARG, "null workspace");
  if (!aligned(b->workspace, 256)) return fail(FA_ERR_ARG, "the workspace must start on a 256-byte boundary");
  if (int64_t(b->workspace_bytes) < w->bytes)
    return fail(FA_ERR_ARG, "a workspace of %llu bytes; %lld are needed",
                (unsigned long long)b->workspace_bytes, (long long)w->bytes);
  return FA_OK;
}

int check_attend(const fa_paged_cache* c, const fa_paged_batch* b, const void* out,
                 int64_t out_stride, int out_dtype) {
  FA_TRY(check_mask(b));
  FA_TRY(check_rows_dtype(out_dtype, "out"));
  if (b->rows > 0 && out == nullptr) return fail(FA_ERR_ARG, "null out");
  if (out_stride < int64_t(c->heads) * c->head_dim)
    return fail(FA_ERR_SHAPE, "out rows %lld apart for %d heads of %d", (long long)out_stride,
                c->heads, c->head_dim);
  if (!aligned(out, out_dtype == FA_BF16 ? 2 : 4)) return fail(FA_ERR_ARG, "a misaligned out");
  return FA_OK;
}

int check_input(const fa_paged_cache* c, const fa_paged_batch* b, int rope, const float* angles,
                const fa_head_norm* norm, const void* qkv, int64_t qkv_stride, int dtype) {
  if (rope < FA_ROPE_NONE || rope > FA_ROPE_INTERLEAVED) return fail(FA_ERR_ARG, "rope %d", rope);
  if (rope != FA_ROPE_NONE && b->rows > 0 && angles == nullptr)
    return fail(FA_ERR_ARG, "RoPE without angles");
  FA_TRY(check_rows_dtype(dtype, "qkv"));
  if (b->rows > 0 && qkv == nullptr) return fail(FA_ERR_ARG, "null qkv");
  if (qkv_stride < int64_t(c->heads + 2 * c->kv_heads) * c->head_dim)
    return fail(FA_ERR_SHAPE, "qkv rows %lld apart for %d + 2 x %d heads of %d",
                (long long)qkv_stride, c->heads, c->kv_heads, c->head_dim);
  if (!aligned(qkv, dtype == FA_BF16 ? 2 : 4) || !aligned(angles, 4) ||
      (norm && (!aligned(norm->q_norm, 4) || !aligned(norm->k_norm, 4))))
    return fail(FA_ERR_ARG, "misaligned qkv, angles or norms");
  return FA_OK;
}

int check_input_pointers(const fa_paged_cache* c, const float* angles, const fa_head_norm* norm,
                         const void* qkv) {
  FA_TRY(fa::host::pointer_on(qkv, c->device, "qkv"));
  FA_TRY(fa::host::pointer_on(angles, c->device, "angles"));
  if (norm) {
    FA_TRY(fa::host::pointer_on(norm->q_norm, c->device, "q_norm"));
    FA_TRY(fa::host::pointer_on(norm->k_norm, c->device, "k_norm"));
  }
  return FA_OK;
}

int write_input(const fa_paged_cache* c, int layer, const fa_paged_batch* b, int rope,
                const float* angles, const fa_head_norm* norm, const void* qkv, int64_t qkv_stride,
                int dtype, void* q_out, int64_t q_out_stride, int q_out_dtype, unsigned* err,
                cudaStream_t s) {
  fa::PagedWriteArgs a{};
  const int e = dtype == FA_BF16 ? 2 : 4, d = c->head_dim;
  a.pool = pool_of(c, layer);
  a.spans = spans_of(b);
  a.heads = c->heads;
  a.rope = rope;
  a.in_bf16 = dtype == FA_BF16;
  a.q_out_bf16 = q_out_dtype == FA_BF16;
  const unsigned char* base = static_cast<const unsigned char*>(qkv);
  a.q = base;
  a.k = base + int64_t(c->heads) * d * e;
  a.v = base + int64_t(c->heads + c->kv_heads) * d * e;
  a.q_stride = a.k_stride = a.v_stride = qkv_stride;
  a.k_head_stride = a.v_head_stride = d;
  a.vec = vectors(qkv, {qkv_stride}, e, 16);
  a.angles = angles;
  a.angles_vec = aligned(angles, 16);
  a.q_norm = norm ? norm->q_norm : nullptr;
  a.k_norm = norm ? norm->k_norm : nullptr;
  a.eps = norm ? norm->eps : 0.0f;
  a.q_out = q_out;
  a.q_out_stride = q_out_stride;
  const int oe = q_out_dtype == FA_BF16 ? 2 : 4;
  a.q_out_vec = vectors(q_out, {q_out_stride}, oe, 16);
  a.err = err;
  const cudaError_t rc = fa::launch_paged_write(a, s);
  if (rc != cudaSuccess) return cuda_fail(rc, "paged write launch");
  return FA_OK;
}

int attend(const fa_paged_cache* c, int layer, const fa_paged_batch* b, const void* q,
           int64_t q_stride, int dtype, void* out, int64_t out_stride, int out_dtype,
           const Workspace& w, int sms, unsigned* err, cudaStream_t s) {
  // (max_rows 0 is a call like any other: the token kernel reports the sequences that have rows)
  if (b->sequences == 0 || b->rows == 0) return FA_OK;
  fa::PagedAttendArgs a{};
  a.pool = pool_of(c, layer);
  a.spans = spans_of(b);
  a.heads = c->heads;
  a.group = c->heads / c->kv_heads;
  a.tile_rows = 128 / a.group;
  a.kind = b->mask;
  a.window = b->window;
  a.token_cols = fa::kPagedTokenCols;
  a.q_bf16 = dtype == FA_BF16;
  a.out_bf16 = out_dtype == FA_BF16;
  a.out_vec = vectors(out, {out_stride}, a.out_bf16 ? 2 : 4, 16);
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.scale_log2 = float((1.0 / std::sqrt(double(c->head_dim))) * 1.4426950408889634);
  unsigned char* base = static_cast<unsigned char*>(b->workspace);
  a.part_ml = reinterpret_cast<float*>(base + w.ml_at);
  a.part_o = reinterpret_cast<float*>(base + w.o_at);
  a.counters = reinterpret_cast<int*>(base);
  a.err = err;
  if (!vectors(q, {q_stride}, a.q_bf16 ? 2 : 4, 16)) {
    // rows that 16-byte loads do not fit are copied (in f32, exactly) to where they do
    float* rows = reinterpret_cast<float*>(base + w.q_at);
    const cudaError_t rc = fa::launch_prepare_queries(dtype == FA_BF16 ? fa::kKtBf16 : fa::kKtF32, q, q_stride,
                                                      0, b->rows, c->heads, c->head_dim, 1.0f, rows, s);
    if (rc != cudaSuccess) return cuda_fail(rc, "query copy launch");
    a.q = rows;
    a.q_stride = int64_t(c->heads) * c->head_dim;
    a.q_bf16 = 0;
  }
  // A batch may hold both kinds of sequences: each kernel leaves the other's alone. Where the
  // rows are as many as sequences of max_rows each make (a uniform batch, a single sequence) the
  // chunk kernel takes every sequence, and where no sequence has many rows the token kernel does:
  // one launch. (The host knows no more of the rows: among chunks of unequal lengths the token kernel
  // finds nothing to do, and padding rows that make up the product send single tokens to the chunk
  // kernel, which is slower and as right.)
  const bool chunks = int64_t(b->max_rows) * a.group > a.token_cols;
  const bool tokens = !chunks || (a.group <= a.token_cols &&
                                  b->rows < int64_t(b->sequences) * b->max_rows);
  if (chunks) {
    fa::PagedAttendArgs ca = a;
    ca.counters += w.chunk_counters;
    // Beside the chunk kernel the token kernel takes sequences of one 8-column product alone (its
    // 16-column form holds twice the accumulators and two CTAs an SM, not three: 59 against 37 us
    // for 24 single tokens of 2000 positions each), where a token fits in it.
    if (!tokens) ca.token_cols = 0;
    else if (a.group <= 8) ca.token_cols = a.token_cols = 8;
    const cudaError_t rc = fa::launch_paged_chunk(ca, sms, s);
    if (rc != cudaSuccess) return cuda_fail(rc, "paged chunk launch");
  }
  if (tokens) {
    const cudaError_t rc = fa::launch_paged_tokens(a, sms, s);
    if (rc != cudaSuccess) return cuda_fail(rc, "paged tokens launch");
  }
  return FA_OK;
}

}  // namespace

extern "C" {

int fa_paged_workspace_bytes(const fa_paged_cache* cache, int32_t rows, int32_t max_rows,
                             uint64_t* bytes) {
  FA_TRY(check_shape(cache));
  if (rows < 0 || rows > (1 << 28) || max_rows < 0 || bytes == nullptr) return fail(FA_ERR_ARG, "bad rows or null bytes");
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  *bytes = uint64_t(workspace_of(cache, rows, max_rows, sms).bytes);
  return FA_OK;
}

int fa_paged_check(const fa_paged_cache* cache, const fa_paged_batch* batch) {
  FA_TRY(check_shape(cache));
  FA_TRY(check_spans(batch));
  const int shift = page_shift(cache);
  const fa::PagedSpans b = spans_of(batch);
  std::vector<int64_t> written;  // (page, slot) of every row
  try {
    for (int s = 0; s < b.sequences; ++s) {
      fa::PagedSpan sp;
      if (!fa::paged_span(b, shift, s, &sp)) {
        const int64_t end = int64_t(sp.first) + b.row_starts[s + 1] - sp.row0;
        if (sp.first >= 0 && sp.row0 >= 0 && b.row_starts[s + 1] >= sp.row0 &&
            b.row_starts[s + 1] <= b.rows && b.row_starts[s + 1] - sp.row0 <= b.max_rows)
          return fail(FA_ERR_CAPACITY,
                      "the pages hold every key the span sees: sequence %d ends at %lld > %lld", s,
                      (long long)end, (long long)b.table_width << shift);
        return fail(FA_ERR_ARG, "sequence %d: rows %d..%d of %d (max_rows %d) at position %d", s,
                    sp.row0, b.row_starts[s + 1], b.rows, b.max_rows, sp.first);
      }
      if (sp.n == 0) continue;
      const int* table = b.tables + int64_t(s) * b.table_stride;
      const int64_t end = int64_t(sp.first) + sp.n;
      for (int64_t p = 0; p < (end + cache->page_size - 1) >> shift; ++p)
        if (!fa::paged_page_ok(table[p], cache->pages))
          return fail(FA_ERR_ARG, "sequence %d: page %d of a pool of %d", s, table[p], cache->pages);
      for (int64_t pos = sp.first; pos < end; ++pos)
        written.push_back((int64_t(table[pos >> shift]) << shift) + (pos & (cache->page_size - 1)));
    }
    std::sort(written.begin(), written.end());
  } catch (const std::bad_alloc&) {
    return fail(FA_ERR_ARG, "no host memory to check %d rows", b.rows);
  }
  if (std::adjacent_find(written.begin(), written.end()) != written.end())
    return fail(FA_ERR_ARG, "two rows of the call lie in one slot");
  return FA_OK;
}

int fa_attention_input_paged(const fa_paged_cache* cache, int32_t layer,
                             const fa_paged_batch* batch, int32_t rope, const float* angles,
                             const fa_head_norm* norm, const void* qkv, int64_t qkv_stride,
                             int32_t dtype, void* q_out, int64_t q_out_stride, void* stream) {
  FA_TRY(check_call(cache, layer, batch));
  FA_TRY(check_input(cache, batch, rope, angles, norm, qkv, qkv_stride, dtype));
  if (q_out != nullptr && q_out_stride < int64_t(cache->heads) * cache->head_dim)
    return fail(FA_ERR_SHAPE, "q_out rows %lld apart for %d heads of %d", (long long)q_out_stride,
                cache->heads, cache->head_dim);
  if (!aligned(q_out, dtype == FA_BF16 ? 2 : 4)) return fail(FA_ERR_ARG, "a misaligned q_out");
  FA_TRY(check_pointers(cache, batch));
  FA_TRY(check_input_pointers(cache, angles, norm, qkv));
  FA_TRY(fa::host::pointer_on(q_out, cache->device, "q_out"));
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  if (batch->sequences == 0 || batch->rows == 0) return FA_OK;
  OnDevice on(cache->device);
  return write_input(cache, layer, batch, rope, angles, norm, qkv, qkv_stride, dtype, q_out,
                     q_out_stride, dtype, err, static_cast<cudaStream_t>(stream));
}

namespace {

// Whether a head row of `d` elements at row * row_stride + head * head_stride shares elements with
// another of the set, or with one of the same set `delta` elements on: whether delta + i row_stride +
// j head_stride, |i| < rows, |j| < heads, comes within d of 0 (with delta 0, but for i = j = 0).
bool head_rows_overlap(int64_t delta, int rows, int heads, int64_t row_stride, int64_t head_stride, int d) {
  if (rows == 1) row_stride = 0;
  if (delta == 0 && ((heads == 1 || head_stride >= d) &&
                     (rows == 1 || row_stride >= (heads - 1) * head_stride + d)))
    return false;  // (heads within rows: no need to look)
  for (int64_t j = 1 - heads; j < heads; ++j) {
    const int64_t x = delta + j * head_stride;
    const int64_t near = row_stride == 0 ? 0 : -x / row_stride;  // (to within one)
    for (int64_t n = near - 1; n <= near + 1; ++n) {
      const int64_t i = std::min<int64_t>(std::max<int64_t>(n, 1 - rows), rows - 1);
      if ((delta != 0 || i != 0 || j != 0) && std::abs(x + i * row_stride) < d) return true;
    }
  }
  return false;
}

// The rows that a read writes: no element from two of them. (keys and values may be one array, which
// then holds the values: a thread stores its values after its keys.)
int check_rows_out(const fa_paged_cache* c, const fa_paged_batch* b, const fa_paged_rows* r) {
  if (b->rows == 0) return FA_OK;
  const int64_t most = int64_t(1) << 34;  // (keeps what follows within 64 bits)
  const int64_t rs = b->rows > 1 ? r->row_stride : 0, hs = c->kv_heads > 1 ? r->head_stride : 0;
  if (rs > most || hs > most) return fail(FA_ERR_ARG, "strides of %lld and %lld elements", (long long)rs, (long long)hs);
  const int d = c->head_dim, e = r->dtype == FA_BF16 ? 2 : 4;
  if (head_rows_overlap(0, b->rows, c->kv_heads, rs, hs, d))
    return fail(FA_ERR_ARG, "rows %lld apart with heads %lld apart overlap", (long long)rs, (long long)hs);
  const int64_t apart = (reinterpret_cast<intptr_t>(r->values) - reinterpret_cast<intptr_t>(r->keys)) / e;
  if (apart != 0 && std::abs(apart) < (b->rows - 1) * rs + (c->kv_heads - 1) * hs + d &&
      head_rows_overlap(apart, b->rows, c->kv_heads, rs, hs, d))
    return fail(FA_ERR_ARG, "keys and values overlap");
  return FA_OK;
}

int check_rows(const fa_paged_cache* c, const fa_paged_batch* b, const fa_paged_rows* r, bool written) {
  if (r == nullptr) return fail(FA_ERR_ARG, "null rows");
  FA_TRY(check_rows_dtype(r->dtype, "rows"));
  if (b->rows > 0 && (r->keys == nullptr || r->values == nullptr))
    return fail(FA_ERR_ARG, "null keys or values");
  if (r->row_stride < 0 || r->head_stride < 0)
    return fail(FA_ERR_ARG, "negative strides");
  const uintptr_t e = r->dtype == FA_BF16 ? 2 : 4;
  if (!aligned(r->keys, e) || !aligned(r->values, e)) return fail(FA_ERR_ARG, "misaligned rows");
  if (written) FA_TRY(check_rows_out(c, b, r));
  FA_TRY(fa::host::pointer_on(r->keys, c->device, "keys of the rows"));
  FA_TRY(fa::host::pointer_on(r->values, c->device, "values of the rows"));
  return FA_OK;
}

}  // namespace

int fa_paged_write(const fa_paged_cache* cache, int32_t layer, const fa_paged_batch* batch,
                   const fa_paged_rows* rows, void* stream) {
  FA_TRY(check_call(cache, layer, batch));
  FA_TRY(check_rows(cache, batch, rows, false));
  FA_TRY(check_pointers(cache, batch));
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  if (batch->sequences == 0 || batch->rows == 0) return FA_OK;
  OnDevice on(cache->device);
  fa::PagedWriteArgs a{};
  const int e = rows->dtype == FA_BF16 ? 2 : 4;
  a.pool = pool_of(cache, layer);
  a.spans = spans_of(batch);
  a.in_bf16 = rows->dtype == FA_BF16;
  a.k = rows->keys;
  a.v = rows->values;
  a.k_stride = a.v_stride = rows->row_stride;
  a.k_head_stride = a.v_head_stride = rows->head_stride;
  a.vec = vectors(rows->keys, {rows->row_stride, rows->head_stride}, e, 16) &&
          aligned(rows->values, 16);
  a.err = err;
  const cudaError_t rc = fa::launch_paged_write(a, static_cast<cudaStream_t>(stream));
  if (rc != cudaSuccess) return cuda_fail(rc, "paged write launch");
  return FA_OK;
}

int fa_paged_read(const fa_paged_cache* cache, int32_t layer, const fa_paged_batch* batch,
                  const fa_paged_rows* rows, void* stream) {
  FA_TRY(check_call(cache, layer, batch));
  FA_TRY(check_rows(cache, batch, rows, true));
  FA_TRY(check_pointers(cache, batch));
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  if (batch->sequences == 0 || batch->rows == 0) return FA_OK;
  OnDevice on(cache->device);
  fa::PagedReadArgs a{};
  const int e = rows->dtype == FA_BF16 ? 2 : 4;
  a.pool = pool_of(cache, layer);
  a.spans = spans_of(batch);
  a.out_bf16 = rows->dtype == FA_BF16;
  a.vec = vectors(rows->keys, {rows->row_stride, rows->head_stride}, e, 16) &&
          aligned(rows->values, 16);
  a.k = rows->keys;
  a.v = rows->values;
  a.k_stride = a.v_stride = rows->row_stride;
  a.k_head_stride = a.v_head_stride = rows->head_stride;
  a.err = err;
  const cudaError_t rc = fa::launch_paged_read(a, static_cast<cudaStream_t>(stream));
  if (rc != cudaSuccess) return cuda_fail(rc, "paged read launch");
  return FA_OK;
}

int fa_attend_paged(const fa_paged_cache* cache, int32_t layer, const fa_paged_batch* batch,
                    const void* q, int64_t q_stride, int32_t dtype, void* out,
                    int64_t out_stride, int32_t out_dtype, void* stream) {
  FA_TRY(check_call(cache, layer, batch));
  FA_TRY(check_rows_dtype(dtype, "q"));
  if (batch->rows > 0 && q == nullptr) return fail(FA_ERR_ARG, "null q");
  if (q_stride < int64_t(cache->heads) * cache->head_dim)
    return fail(FA_ERR_SHAPE, "q rows %lld apart for %d heads of %d", (long long)q_stride,
                cache->heads, cache->head_dim);
  if (!aligned(q, dtype == FA_BF16 ? 2 : 4)) return fail(FA_ERR_ARG, "a misaligned q");
  FA_TRY(check_attend(cache, batch, out, out_stride, out_dtype));
  FA_TRY(check_pointers(cache, batch));
  FA_TRY(fa::host::pointer_on(q, cache->device, "q"));
  FA_TRY(fa::host::pointer_on(out, cache->device, "out"));
  FA_TRY(fa::host::pointer_on(batch->workspace, cache->device, "workspace"));
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  Workspace w;
  FA_TRY(check_workspace(cache, batch, sms, &w));
  OnDevice on(cache->device);
  return attend(cache, layer, batch, q, q_stride, dtype, out, out_stride, out_dtype, w, sms, err,
                static_cast<cudaStream_t>(stream));
}

int fa_attention_paged(const fa_paged_cache* cache, int32_t layer, const fa_paged_batch* batch,
                       int32_t rope, const float* angles, const fa_head_norm* norm,
                       const void* qkv, int64_t qkv_stride, int32_t dtype, void* out,
                       int64_t out_stride, int32_t out_dtype, void* stream) {
  FA_TRY(check_call(cache, layer, batch));
  FA_TRY(check_input(cache, batch, rope, angles, norm, qkv, qkv_stride, dtype));
  FA_TRY(check_attend(cache, batch, out, out_stride, out_dtype));
  FA_TRY(check_pointers(cache, batch));
  FA_TRY(check_input_pointers(cache, angles, norm, qkv));
  FA_TRY(fa::host::pointer_on(out, cache->device, "out"));
  FA_TRY(fa::host::pointer_on(batch->workspace, cache->device, "workspace"));
  int sms = 0;
  unsigned* err = nullptr;
  FA_TRY(fa::host::device_info(cache->device, &sms, &err));
  Workspace w;
  FA_TRY(check_workspace(cache, batch, sms, &w));
  if (batch->sequences == 0 || batch->rows == 0) return FA_OK;
  OnDevice on(cache->device);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the rotated queries stay f32 over 8-bit pages, whose products round them to no less than f16;
  // over bf16 pages they are kept in bf16, as the tensor cores take them
  void* q = static_cast<unsigned char*>(batch->workspace) + w.q_at;
  const int64_t width = int64_t(cache->heads) * cache->head_dim;
  const int q_dtype = cache->dtype == FA_Q8 ? FA_F32 : FA_BF16;
  FA_TRY(write_input(cache, layer, batch, rope, angles, norm, qkv, qkv_stride, dtype, q, width,
                     q_dtype, err, s));
  return attend(cache, layer, batch, q, width, q_dtype, out, out_stride, out_dtype, w, sms, err, s);
}

}  // extern "C"

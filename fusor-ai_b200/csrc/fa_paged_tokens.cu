// The token kernel's instantiations (fa_paged_tokens.cuh) and its launch.
#include <algorithm>
#include <atomic>

#include "fa_launch.cuh"
#include "fa_paged_tokens.cuh"

namespace fa {

namespace {

template <int D, bool Q8, int NT>
cudaError_t launch_tokens(PagedAttendArgs a, int sms, cudaStream_t stream) {
  using S = TokShape<D, Q8, NT>;
  auto kernel = paged_tokens_kernel<D, Q8, NT>;
  static std::atomic<bool> configured[64];  // per instantiation, per device
  cudaError_t e = smem_limit_once(kernel, S::smem(S::kCols, kMaxPagedSequences), configured);
  if (e != cudaSuccess) return e;
  a.merge_cols = int(std::min<int64_t>(a.token_cols, int64_t(a.spans.max_rows) * a.group));
  const int smem = S::smem(a.merge_cols, a.spans.sequences);
  // the CTAs that an SM holds: 228 KB, of which each takes 1 KB besides its own (and its statics)
  const int fit = std::max(1, std::min(S::kCtas, (228 * 1024) / (smem + 1024 + 128)));
  return launch_pdl(kernel, dim3(unsigned(sms * fit)), dim3(kTokThreads), size_t(smem), stream, a);
}

template <int D>
cudaError_t launch_dim(const PagedAttendArgs& a, int sms, cudaStream_t stream) {
  // 8 columns where no sequence has more: half the products and accumulators
  const bool wide = std::min<int64_t>(int64_t(a.spans.max_rows) * a.group, a.token_cols) > 8;
  if (a.pool.q8)
    return wide ? launch_tokens<D, true, 2>(a, sms, stream) : launch_tokens<D, true, 1>(a, sms, stream);
  return wide ? launch_tokens<D, false, 2>(a, sms, stream) : launch_tokens<D, false, 1>(a, sms, stream);
}

}  // namespace

void paged_tokens_workspace(int head_dim, int sms, int64_t* o_floats, int64_t* ml_floats,
                            int* counters) {
  const int64_t ctas = int64_t(sms) * 3;  // the most that any instantiation runs per SM
  *o_floats = ctas * 2 * kPagedTokenCols * head_dim;
  *ml_floats = ctas * 2 * kPagedTokenCols * 2;
  *counters = int(ctas);
}

cudaError_t launch_paged_tokens(const PagedAttendArgs& a, int sms, cudaStream_t stream) {
  switch (a.pool.head_dim) {
    case 64: return launch_dim<64>(a, sms, stream);
    case 128: return launch_dim<128>(a, sms, stream);
    case 256: return launch_dim<256>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace fa

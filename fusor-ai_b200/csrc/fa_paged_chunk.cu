// The chunk kernel's instantiations (fa_paged_chunk.cuh) and its launch.
#include <atomic>

#include "fa_launch.cuh"
#include "fa_paged_chunk.cuh"

namespace fa {

namespace {

template <int D, bool Q8>
cudaError_t launch_chunk(const PagedAttendArgs& a, int sms, cudaStream_t stream) {
  using S = ChunkShape<D, Q8>;
  auto kernel = paged_chunk_kernel<D, Q8>;
  static std::atomic<bool> configured[64];  // per instantiation, per device
  cudaError_t e = smem_limit_once(kernel, int(S::kSmemBytes), configured);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(unsigned(sms)), dim3(S::kThreads), S::kSmemBytes, stream, a);
}

}  // namespace

void paged_chunk_workspace(int head_dim, int sms, int64_t* o_floats, int64_t* ml_floats,
                           int* counters) {
  const int64_t slots = int64_t(sms) * 2 * (head_dim == 256 ? 1 : 2);
  *o_floats = slots * 128 * head_dim;
  *ml_floats = slots * 128 * 2;
  *counters = sms * 8;
}

cudaError_t launch_paged_chunk(const PagedAttendArgs& a, int sms, cudaStream_t stream) {
  switch (a.pool.head_dim) {
    case 64: return a.pool.q8 ? launch_chunk<64, true>(a, sms, stream) : launch_chunk<64, false>(a, sms, stream);
    case 128: return a.pool.q8 ? launch_chunk<128, true>(a, sms, stream) : launch_chunk<128, false>(a, sms, stream);
    case 256: return a.pool.q8 ? launch_chunk<256, true>(a, sms, stream) : launch_chunk<256, false>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace fa

// Chunks of many rows over a paged cache: not supported yet (the launch says so).
#include "fa_paged.h"
namespace fa {
void paged_chunk_workspace(int, int, int64_t* o, int64_t* ml, int* n) { *o = *ml = 0; *n = 0; }
cudaError_t launch_paged_chunk(const PagedAttendArgs&, int, cudaStream_t) { return cudaErrorNotSupported; }
}  // namespace fa

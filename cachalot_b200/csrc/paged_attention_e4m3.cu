// Paged attention over E4M3 caches, bfloat16 results (kernel and reasons: paged_attention.cuh).
#include "paged_attention.cuh"

namespace cachalot {
int launch_attend_e4m3(AttendArgs& a, int dim, int ctas, cudaStream_t stream) { return launch_attend<__half, true, 1>(a, dim, ctas, stream); }
}  // namespace cachalot

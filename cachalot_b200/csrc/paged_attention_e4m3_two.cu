// Paged attention over E4M3 caches with two terms of the softmax weights, for results that are not bfloat16 (kernel and reasons: paged_attention.cuh).
#include "paged_attention.cuh"

namespace cachalot {
int launch_attend_e4m3_two(AttendArgs& a, int dim, int ctas, cudaStream_t stream) { return launch_attend<__half, true, 2>(a, dim, ctas, stream); }
}  // namespace cachalot

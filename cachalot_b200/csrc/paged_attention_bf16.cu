// Paged attention over bfloat16 caches (kernel and reasons: paged_attention.cuh).
#include "paged_attention.cuh"

namespace cachalot {
int launch_attend_bf16(AttendArgs& a, int dim, int ctas, cudaStream_t stream) { return launch_attend<__nv_bfloat16, false, 2>(a, dim, ctas, stream); }
}  // namespace cachalot

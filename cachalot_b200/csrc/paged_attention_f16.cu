// Paged attention over float16 caches (kernel and reasons: paged_attention.cuh).
#include "paged_attention.cuh"

namespace cachalot {
int launch_attend_f16(AttendArgs& a, int dim, int ctas, cudaStream_t stream) { return launch_attend<__half, false, 2>(a, dim, ctas, stream); }
}  // namespace cachalot

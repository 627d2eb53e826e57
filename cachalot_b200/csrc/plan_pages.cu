// Page plan of a step: block tables, slots and positions of the new tokens, from request lengths that only the device
// knows.  Two exclusive sums over the requests (new tokens, new pages) and one lookup per token.
//
// A few hundred bytes of input: bound by latency.  One launch: every CTA redoes the two sums over all requests in shared
// memory (a load and two block scans, instead of a second launch or a grid-wide wait) and then places its own 256 tokens
// by binary search in the first.  The token at a page's start writes the page's table entry: every page that is new holds
// its first token among the new ones, so no CTA reads what another one writes.
#include "paged.cuh"

namespace cachalot {
namespace {

constexpr int PP_THREADS = 256;
constexpr int PP_MAX_REQUESTS = 8192;

// inclusive sum over the block; `total` = sum of all threads.  warp_sums: shared, one per warp.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PP_THREADS / 32; ++w) {
    const long long s = warp_sums[w];
    before += w < warp ? s : 0;
    total += s;
  }
  __syncthreads();
  return v + before;
}

struct PlanArgs {
  const int32_t *context, *fresh;
  int32_t* table;
  long long table_stride;
  const int32_t *free_pages, *free_count;
  int requests, width, n_free, page_size, tokens;
  int32_t *starts, *request_of, *positions, *slots, *lens, *free_out;
  int* status;
};

__global__ void __launch_bounds__(PP_THREADS) plan_pages_kernel(PlanArgs a) {
  extern __shared__ int sm[];
  wait_for_predecessor();
  __shared__ long long warp_sums[PP_THREADS / 32];
  int* start = sm;                     // [requests + 1] first token
  int* page0 = sm + a.requests + 1;    // [requests] pages taken by the requests before
  const int p = a.page_size;
  const bool first_cta = blockIdx.x == 0;
  int flags = 0;
  long long tokens_before = 0, pages_before = 0;
  for (int r0 = 0; r0 < a.requests; r0 += PP_THREADS) {
    const int r = r0 + threadIdx.x;
    const bool live = r < a.requests;
    int c = live ? a.context[r] : 0;
    int n = live ? a.fresh[r] : 0;
    if (c < 0 || n < 0) flags |= CACHALOT_STATUS_LENGTH, c = max(c, 0), n = max(n, 0);
    long long total;
    const long long end = tokens_before + block_scan(n, warp_sums, total);
    tokens_before += total;
    const int s = (int)min(end - n, (long long)a.tokens);
    const int kept = min(n, a.tokens - s);
    if (kept < n) flags |= CACHALOT_STATUS_LENGTH;
    const long long len = (long long)c + kept;
    if (len > (long long)a.width * p) flags |= CACHALOT_STATUS_LENGTH;
    const int held = (int)min(((long long)c + p - 1) / p, (long long)a.width);
    const int need = (int)min((len + p - 1) / p, (long long)a.width) - held;
    const long long pages_end = pages_before + block_scan(need, warp_sums, total);
    pages_before += total;
    if (live) {
      start[r] = s;
      page0[r] = (int)min(pages_end - need, 0x7fffffffLL);
      if (first_cta) a.starts[r] = s, a.lens[r] = (int)min(len, 0x7fffffffLL);
    }
  }
  const int placed = (int)min(tokens_before, (long long)a.tokens);
  int available = *a.free_count;
  if (available < 0 || available > a.n_free) flags |= CACHALOT_STATUS_LENGTH, available = min(max(available, 0), a.n_free);
  if (pages_before > available) flags |= CACHALOT_STATUS_NO_PAGE;
  if (threadIdx.x == 0) {
    start[a.requests] = placed;
    if (first_cta) a.starts[a.requests] = placed, *a.free_out = (int)max((long long)available - pages_before, 0LL);
  }
  __syncthreads();
  const int t = blockIdx.x * PP_THREADS + threadIdx.x;
  if (t < a.tokens) {
    int request = -1, slot = -1;
    long long pos = 0;
    if (t < placed) {
      int lo = 0, hi = a.requests;  // the last request whose first token is not past t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
      }
      request = lo;
      const int c = max(a.context[request], 0);
      pos = (long long)c + (t - start[request]);
      const long long j = pos / p;
      const int off = (int)(pos - j * p);
      if (j < a.width) {
        const int held = (int)(((long long)c + p - 1) / p);  // <= j + 1 <= width
        int32_t* entry = a.table + request * a.table_stride + j;
        int page;
        if (j < held) {
          page = *entry;
        } else {
          const long long rank = (long long)page0[request] + (j - held);
          page = rank < available ? a.free_pages[available - 1 - rank] : -1;
          if (off == 0) *entry = page;
        }
        const long long s = (long long)page * p + off;
        if (page >= 0 && s > 0x7fffffffLL) flags |= CACHALOT_STATUS_SLOT_RANGE;
        else if (page >= 0) slot = (int)s;
      }
    }
    a.request_of[t] = request;
    a.positions[t] = (int)min(pos, 0x7fffffffLL);
    a.slots[t] = slot;
  }
  if (a.status && flags) atomicOr(a.status, flags);
}

}  // namespace
}  // namespace cachalot

using namespace cachalot;

extern "C" int cachalot_plan_pages(const int32_t* context_lens, const int32_t* new_lens, int requests, int32_t* block_table,
                                   int64_t table_stride, int width, const int32_t* free_pages, int n_free, const int32_t* free_count,
                                   int page_size, int tokens, int32_t* starts, int32_t* request_of, int32_t* positions, int32_t* slots,
                                   int32_t* lens, int32_t* free_count_out, int* status, cachalot_stream_t stream) {
  if (requests < 0 || tokens < 0 || width < 0 || n_free < 0) return fail(CACHALOT_EINVAL, "plan_pages: negative size");
  if (page_size <= 0) return fail(CACHALOT_EINVAL, "plan_pages: page_size must be positive, got %d", page_size);
  if (requests > PP_MAX_REQUESTS) return fail(CACHALOT_EUNSUPPORTED, "plan_pages: %d requests (at most %d)", requests, PP_MAX_REQUESTS);
  if (!free_count || !free_count_out || !starts || (n_free && !free_pages)) return fail(CACHALOT_EINVAL, "plan_pages: null pointer");
  if (requests && (!context_lens || !new_lens || !lens || (width && !block_table))) return fail(CACHALOT_EINVAL, "plan_pages: null pointer");
  if (tokens && (!request_of || !positions || !slots)) return fail(CACHALOT_EINVAL, "plan_pages: null pointer");
  if (requests > 1 && table_stride < width) return fail(CACHALOT_EINVAL, "plan_pages: block table rows overlap");
  PlanArgs a{context_lens, new_lens, block_table, table_stride, free_pages, free_count, requests, width, n_free, page_size, tokens,
             starts, request_of, positions, slots, lens, free_count_out, status};
  const size_t smem = (2 * (size_t)requests + 1) * sizeof(int);
  if (smem > 40 * 1024) {  // without it 48 KB is the limit, of these and of the kernel's static arrays together
    const cudaError_t e = smem_optin_once(plan_pages_kernel, (2 * PP_MAX_REQUESTS + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "plan_pages: %s", cudaGetErrorString(e));
  }
  const unsigned grid = tokens ? (unsigned)(((long long)tokens + PP_THREADS - 1) / PP_THREADS) : 1u;
  const cudaError_t e = launch_early(plan_pages_kernel, dim3(grid), PP_THREADS, smem, (cudaStream_t)stream, 1, a);
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "plan_pages: %s", cudaGetErrorString(e));
  return check_launch("plan_pages");
}

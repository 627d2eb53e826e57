// Paged attention: argument checks, workspace, and the join of units that lie in several CTAs (the kernel itself:
// paged_attention.cuh).
#include "paged_attention.cuh"

namespace cachalot {
namespace {

constexpr int PA_MAX_SMS = 160;

struct JoinArgs {
  const float* part_o;
  const float2* part_ml;
  const int4* parts;
  int unit_heads, head_blocks, heads, group, dim;
  float shift;
  const float* v_scale;
  void* out;
  int out_dtype;
  float* lse;
};

// One CTA per CTA of the attention kernel.  The n CTAs that hold a part of a unit share its heads: head i belongs to the
// (i mod n)-th of them.  Few parts (n below the number of heads): a warp takes a head of its own; many parts: the four
// warps split a head's parts and meet in shared memory.  Part 0 of a unit is the second record of its CTA (the unit
// began there), the others are the first record of theirs.
template <int D>
__global__ void __launch_bounds__(PA_THREADS) attend_join_kernel(const JoinArgs a) {
  constexpr int E = D / 32;
  __shared__ float sums[PA_WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int which = 0; which < 2; ++which) {
    const int4 u = a.parts[blockIdx.x * 2 + which];  // request, unit, first CTA, CTAs
    if (u.w == 0) continue;
    const int n = u.w, h = u.y / a.head_blocks, head0 = u.y % a.head_blocks * a.unit_heads;
    const int heads = min(a.unit_heads, a.group - head0);
    const bool together = n >= heads;
    const long long row0 = (long long)u.x * a.heads + (long long)h * a.group + head0;
    const float v_scale = a.v_scale ? a.v_scale[h] : 1.f;
    for (int i = (int)blockIdx.x - u.z + (together ? 0 : warp * n); i < heads; i += together ? n : PA_WARPS * n) {
      auto slot = [&](int p) { return ((long long)(u.z + p) * 2 + (p == 0)) * a.unit_heads + i; };
      float top = -INFINITY, sum = 0.f;
      for (int p = lane; p < n; p += 32) top = fmaxf(top, a.part_ml[slot(p)].x);
      top = warp_max(top);
      for (int p = lane; p < n; p += 32) {
        const float2 ml = a.part_ml[slot(p)];
        sum += ml.x == -INFINITY ? 0.f : ml.y * ex2(ml.x - top);
      }
      sum = warp_sum(sum);
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
      for (int p = together ? warp : 0; p < n; p += together ? PA_WARPS : 1) {
        const float m = a.part_ml[slot(p)].x, f = m == -INFINITY ? 0.f : ex2(m - top);
        const float* from = a.part_o + slot(p) * D + lane;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(from[32 * e], f, v[e]);
      }
      const float inv = sum == 0.f ? 0.f : v_scale / sum;
      if (together) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) sums[warp][lane + 32 * e] = v[e];
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += PA_THREADS)
          store_out(a.out, a.out_dtype, (row0 + i) * D + d, (sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d]) * inv);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) store_out(a.out, a.out_dtype, (row0 + i) * D + lane + 32 * e, v[e] * inv);
      }
      if (a.lse && lane == 0 && (!together || warp == 0)) a.lse[row0 + i] = sum == 0.f ? -INFINITY : (top - a.shift + log2f(sum)) * PA_LN2;
    }
  }
}

bool shape_of(bool f8, int dim, int group, AttendLaunch* l) {
  auto take = [&](auto, auto, const AttendLaunch& s) { *l = s; };
  return f8 ? attend_dispatch<true>(dim, group, take) : attend_dispatch<false>(dim, group, take);
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    (void)cudaGetLastError();
    sms = PA_MAX_SMS;  // no device: sizes only
  }
  return sms < PA_MAX_SMS ? sms : PA_MAX_SMS;
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }

size_t workspace_of(const AttendLaunch& l, int dim, int ctas) {
  return up((size_t)ctas * 2 * sizeof(int4)) + up((size_t)ctas * 2 * l.unit_heads * sizeof(float2)) + (size_t)ctas * 2 * l.unit_heads * dim * sizeof(float);
}

}  // namespace
}  // namespace cachalot

using namespace cachalot;

extern "C" size_t cachalot_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int cache_dtype) {
  AttendLaunch l;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || !shape_of(cache_dtype == CACHALOT_E4M3, head_dim, heads / kv_heads, &l)) return 0;
  return workspace_of(l, head_dim, sm_count() * l.ctas_per_sm);
}

extern "C" int cachalot_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, int q_dtype, int requests, int heads,
                                        const cachalot_paged_kv* cache, const int32_t* block_table, int64_t table_stride, int width,
                                        const int32_t* lens, float scale, int window, float softcap, void* workspace,
                                        size_t workspace_bytes, void* out, int out_dtype, float* lse, int* status,
                                        cachalot_stream_t stream) {
  AttendArgs a = {};
  if (requests < 0 || heads <= 0 || width < 0) return fail(CACHALOT_EINVAL, "paged_attention: bad shape");
  if (q_dtype != CACHALOT_F16 && q_dtype != CACHALOT_BF16) return fail(CACHALOT_EINVAL, "paged_attention: queries are float16 or bfloat16");
  if (out_dtype != CACHALOT_F16 && out_dtype != CACHALOT_BF16 && out_dtype != CACHALOT_F32)
    return fail(CACHALOT_EINVAL, "paged_attention: output is float16, bfloat16 or float32");
  if (const int rc = paged_view("paged_attention", cache, &a.c)) return rc;
  if (heads % a.c.kv_heads) return fail(CACHALOT_EINVAL, "paged_attention: %d query heads over %d key-value heads", heads, a.c.kv_heads);
  if (a.c.dtype != CACHALOT_E4M3 && a.c.dtype != q_dtype) return fail(CACHALOT_EINVAL, "paged_attention: cache and queries differ in type");
  if (window < 0 || !(softcap >= 0.f)) return fail(CACHALOT_EINVAL, "paged_attention: window and softcap must not be negative");
  for (long long stride : {a.c.k_page, a.c.k_token, a.c.v_page, a.c.v_token})
    if (stride > 0xffffffffLL) return fail(CACHALOT_EUNSUPPORTED, "paged_attention: pages or tokens %lld bytes apart", stride);
  const bool f8 = a.c.dtype == CACHALOT_E4M3;
  AttendLaunch l;
  if (!shape_of(f8, a.c.head_dim, heads / a.c.kv_heads, &l))
    return fail(CACHALOT_EUNSUPPORTED, "paged_attention: head size %d (64, 96, 128, 192 and 256 are built)", a.c.head_dim);
  if (requests == 0) return CACHALOT_OK;
  if (!q || !lens || !out || (width && !block_table) || !workspace) return fail(CACHALOT_EINVAL, "paged_attention: null pointer");
  if (!aligned(q, 4) || q_row_stride % 2 || q_head_stride % 2) return fail(CACHALOT_EALIGN, "paged_attention: query heads need 4-byte alignment");
  if (requests > 1 && table_stride < width) return fail(CACHALOT_EINVAL, "paged_attention: block table rows overlap");
  if (!aligned(workspace, 256)) return fail(CACHALOT_EALIGN, "paged_attention: workspace needs 256-byte alignment");
  const int most = sm_count() * l.ctas_per_sm;
  if (workspace_bytes < workspace_of(l, a.c.head_dim, most))
    return fail(CACHALOT_ESCRATCH, "paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, workspace_of(l, a.c.head_dim, most));
  a.q = q, a.q_row = q_row_stride, a.q_head = q_head_stride, a.q_bf16 = q_dtype == CACHALOT_BF16;
  a.table = block_table, a.table_stride = table_stride, a.lens = lens;
  const long long room = (long long)width * a.c.page_size;
  a.room = room < 0x7fffff00LL ? (int)room : 0x7fffff00;
  a.requests = requests, a.heads = heads, a.group = heads / a.c.kv_heads, a.tiles = l.tiles, a.head_blocks = l.head_blocks;
  a.page_shift = -1;
  for (int s = 0; s < 28; ++s)
    if (a.c.page_size == 8 << s) a.page_shift = s;
  const int step_bytes = l.step * 2 * a.c.head_dim * paged_elem_bytes(a.c.dtype);
  a.unit_cost = (48 * 1024 + step_bytes - 1) / step_bytes;
  a.scale = scale, a.softcap = softcap, a.window = window, a.out = out, a.out_dtype = out_dtype, a.lse = lse, a.status = status;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  a.parts = reinterpret_cast<int4*>(w), w += up((size_t)most * 2 * sizeof(int4));
  a.part_ml = reinterpret_cast<float2*>(w), w += up((size_t)most * 2 * l.unit_heads * sizeof(float2));
  a.part_o = reinterpret_cast<float*>(w);
  // no more CTAs than there can be steps
  const long long steps = (a.room + l.step - 1) / l.step + 1 + a.unit_cost;
  const long long bound = steps * requests * a.c.kv_heads * l.head_blocks;
  const int ctas = (int)(bound < most ? bound : most);
  cudaStream_t s = (cudaStream_t)stream;
  const int rc = f8 ? launch_attend_e4m3(a, a.c.head_dim, ctas, s) : q_dtype == CACHALOT_BF16 ? launch_attend_bf16(a, a.c.head_dim, ctas, s)
                                                                                            : launch_attend_f16(a, a.c.head_dim, ctas, s);
  if (rc) return rc;
  JoinArgs j{a.part_o, a.part_ml, a.parts, l.unit_heads, l.head_blocks, heads, a.group, a.c.head_dim,
             f8 || q_dtype == CACHALOT_F16 ? 7.f : 0.f, f8 ? a.c.v_scale : nullptr, out, out_dtype, lse};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(PA_THREADS), cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = 1;
  cudaError_t e = cudaSuccess;
  switch (a.c.head_dim) {
    case 64: e = cudaLaunchKernelEx(&cfg, attend_join_kernel<64>, j); break;
    case 96: e = cudaLaunchKernelEx(&cfg, attend_join_kernel<96>, j); break;
    case 128: e = cudaLaunchKernelEx(&cfg, attend_join_kernel<128>, j); break;
    case 192: e = cudaLaunchKernelEx(&cfg, attend_join_kernel<192>, j); break;
    default: e = cudaLaunchKernelEx(&cfg, attend_join_kernel<256>, j); break;
  }
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "paged_attention: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}

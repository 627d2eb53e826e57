// Paged attention: argument checks, workspace, and the join of units that lie in several CTAs (the kernel itself:
// paged_attention.cuh).
#include <algorithm>
#include <cmath>

#include "paged_attention.cuh"

namespace cachalot {
namespace {

constexpr int PA_MAX_SMS = 160;

struct JoinArgs {
  const float* part_o;
  const float2* part_ml;
  const int4* parts;
  int unit_heads, head_blocks, heads, group;
  float shift;
  const float* v_scale;
  void* out;
  int out_dtype;
  float* lse;
};

// Some elements of an output head in the making, from the parts that a lane has seen: running maximum and sum with them.
template <int E>
struct Joined {
  float m = -INFINITY, l = 0.f, v[E] = {};
  // (a part without a maximum has a sum of 0, or of NaN, which 0 * NaN carries on)
  __device__ __forceinline__ void add(float om, float ol, const float (&o)[E]) {
    const float top = fmaxf(m, om), f = m == -INFINITY ? 0.f : ex2(m - top), g = om == -INFINITY ? 0.f : ex2(om - top);
    m = top, l = l * f + ol * g;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] * f + o[e] * g;
  }
  __device__ __forceinline__ void across(int lanes) {  // with the lane `lanes` away
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = __shfl_xor_sync(0xffffffffu, v[e], lanes);
    add(__shfl_xor_sync(0xffffffffu, m, lanes), __shfl_xor_sync(0xffffffffu, l, lanes), o);
  }
};

// One CTA per CTA of the attention kernel.  The n CTAs that hold a part of a unit share its work:
//   n <= 8   a task is a head, a warp's; its lanes hold the whole head and go through the parts
//   n <= 32  a task is 32 elements of a head, a warp's; eight lanes hold them, four parts at a time
//   n > 32   the same for a whole CTA, 16 parts at a time
// so that there are one or two rounds of loads in each case.  Part 0 of a unit is the second record of its CTA (the unit
// began there), the others are the first record of theirs.
template <int D>
__global__ void __launch_bounds__(PA_THREADS) attend_join_kernel(const JoinArgs a) {
  __shared__ Joined<4> shared[PA_WARPS][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_predecessor();
  for (int which = 0; which < 2; ++which) {
    const int4 u = a.parts[blockIdx.x * 2 + which];  // request, unit, first CTA, CTAs
    if (u.w == 0) continue;
    const int n = u.w, h = u.y / a.head_blocks, head0 = u.y % a.head_blocks * a.unit_heads, me = (int)blockIdx.x - u.z;
    const int heads = min(a.unit_heads, a.group - head0);
    const long long row0 = (long long)u.x * a.heads + (long long)h * a.group + head0;
    const float v_scale = a.v_scale ? a.v_scale[h] : 1.f;
    // parts p0, p0 + every, .. of elements d, d + stride, .. of a head
    auto gather = [&](auto& j, int p0, int every, int head, int d, auto vec) {
      constexpr int E = sizeof(j.v) / sizeof(float);
      for (int p = p0; p < n; p += 4 * every) {
        float2 ml[4];
        float o[4][E];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int q = p + i * every;
          const long long slot = ((long long)(u.z + q) * 2 + (q == 0)) * a.unit_heads + head;
          ml[i] = q < n ? a.part_ml[slot] : make_float2(-INFINITY, 0.f);
          const float* from = a.part_o + slot * D + d;
          if constexpr (decltype(vec)::value) {
            const float4 x = q < n ? *reinterpret_cast<const float4*>(from) : make_float4(0.f, 0.f, 0.f, 0.f);
            o[i][0] = x.x, o[i][1] = x.y, o[i][2] = x.z, o[i][3] = x.w;
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) o[i][e] = q < n ? from[32 * e] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) j.add(ml[i].x, ml[i].y, o[i]);
      }
    };
    auto finish = [&](const auto& j, int head, int d, int stride) {
      constexpr int E = sizeof(j.v) / sizeof(float);
      const float inv = j.l == 0.f ? 0.f : v_scale / j.l;
#pragma unroll
      for (int e = 0; e < E; ++e) store_out(a.out, a.out_dtype, (row0 + head) * D + d + e * stride, j.v[e] * inv);
      if (a.lse && d == 0) a.lse[row0 + head] = j.l == 0.f ? -INFINITY : (j.m - a.shift + log2f(j.l)) * PA_LN2;
    };
    if (n <= 8) {
      for (int head = me * PA_WARPS + warp; head < heads; head += n * PA_WARPS) {
        Joined<D / 32> j;
        gather(j, 0, 1, head, lane, std::false_type{});
        finish(j, head, lane, 32);
      }
      continue;
    }
    const bool together = n > 32;
    const int sub = lane >> 3, at = (lane & 7) * 4;
    for (int task = together ? me : me * PA_WARPS + warp; task < heads * (D / 32); task += together ? n : n * PA_WARPS) {
      const int head = task / (D / 32), d = task % (D / 32) * 32 + at;
      Joined<4> j;
      gather(j, together ? warp * 4 + sub : sub, together ? 4 * PA_WARPS : 4, head, d, std::true_type{});
      __syncwarp();
      j.across(8), j.across(16);
      if (together) {
        if (sub == 0) shared[warp][lane] = j;
        __syncthreads();
        j = shared[sub][lane & 7];
        j.across(8), j.across(16);
        __syncthreads();
        if (warp) continue;
      }
      if (sub == 0) finish(j, head, d, 1);
    }
  }
}

bool shape_of(bool f8, int dim, int group, AttendLaunch* l) {
  auto take = [&](auto, auto, const AttendLaunch& s) { *l = s; };
  return f8 ? attend_dispatch<true>(dim, group, take) : attend_dispatch<false>(dim, group, take);
}

int sm_count() { return std::min(device_sms(PA_MAX_SMS), PA_MAX_SMS); }  // no device: sizes only

size_t up(size_t v) { return (v + 255) / 256 * 256; }

// CTAs of one warp: as many warps as in CTAs of four
void make_one_warp(AttendLaunch* l) { l->ctas_per_sm *= PA_WARPS, l->step /= PA_WARPS; }

size_t workspace_of(const AttendLaunch& l, int dim, int ctas) {
  return up((size_t)ctas * 2 * sizeof(int4)) + up((size_t)ctas * 2 * l.unit_heads * sizeof(float2)) + (size_t)ctas * 2 * l.unit_heads * dim * sizeof(float);
}

}  // namespace
}  // namespace cachalot

using namespace cachalot;

extern "C" size_t cachalot_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int cache_dtype) {
  AttendLaunch l;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || !shape_of(cache_dtype == CACHALOT_E4M3, head_dim, heads / kv_heads, &l)) return 0;
  if (l.tiles == 1 && l.unit_heads <= 16) make_one_warp(&l);  // whichever form a call takes
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
  if (window < 0 || !(softcap >= 0.f) || std::isinf(softcap)) return fail(CACHALOT_EINVAL, "paged_attention: window and softcap must be finite and not negative");
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
  // CTAs of one warp where every CTA of four would begin more than one unit and no request is long: the four warps meet three
  // times for every unit, and what a unit costs besides its tokens (7 us) is then paid by one warp, not by four.  Heads of
  // 128, 8 heads to each of 8 key-value heads, one against four warps (us), bf16 and E4M3: 500 requests of up to 60 tokens 27
  // and 48, 35 and 56; 2000 86 and 182, 113 and 218; 160 of up to 400 22 and 29, 24 and 30; of up to 800 55 and 57, 45 and 52;
  // of up to 3000 57 and 54, 44 and 50; of up to 16000 188 and 170, 108 and 105 (more parts to join); with fewer units, 40
  // requests of up to 200, 12.8 and 11.4, 13.7 and 11.8.
  // The lengths are on the device, so "long" is what a row of the table holds, or the window: a table for 32768 tokens keeps
  // short requests with the four warps (lengths spread evenly, bf16 and E4M3: 500 of up to 60 52 us instead of 33, 60 instead
  // of 37; 2000 of up to 60 183 instead of 99, 212 instead of 112; 256 of up to 100, bf16, 32 instead of 27).
  const long long units = (long long)requests * a.c.kv_heads * l.head_blocks, table_room = (long long)width * a.c.page_size;
  const long long reach = window > 0 && window < table_room ? window : table_room;
  a.one_warp = l.tiles == 1 && l.unit_heads <= 16 && a.c.page_size % 8 == 0 && units > sm_count() * l.ctas_per_sm &&
               reach <= (f8 ? 4096 : 1024);
  const int cost_share = a.one_warp ? PA_WARPS : 1;
  if (a.one_warp) make_one_warp(&l);
  const int most = sm_count() * l.ctas_per_sm;
  if (workspace_bytes < workspace_of(l, a.c.head_dim, most))
    return fail(CACHALOT_ESCRATCH, "paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, workspace_of(l, a.c.head_dim, most));
  a.q = q, a.q_row = q_row_stride, a.q_head = q_head_stride, a.q_bf16 = q_dtype == CACHALOT_BF16;
  a.table = block_table, a.table_stride = table_stride, a.lens = lens;
  a.room = table_room < 0x7fffff00LL ? (int)table_room : 0x7fffff00;
  a.requests = requests, a.heads = heads, a.group = heads / a.c.kv_heads, a.tiles = l.tiles, a.head_blocks = l.head_blocks;
  a.page_shift = -1;
  for (int s = 0; s < 28; ++s)
    if (a.c.page_size == 8 << s) a.page_shift = s;
  const uint64_t pieces = (uint64_t)a.c.page_size / 8;
  a.page_magic = pieces > 0 && pieces < 128 ? ((1ull << 35) + pieces - 1) / pieces : 0;
  const int step_bytes = l.step * 2 * a.c.head_dim * paged_elem_bytes(a.c.dtype);
  // 48 KB: two steps of 128-element heads (a batch of very different lengths 44.7 us, with three 46.2); with two CTAs per SM, each
  // of which gets more of the bandwidth, 96 KB (16 heads to a key-value head 105 us, with 48 KB 113); over an E4M3 cache,
  // where instructions count for more than bytes, 384 tokens: three steps (batch of 64: 7 us less than with two)
  const int cost_bytes = (l.ctas_per_sm / cost_share > 2 ? 48 * 1024 : 96 * 1024) / cost_share;
  a.unit_cost = f8 ? (384 / cost_share + l.step - 1) / l.step : (cost_bytes + step_bytes - 1) / step_bytes;
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
  const auto launch = f8                        ? (out_dtype == CACHALOT_BF16 ? launch_attend_e4m3 : launch_attend_e4m3_two)
                      : q_dtype == CACHALOT_BF16 ? launch_attend_bf16 : launch_attend_f16;
  const int rc = launch(a, a.c.head_dim, ctas, s);
  if (rc) return rc;
  JoinArgs j{a.part_o, a.part_ml, a.parts, l.unit_heads, l.head_blocks, heads, a.group,
             f8 || q_dtype == CACHALOT_F16 ? 7.f : 0.f, f8 ? a.c.v_scale : nullptr, out, out_dtype, lse};
  cudaError_t e = cudaSuccess;
  auto join = [&](auto kern) { e = launch_early(kern, dim3(ctas), PA_THREADS, 0, s, 1, j); };
  switch (a.c.head_dim) {
    case 64: join(attend_join_kernel<64>); break;
    case 96: join(attend_join_kernel<96>); break;
    case 128: join(attend_join_kernel<128>); break;
    case 192: join(attend_join_kernel<192>); break;
    default: join(attend_join_kernel<256>); break;
  }
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "paged_attention: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}

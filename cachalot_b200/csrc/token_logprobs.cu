// Log probability of a given token, entropy and the n most likely tokens, per row of logits, in one pass over the row.
//
//   m running maximum, S = sum e^(x - m), U = sum e^(x - m) (x - m):
//   logprob(t) = x_t - m - ln S,  H = ln S - U / S;  when m moves to m': S' = f S, U' = f (U + S (m - m')), f = e^(m - m')
//
// HBM-bound: every logit is read once, 4 or 2 bytes, for one exponential and five other instructions.  Each thread keeps
// (m, S, U) of its own elements, 16-byte loads four deep.  A row is split over a cluster of CTAs where there are few rows,
// joined through distributed shared memory: one launch, no workspace.
// The alternatives: every warp keeps its n best so far sorted across its lanes (n <= 32) and only looks closer at loads
// whose maximum beats its last one and the last one of the CTA's best list; on logits in no particular order that is
// n (1 + ln(vocabulary / n)) insertions per CTA.  Ties go to the lower index: a warp walks the row upwards, so a later equal value
// never displaces an earlier one, and insertions and merges compare (value, index).
#include <cfloat>
#include <cooperative_groups.h>

#include "common.cuh"

namespace cachalot {
namespace {

namespace cg = cooperative_groups;

constexpr int TL_THREADS = 256, TL_WARPS = TL_THREADS / 32, TL_MAX_TOP = 32, TL_LOADS = 4;
constexpr float TL_LOG2E = 1.4426950408889634f;
constexpr float TL_FAR = -200.f;  // e^-200 is zero in fp32; stands for -inf, which would make 0 * -inf

__device__ __forceinline__ float fmax_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float exp_fast(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * TL_LOG2E));
  return y;
}

struct Sums {  // a maximum that covers the terms (never below -FLT_MAX), sum, sum weighted by distance
  float m, s, u;
  __device__ __forceinline__ void move(float to) {
    const float d = fmax_nan(m - to, TL_FAR), f = exp_fast(d);
    u = f * fmaf(s, d, u), s *= f, m = to;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float to = fmaxf(m, o.m);
    move(to), o.move(to);
    s += o.s, u += o.u;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = fmax_nan(x - m, TL_FAR), p = exp_fast(d);
    s += p, u = fmaf(p, d, u);
  }
};

struct Best {  // lane i holds the i-th best of a warp; empty: (-inf, INT_MAX)
  float v;
  int i;
};
__device__ __forceinline__ bool before(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }
// the whole warp inserts one candidate
__device__ __forceinline__ void insert(Best& b, int lane, float v, int i) {
  const int at = __popc(__ballot_sync(0xffffffffu, before(b.v, b.i, v, i)));
  const float uv = __shfl_up_sync(0xffffffffu, b.v, 1);
  const int ui = __shfl_up_sync(0xffffffffu, b.i, 1);
  if (lane > at) b.v = uv, b.i = ui;
  if (lane == at) b.v = v, b.i = i;
}
// ... the candidates that lanes hold, those that pass `take`
__device__ __forceinline__ void insert_all(Best& b, int lane, bool take, float v, int i) {
  for (unsigned hit = __ballot_sync(0xffffffffu, take); hit; hit &= hit - 1) {
    const int from = __ffs(hit) - 1;
    insert(b, lane, __shfl_sync(0xffffffffu, v, from), __shfl_sync(0xffffffffu, i, from));
  }
}

// order-preserving map of floats to unsigned (NaN does not occur here)
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned b = __float_as_uint(v);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }

template <typename T>
__device__ __forceinline__ float widen(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(TL_THREADS) token_logprobs_kernel(const T* __restrict__ logits, long long stride, int vocab,
                                                                    const int32_t* __restrict__ tokens, int top, float* __restrict__ logprobs,
                                                                    float* __restrict__ entropy, int32_t* __restrict__ top_ids,
                                                                    float* __restrict__ top_logprobs, int* status) {
  constexpr int PER = 16 / sizeof(T);
  __shared__ Sums parts[TL_WARPS];
  __shared__ float list_v[TL_WARPS][TL_MAX_TOP];
  __shared__ int list_i[TL_WARPS][TL_MAX_TOP];
  __shared__ unsigned bar;  // key of the best n-th value of any of the CTA's warps
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ctas, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = logits + row * stride;
  const int head = min(vocab, (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));  // elements before the first 16-byte boundary
  const int vectors = (vocab - head) / PER;
  const T* body = x + head;

  Sums sum{-FLT_MAX, 0.f, 0.f};
  Best best{-INFINITY, 0x7fffffff};
  float last = -INFINITY;   // the warp's n-th best
  bool full = false;
  if (TOP && threadIdx.x == 0) bar = 0;
  if (TOP) __syncthreads();

  auto settle = [&](int n) {  // after insertions
    last = __shfl_sync(0xffffffffu, best.v, n - 1);
    full = __shfl_sync(0xffffffffu, best.i, n - 1) != 0x7fffffff;
    if (full && lane == 0) atomicMax(&bar, key_of(last));
  };
  auto single = [&](int at, int end) {  // the warp takes up to 32 elements outside the 16-byte body
    const bool live = at + lane < end;
    const float v = live ? widen(x[at + lane]) : -INFINITY;
    if (live) {
      if (v > sum.m) sum.move(v);
      sum.add(v);
    }
    if (TOP) {
      insert_all(best, lane, live && v >= last, v, at + lane);
      settle(top);
    }
  };

  if (head && rank == 0 && warp == 0) single(0, head);
  const int walkers = ctas * TL_WARPS, me = rank * TL_WARPS + warp;
  for (int v0 = me * TL_LOADS * 32; v0 < vectors; v0 += walkers * TL_LOADS * 32) {
    float e[TL_LOADS][PER];
    float most = -INFINITY;
    uint4 raw[TL_LOADS];
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k) {
      const int at = v0 + k * 32 + lane;
      if (at < vectors) raw[k] = ld_stream_u4(body + (long long)at * PER);
    }
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k) {
      const bool live = v0 + k * 32 + lane < vectors;
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        float f;
        if constexpr (sizeof(T) == 4) f = __uint_as_float(w[j]);
        else if constexpr (std::is_same<T, __half>::value) f = __half2float(reinterpret_cast<const __half*>(w)[j]);
        else f = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        e[k][j] = live ? f : -INFINITY;
        most = fmaxf(most, e[k][j]);
      }
    }
    if (most > sum.m) sum.move(most);
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k)
#pragma unroll
      for (int j = 0; j < PER; ++j) sum.add(e[k][j]);
    if constexpr (TOP) {
      const unsigned b = *(volatile unsigned*)&bar;
      const float shared_last = b ? value_of(b) : -INFINITY;
      // strictly above the warp's own last one (all of its list comes before these), or at least the CTA's
      const bool look = full ? most > last && most >= shared_last : true;
      if (__any_sync(0xffffffffu, look)) {
        const float bound = fmaxf(last, shared_last);
#pragma unroll
        for (int k = 0; k < TL_LOADS; ++k) {
          const int at = v0 + k * 32 + lane;
#pragma unroll
          for (int j = 0; j < PER; ++j) insert_all(best, lane, at < vectors && e[k][j] >= bound, e[k][j], head + at * PER + j);
        }
        settle(top);
      }
    }
  }
  if (rank == ctas - 1 && warp == TL_WARPS - 1 && head + vectors * PER < vocab) single(head + vectors * PER, vocab);

  // ---- warps, then CTAs ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums other{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o), __shfl_xor_sync(0xffffffffu, sum.u, o)};
    sum.join(other);
  }
  if (lane == 0) parts[warp] = sum;
  if (TOP) list_v[warp][lane] = best.v, list_i[warp][lane] = best.i;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < TL_WARPS; ++w) {
      sum.join(parts[w]);
      if (TOP) {
        const float v = list_v[w][lane];
        const int i = list_i[w][lane];
        const float lv = __shfl_sync(0xffffffffu, best.v, top - 1);
        const int li = __shfl_sync(0xffffffffu, best.i, top - 1);
        insert_all(best, lane, lane < top && before(v, i, lv, li), v, i);
      }
    }
    __syncwarp();
    if (lane == 0) parts[0] = sum;
    if (TOP) list_v[0][lane] = best.v, list_i[0][lane] = best.i;
  }
  if (ctas > 1) {
    cluster.sync();
    if (rank == 0 && warp == 0) {
      for (int c = 1; c < ctas; ++c) {
        sum.join(*cluster.map_shared_rank(&parts[0], c));
        if (TOP) {
          const float v = *cluster.map_shared_rank(&list_v[0][lane], c);
          const int i = *cluster.map_shared_rank(&list_i[0][lane], c);
          const float lv = __shfl_sync(0xffffffffu, best.v, top - 1);
          const int li = __shfl_sync(0xffffffffu, best.i, top - 1);
          insert_all(best, lane, lane < top && before(v, i, lv, li), v, i);
        }
      }
    }
    cluster.sync();  // nobody leaves before its shared memory has been read
  }
  if (rank == 0 && warp == 0) {
    const float log_s = logf(sum.s);
    const bool none = sum.s == 0.f;  // every logit is -inf
    auto logp = [&](float v) { return none ? -INFINITY : v - sum.m - log_s; };
    if (lane == 0) {
      const int t = tokens[row];
      if (t >= vocab && status) atomicOr(status, CACHALOT_STATUS_ID_RANGE);
      logprobs[row] = t >= 0 && t < vocab ? logp(widen(x[t])) : 0.f;
      const float h = log_s - sum.u / sum.s;
      entropy[row] = none || h < 0.f ? 0.f : h;
    }
    if (TOP && lane < top) {
      const bool there = best.i != 0x7fffffff;
      top_ids[(long long)row * top + lane] = there ? best.i : -1;
      top_logprobs[(long long)row * top + lane] = there ? logp(best.v) : -INFINITY;
    }
  }
}

template <typename T>
cudaError_t launch(bool with_top, const cudaLaunchConfig_t& cfg, const void* logits, long long stride, int vocab, const int32_t* tokens, int top,
                   float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, int* status) {
  const T* x = static_cast<const T*>(logits);
  return with_top ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, x, stride, vocab, tokens, top, logprobs, entropy, top_ids, top_logprobs, status)
                  : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, x, stride, vocab, tokens, top, logprobs, entropy, top_ids, top_logprobs, status);
}

}  // namespace
}  // namespace cachalot

using namespace cachalot;

extern "C" int cachalot_token_logprobs(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const int32_t* tokens, int top,
                                       float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, int* status,
                                       cachalot_stream_t stream) {
  if (rows < 0 || vocab <= 0) return fail(CACHALOT_EINVAL, "token_logprobs: bad shape");
  if (dtype != CACHALOT_F32 && dtype != CACHALOT_BF16 && dtype != CACHALOT_F16)
    return fail(CACHALOT_EINVAL, "token_logprobs: logits are float32, bfloat16 or float16");
  if (top < 0 || top > vocab) return fail(CACHALOT_EINVAL, "token_logprobs: %d alternatives of %d tokens", top, vocab);
  if (top > TL_MAX_TOP) return fail(CACHALOT_EUNSUPPORTED, "token_logprobs: %d alternatives (at most %d)", top, TL_MAX_TOP);
  if (rows == 0) return CACHALOT_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top && (!top_ids || !top_logprobs))) return fail(CACHALOT_EINVAL, "token_logprobs: null pointer");
  const int es = dtype == CACHALOT_F32 ? 4 : 2;
  if (!aligned(logits, es)) return fail(CACHALOT_EALIGN, "token_logprobs: logits are not aligned to their type");
  if (vocab > 0x7fffffff - 65536) return fail(CACHALOT_EUNSUPPORTED, "token_logprobs: vocabulary of %d", vocab);
  // CTAs of a row: enough to fill the GPU with few rows, a power of two up to the portable cluster size
  int ctas = 1;
  while (ctas < 8 && (long long)rows * ctas * 2 <= 1184 && (long long)vocab * es / ctas > 32768) ctas *= 2;
  if ((long long)rows * ctas > 0x7fffffffLL) return fail(CACHALOT_EUNSUPPORTED, "token_logprobs: %d rows", rows);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)ctas, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas), cfg.blockDim = dim3(TL_THREADS), cfg.stream = (cudaStream_t)stream, cfg.attrs = &attr, cfg.numAttrs = 1;
  const auto go = dtype == CACHALOT_F32 ? launch<float> : dtype == CACHALOT_BF16 ? launch<__nv_bfloat16> : launch<__half>;
  const cudaError_t e = go(top > 0, cfg, logits, row_stride, vocab, tokens, top, logprobs, entropy, top_ids, top_logprobs, status);
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "token_logprobs: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}

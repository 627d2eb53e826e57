// Log probability of a given token, entropy and the n most likely tokens, per row of logits, in one pass over the row.
//
//   m running maximum, S = sum e^(x - m), U = sum e^(x - m) (x - m):
//   logprob(t) = x_t - m - ln S,  H = ln S - U / S;  when m moves to m': S' = f S, U' = f (U + S (m - m')), f = e^(m - m')
//
// HBM-bound: every logit is read once, 4 or 2 bytes, for one exponential and six other instructions.  Each thread keeps
// (m, S, U) of its own elements; the 16-byte loads of a round (four per thread) are issued before the round in hand is
// worked on.  A row is split over a cluster of CTAs where there are few rows, joined through distributed shared memory:
// one launch, no workspace.
//
// The alternatives.  The first round of a CTA finds the n-th largest of its threads' own maxima, a lower bound ("bar")
// of the n-th best that about n threads reach; from then on a thread whose maximum reaches the bar appends that maximum and
// its place to a list in shared memory, and after 4, 8, 16 .. rounds the bar is raised to the list's n-th largest: about n
// entries per doubling on logits in no particular order.  At the end the entries that reach the last bar, about n, are read again, an
// element per lane, and their elements that reach it sorted as 64-bit keys (value mapped to an ordered integer, complement
// of the index: all distinct, ties to the lower index).  Where a list overflows (rising logits, many equal ones) the share is
// read once more, bar raised as needed.  Selections are bitonic: warps sort 32 keys across their lanes and merge sorted lists.
// (Keeping the elements themselves while passing by cost 500 instructions for every thread that had one.)
#include <cfloat>
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "pairs.cuh"

namespace cachalot {
namespace {

namespace cg = cooperative_groups;

constexpr int TL_WARPS = 8;    // of a CTA; 4 or 2 for many rows
constexpr int TL_MAX_TOP = 32, TL_LOADS = 4;
constexpr int TL_CTAS = 4;     // of 8 warps per SM: up to 64 KB of loads in flight
constexpr int TL_LIST = 1088;  // 32 kept + 32 threads of 32 elements
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
};
struct PairSums {  // terms relative to one maximum, two at a time
  f32x2 s = 0, u = 0;
  __device__ __forceinline__ void add(float x, float y, f32x2 minus_m) {
    const float2 f = both(add2(pair(x, y), minus_m));
    const f32x2 d = pair(fmax_nan(f.x, TL_FAR), fmax_nan(f.y, TL_FAR));
    const float2 e = both(mul2(d, pair(TL_LOG2E, TL_LOG2E)));
    float2 v;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v.y) : "f"(e.y));
    const f32x2 p = pair(v.x, v.y);
    s = add2(s, p), u = fma2(p, d, u);
  }
};

using Key = unsigned long long;  // 0: none
__device__ __forceinline__ unsigned order_of(float v) {
  const unsigned b = __float_as_uint(v + 0.f);  // -0 counts as 0
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned b) { return b ? __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b) : -INFINITY; }
__device__ __forceinline__ Key key_of(float v, int i) { return (Key)order_of(v) << 32 | (unsigned)~i; }
__device__ __forceinline__ float value_of(Key k) {
  return value_of((unsigned)(k >> 32));
}
__device__ __forceinline__ int index_of(Key k) { return k ? (int)~(unsigned)k : -1; }

__device__ __forceinline__ Key swap_step(Key x, int lane, int j, bool down) {
  const Key y = __shfl_xor_sync(0xffffffffu, x, j);
  return ((lane & j) == 0) == down ? max(x, y) : min(x, y);
}
// 32 keys across the lanes, largest first
__device__ __forceinline__ Key sort32(Key x, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) x = swap_step(x, lane, j, (lane & k) == 0);
  return x;
}
// the 32 largest of two sorted lists, sorted
__device__ __forceinline__ Key merge32(Key a, Key b, int lane) {
  Key x = max(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) x = swap_step(x, lane, j, true);
  return x;
}
// the same of 32-bit keys (values alone), for bars
__device__ __forceinline__ unsigned swap_step(unsigned x, int lane, int j, bool down) {
  const unsigned y = __shfl_xor_sync(0xffffffffu, x, j);
  return ((lane & j) == 0) == down ? max(x, y) : min(x, y);
}
__device__ __forceinline__ unsigned sort32(unsigned x, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) x = swap_step(x, lane, j, (lane & k) == 0);
  return x;
}
__device__ __forceinline__ unsigned merge32(unsigned a, unsigned b, int lane) {
  unsigned x = max(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) x = swap_step(x, lane, j, true);
  return x;
}

// ... of the first `n` warps' sorted lists, in warp 0 and in lists[0]; the others' lists are empty
template <typename K>
__device__ __forceinline__ K merge_block(K x, K (*lists)[32], int warp, int lane, int n) {
  lists[warp][lane] = x;
  for (int step = 1; step < n; step <<= 1) {
    __syncthreads();
    if (warp % (2 * step) == 0) lists[warp][lane] = x = merge32(x, lists[warp + step][lane], lane);
  }
  __syncthreads();
  return x;
}
// warps of `all` that sort a list of this length, 32 at a time each
__device__ __forceinline__ int warps_of(int length, int all) { return min((length + 31) / 32, all); }

// 16 bytes of logits
template <typename T>
struct Vec {
  static constexpr int PER = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float at(int j) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(reinterpret_cast<const __half*>(w)[j]);
    else return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
  // the largest, NaN left out (-inf or NaN where there is nothing else)
  __device__ __forceinline__ float top() const {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const T2* h = reinterpret_cast<const T2*>(w);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(widen(m.x), widen(m.y));
    }
  }
  __device__ static __forceinline__ float widen(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
  }
  __device__ static __forceinline__ uint32_t bits(T x) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(x);
    else if constexpr (std::is_same<T, __half>::value) return __half_as_ushort(x);
    else return __bfloat16_as_ushort(x);
  }
  // elements [from, from + PER) of a row, -inf outside [0, vocab)
  __device__ __forceinline__ void load(const T* row, int from, int vocab) {
    if (from >= 0 && from + PER <= vocab) {
      raw = ld_once_u4(row + from);
      return;
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = from + j;
      uint32_t b = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
      if (i >= 0 && i < vocab) b = bits(row[i]);
      w[j * (int)sizeof(T) / 4] |= b << (sizeof(T) == 4 ? 0 : (j & 1) * 16);
    }
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A CTA's share of a row: 16-byte vectors (the first and the last of the row may reach over its ends), in rounds of
// TL_LOADS per thread, upwards.
template <typename T, int WARPS>
struct Share {
  static constexpr int THREADS = WARPS * 32;
  const T* row;
  int vocab, shift, ctas, rank, rounds;
  __device__ __forceinline__ Share(const T* r, int n, int c, int k) : row(r), vocab(n), ctas(c), rank(k) {
    shift = (int)(reinterpret_cast<uintptr_t>(r) % 16 / sizeof(T));
    rounds = ((n + shift + Vec<T>::PER - 1) / Vec<T>::PER + c * TL_LOADS * THREADS - 1) / (c * TL_LOADS * THREADS);
  }
  __device__ __forceinline__ int index(int round, int k, int thread) const {  // of the first element of a thread's k-th vector
    return (((round * ctas + rank) * TL_LOADS + k) * THREADS + thread) * Vec<T>::PER - shift;
  }
  __device__ __forceinline__ int index(int round, int k) const { return index(round, k, (int)threadIdx.x); }
  __device__ __forceinline__ void fetch(Vec<T> (&v)[TL_LOADS], int round) const {
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k) v[k].load(row, index(round, k), vocab);
  }
};

// A thread's best element of a round, the first of equal ones.
template <typename T, int WARPS>
__device__ __forceinline__ Key best_of(const Share<T, WARPS>& sh, const Vec<T> (&v)[TL_LOADS], int round, float most) {
  Key best = 0;
#pragma unroll
  for (int k = TL_LOADS - 1; k >= 0; --k)
#pragma unroll
    for (int j = Vec<T>::PER - 1; j >= 0; --j) {
      const int i = sh.index(round, k) + j;
      if (v[k].at(j) == most && i >= 0 && i < sh.vocab) best = key_of(most, i);
    }
  return best;
}
// A thread's elements of a round that reach the bar, appended to the list.
template <typename T, int WARPS>
__device__ __forceinline__ void offer(const Share<T, WARPS>& sh, const Vec<T> (&v)[TL_LOADS], int round, Key bar, float bar_value, Key* list, int base, int* count) {
#pragma unroll
  for (int k = 0; k < TL_LOADS; ++k) {
    if (!(v[k].top() >= bar_value)) continue;
#pragma unroll
    for (int j = 0; j < Vec<T>::PER; ++j) {
      const float x = v[k].at(j);
      const int i = sh.index(round, k) + j;
      if (x >= bar_value && i >= 0 && i < sh.vocab) {
        const Key key = key_of(x, i);
        if (key >= bar) {
          const int at = base + atomicAdd(count, 1);
          if (at < TL_LIST) list[at] = key;
        }
      }
    }
  }
}

// The careful selection, for rows where a list overflowed: over the share once more, the bar raised in every round that would
// overflow the list, from the list and the threads' own best together (at most n threads reach it, so at most 32 n elements).
// Returns the length of the list.  `added`: three counters for the rounds in turn (one counted, one still read, one cleared).
template <typename T, int WARPS>
__device__ __noinline__ int select_carefully(const Share<T, WARPS> sh, int top, Key* list, Key (*lists)[32], int* added) {
  constexpr int THREADS = WARPS * 32, CHUNKS = (TL_LIST + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int held = 0;
  Key bar = 0;
  float bar_value = -INFINITY;
  __syncthreads();
  if (tid < 3) added[tid] = 0;
  __syncthreads();
  for (int round = 0; round < sh.rounds; ++round) {
    Vec<T> v[TL_LOADS];
    sh.fetch(v, round);
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k) most = fmaxf(most, v[k].top());
    int* count = &added[round % 3];
    if (tid == 0) added[(round + 1) % 3] = 0;
    auto offer_all = [&](int base) {
      if (most >= bar_value) offer(sh, v, round, bar, bar_value, list, base, count);
    };
    if (round > 0) {
      offer_all(held);
      __syncthreads();
      const int n = *count;
      if (held + n <= TL_LIST) {
        held += n;
        continue;
      }
    }
    Key mine = sort32(best_of(sh, v, round, most), lane);  // what the round has added to the list is given up
    for (int at = warp * 32; at < held; at += THREADS) mine = merge32(mine, sort32(at + lane < held ? list[at + lane] : 0, lane), lane);
    merge_block(mine, lists, warp, lane, WARPS);
    bar = lists[0][top - 1], bar_value = value_of(bar);
    Key kept[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) kept[c] = c * THREADS + tid < held ? list[c * THREADS + tid] : 0;
    if (tid == 0) *count = 0;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (kept[c] && kept[c] >= bar) list[atomicAdd(count, 1)] = kept[c];
    offer_all(0);
    __syncthreads();
    held = *count;
  }
  return held;
}

template <typename T, bool TOP, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, TL_CTAS * TL_WARPS / WARPS) token_logprobs_kernel(const T* logits, long long stride, int vocab,
                                                                             const int32_t* tokens, int top, float* logprobs,
                                                                             float* entropy, int32_t* top_ids,
                                                                             float* top_logprobs, int* status) {
  using V = Vec<T>;
  constexpr int PER = V::PER, THREADS = WARPS * 32, SEEN = 128 * WARPS;
  __shared__ Sums parts[WARPS];
  __shared__ Key lists[TOP ? WARPS : 1][32];
  __shared__ Key list[TOP ? TL_LIST : 1];
  __shared__ uint2 seen[TOP ? SEEN : 1];  // maxima that reached the bar: ordered value, round * threads + thread
  __shared__ int added[3], noted;
  unsigned(*bars)[32] = reinterpret_cast<unsigned(*)[32]>(lists);
  wait_for_predecessor();
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = logits + row * stride;
  const Share<T, WARPS> sh(x, vocab, ctas, rank);

  Sums sum{-FLT_MAX, 0.f, 0.f};
  float bar = -INFINITY;  // nothing below it is among the best
  V next[TL_LOADS];
  sh.fetch(next, 0);
  if (TOP && tid == 0) added[0] = noted = 0;
  auto nth = [&](unsigned sorted, int warps) {  // of the warps' sorted values the n-th largest
    merge_block(sorted, bars, warp, lane, warps);
    const unsigned r = bars[0][top - 1];
    __syncthreads();
    return r;
  };
  auto raise = [&] {  // to the n-th largest of the maxima so far
    __syncthreads();
    const int n = noted;
    if (n > SEEN) return;
    unsigned mine = 0;
    for (int at = warp * 32; at < n; at += THREADS) mine = merge32(mine, sort32(at + lane < n ? seen[at + lane].x : 0u, lane), lane);
    bar = fmaxf(bar, value_of(nth(mine, warps_of(n, WARPS))));
  };
  for (int round = 0; round < sh.rounds; ++round) {
    V now[TL_LOADS];
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k) now[k] = next[k], most = fmaxf(most, now[k].top());
    if (round + 1 < sh.rounds) sh.fetch(next, round + 1);
    if (most > sum.m) sum.move(most);
    PairSums part;
    const f32x2 minus_m = pair(-sum.m, -sum.m);
#pragma unroll
    for (int k = 0; k < TL_LOADS; ++k)
#pragma unroll
      for (int j = 0; j < PER; j += 2) part.add(now[k].at(j), now[k].at(j + 1), minus_m);
    const float2 s2 = both(part.s), u2 = both(part.u);
    sum.s += s2.x + s2.y, sum.u += u2.x + u2.y;
    if constexpr (TOP) {
      if (round == 0) bar = value_of(nth(sort32(order_of(most), lane), WARPS));
      if (most >= bar && sh.index(round, 0) < vocab) {  // a thread past the row has nothing to note
        const int at = atomicAdd(&noted, 1);
        if (at < SEEN) seen[at] = make_uint2(order_of(most), round * THREADS + tid);
      }
      if (round > 2 && (round & (round + 1)) == 0 && round + 1 < sh.rounds) raise();
    }
  }

  // ---- warps, then CTAs ----
  auto join_lanes = [&](int from) {
    for (int o = from; o > 0; o >>= 1) {
      Sums other{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o), __shfl_xor_sync(0xffffffffu, sum.u, o)};
      sum.join(other);
    }
  };
  join_lanes(16);
  if (lane == 0) parts[warp] = sum;
  Key best = 0;
  __syncthreads();
  if constexpr (TOP) {
    raise();
    const int n = noted;
    int held = TL_LIST + 1;
    if (n <= SEEN) {  // the elements of the entries that reach the bar, a lane each
      for (int at = warp; at < n; at += WARPS) {
        const uint2 entry = seen[at];
        if (!(value_of(entry.x) >= bar)) continue;
        const int i = sh.index(entry.y / THREADS, lane / PER % TL_LOADS, entry.y % THREADS) + lane % PER;
        const bool there = lane < PER * TL_LOADS && i >= 0 && i < vocab;
        const float v = there ? V::widen(x[i]) : 0.f;
        const unsigned hit = __ballot_sync(0xffffffffu, there && v >= bar);
        int to = 0;
        if (lane == 0) to = atomicAdd(added, __popc(hit));
        to = __shfl_sync(0xffffffffu, to, 0) + __popc(hit & ((1u << lane) - 1));
        if ((hit >> lane & 1) && to < TL_LIST) list[to] = key_of(v, i);
      }
      __syncthreads();
      held = added[0];
    }
    if (held > TL_LIST) held = select_carefully(sh, top, list, lists, added);
    for (int at = warp * 32; at < held; at += THREADS) best = merge32(best, sort32(at + lane < held ? list[at + lane] : 0, lane), lane);
    best = merge_block(best, lists, warp, lane, warps_of(held, WARPS));
  }
  if (warp == 0) {
    sum = parts[lane % WARPS];
    join_lanes(WARPS / 2);
  }
  if (ctas > 1) {  // ctas <= WARPS: a warp for each CTA's list, lanes for their sums
    __syncthreads();
    if (tid == 0) parts[0] = sum;
    cluster.sync();
    if (rank == 0) {
      if (TOP && warp < ctas) best = *cluster.map_shared_rank(&lists[0][lane], warp);
      if (warp == 0) {
        sum = *cluster.map_shared_rank(&parts[0], lane % ctas);
        join_lanes(ctas / 2);
      }
    }
    cluster.sync();  // nobody leaves, and no list is written, before all have been read
    if (TOP && rank == 0) best = merge_block(warp < ctas ? best : 0, lists, warp, lane, ctas);
  }
  if (rank == 0 && warp == 0) {
    const float log_s = logf(sum.s);
    const bool none = sum.s == 0.f;  // every logit is -inf
    auto logp = [&](float v) { return none ? -INFINITY : v - sum.m - log_s; };
    if (lane == 0) {
      const int t = tokens[row];
      if (t >= vocab && status) atomicOr(status, CACHALOT_STATUS_ID_RANGE);
      logprobs[row] = t >= 0 && t < vocab ? logp(V::widen(x[t])) : 0.f;
      const float h = log_s - sum.u / sum.s;
      entropy[row] = none || h < 0.f ? 0.f : h;
    }
    if (TOP && lane < top) {
      top_ids[(long long)row * top + lane] = index_of(best);
      top_logprobs[(long long)row * top + lane] = best ? logp(value_of(best)) : -INFINITY;
    }
  }
}

template <typename T>
cudaError_t launch(bool with_top, int warps, int rows, int ctas, cudaStream_t stream, const void* logits, long long stride, int vocab, const int32_t* tokens, int top,
                   float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, int* status) {
  auto pick = [&](auto n) {
    constexpr int WARPS = decltype(n)::value;
    return with_top ? token_logprobs_kernel<T, true, WARPS> : token_logprobs_kernel<T, false, WARPS>;
  };
  using std::integral_constant;
  const auto kern = warps == 2 ? pick(integral_constant<int, 2>{})
                    : warps == 4 ? pick(integral_constant<int, 4>{}) : pick(integral_constant<int, TL_WARPS>{});
  return launch_early(kern, dim3((unsigned)rows * ctas), warps * 32, 0, stream, ctas, static_cast<const T*>(logits), stride, vocab, tokens, top, logprobs,
                      entropy, top_ids, top_logprobs, status);
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
  if (vocab > 0x7fffffff - 131072) return fail(CACHALOT_EUNSUPPORTED, "token_logprobs: vocabulary of %d", vocab);
  // What ends a row costs its CTA the same for any number of warps, so many rows get small CTAs (us with 2, 4 and 8 warps):
  // 600 rows of 4000 bf16 12.2, 8.4, 13.2; 600 of 129280 71.9, 52.2, 52.1; 1300 of 16000 26.2, 26.3, 27.4; 4096 of 4000 and the
  // 32 largest 41, 42, 62; 16384 of 32000 240, 267, 312; 2048 of 129280 119, 113, 116.
  const int places = device_sms(148) * TL_CTAS;  // 592 on a B200
  const int warps = rows > 2 * places && (long long)vocab * es <= 65536 ? 2 : rows > places ? 4 : TL_WARPS;
  // CTAs of a row: what takes the least time with 16 GB/s and a fixed part each, and the cluster's meeting where there is
  // more than one
  const double row_us = (double)vocab * es / 16e3, fixed_us = top ? 3.0 : 1.0, meet_us = top ? 3.0 : 1.5;
  int ctas = 1;
  double least = 1e30;
  for (int c = 1; c <= 8 && warps == TL_WARPS; c *= 2) {
    const double us = ceil((double)rows * c / places) * (row_us / c + fixed_us) + (c > 1 ? meet_us : 0.0);
    if (us < least) least = us, ctas = c;
  }
  if ((long long)rows * ctas > 0x7fffffffLL) return fail(CACHALOT_EUNSUPPORTED, "token_logprobs: %d rows", rows);
  const auto go = dtype == CACHALOT_F32 ? launch<float> : dtype == CACHALOT_BF16 ? launch<__nv_bfloat16> : launch<__half>;
  const cudaError_t e = go(top > 0, warps, rows, ctas, (cudaStream_t)stream, logits, row_stride, vocab, tokens, top, logprobs, entropy, top_ids, top_logprobs, status);
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "token_logprobs: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}

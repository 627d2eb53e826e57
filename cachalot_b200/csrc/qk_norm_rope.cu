// Queries, keys and values of new tokens on their way from the projection to attention, one pass: RMS norm of every query
// and key head, position rotation of (part of) the head, write of keys and values into a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          per head, w optional, all in fp32
//   (y_a, y_b) -> m (y_a cos - y_b sin, y_b cos + y_a sin)   pairs (i, i + r/2) or (2i, 2i + 1), i < r/2; the rest stays
//   one rounding at the end, to the activation type or to E4M3 of y / scale (saturated at 448)
//
// HBM-bound: 2 bytes in and 2 (or 1) out per element.  A head is a group of 8, 16 or 32 lanes with 8 elements (16 bytes)
// each, so the norm is a shuffle tree.  A CTA works on one token, so everything but the norm is the same for all of its
// heads: an output element is r (x A + p B), r the head's 1 / rms, p the partner element, A = m w cos, B = -/+ m w_p sin
// in registers.  Interleaved partners are in the same lane; those of the half layout are a second 16-byte load that hits
// L1 (fp32 values handed through shared memory instead: 365 instead of about 100 instructions per two heads, 124 us for
// 4096 tokens of 64 + 16 + 16 heads of 128; now 40 us).  Halves that are no whole 16-byte pieces go through shared memory as they are.
// Angles are computed once per token: position * frequency in 64 bits, reduced to a fraction of a turn there (a float
// product is off by 0.06 rad at position 10^6), then sincospif.
#include <cuda_fp8.h>

#include <type_traits>

#include "paged.cuh"
#include "pairs.cuh"

namespace cachalot {
namespace {

constexpr int QR_THREADS = 128;
constexpr int QR_BATCH = 4;  // query heads a group has in flight
constexpr int QR_MAX_DIM = 256;

struct Rows {  // activation rows, strides in elements
  const void* x;
  long long token, head;
};
struct RopeArgs {
  Rows q, k, v;
  const void *q_weight, *k_weight;
  int w_f32;
  float eps, magnitude;
  const int32_t* positions;
  const double* inv_freq;
  int half;
  int tokens, heads, kv_heads, dim;
  int crew_log2;  // groups of a CTA on one token
  float inv_dim;
  void *q_out, *k_out;
  PagedView cache;  // cache.k null: none
  const int32_t* slots;
  int* status;
};

// 16 bytes of activations as four pairs, and back
template <typename T>
__device__ __forceinline__ void widen8(const uint4& u, f32x2 (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pair(p.x, p.y);
    } else {
      f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 round8(const f32x2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = both(f[i]);
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 e4m3_8(const f32x2 (&f)[4]) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __nv_cvt_float2_to_fp8x2(both(f[i]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}
// elements at .. at + 8 of a norm weight, 1 without one
template <typename T>
__device__ __forceinline__ float weight(const void* w, int f32, int at) {
  if (!w) return 1.f;
  if (f32) return static_cast<const float*>(w)[at];
  if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const T*>(w)[at]);
  else return __bfloat162float(static_cast<const T*>(w)[at]);
}
template <typename T>
__device__ __forceinline__ void weights8(const void* w, int f32, int at, f32x2 (&f)[4]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair(1.f, 1.f);
  } else if (f32) {
    const float4 a = static_cast<const float4*>(w)[at / 4], b = static_cast<const float4*>(w)[at / 4 + 1];
    f[0] = pair(a.x, a.y), f[1] = pair(a.z, a.w), f[2] = pair(b.x, b.y), f[3] = pair(b.z, b.w);
  } else {
    widen8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(w) + at), f);
  }
}
__device__ __forceinline__ f32x2 swapped(f32x2 p) {
  const float2 v = both(p);
  return pair(v.y, v.x);
}

enum { PAIRS_ADJACENT, PAIRS_HALF, PAIRS_ANY };  // (2i, 2i+1); (i, i+r/2) in whole 16-byte pieces; (i, i+r/2) in any place

template <typename T, int L, int PAIRS>
struct Lane {  // what a lane does to its 8 elements of a query or key head
  f32x2 a[4], b[4];
  int turns;     // the rotated ones: a bit per pair (adjacent) or per element
  int partner;   // PAIRS_HALF: first element of the piece the partners are in
  int half, at;

  __device__ __forceinline__ int mate(int i) const { return i < half ? i + half : i - half; }
  __device__ __forceinline__ void place(int first, int h) {
    at = first, half = h, turns = 0;
#pragma unroll
    for (int e = 0; e < (PAIRS == PAIRS_ADJACENT ? 4 : 8); ++e) turns |= (PAIRS == PAIRS_ADJACENT ? at / 2 + e < half : at + e < 2 * half) << e;
    partner = PAIRS == PAIRS_HALF && turns ? mate(at) : at;
  }
  __device__ __forceinline__ void set(const void* w, int f32, const float* cs, const float* sn) {
    weights8<T>(w, f32, at, a);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = pair(0.f, 0.f);
    if (!turns) return;
    if constexpr (PAIRS == PAIRS_ANY) {
      float x[8], z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = at + e, k = i < half ? i : i - half;
        const bool on = turns >> e & 1;
        x[e] = weight<T>(w, f32, i) * (on ? cs[k] : 1.f);
        z[e] = on ? weight<T>(w, f32, mate(i)) * (i < half ? -sn[k] : sn[k]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = pair(x[2 * i], x[2 * i + 1]), b[i] = pair(z[2 * i], z[2 * i + 1]);
    } else if constexpr (PAIRS == PAIRS_ADJACENT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(turns >> i & 1)) continue;
        const float c = cs[at / 2 + i], s = sn[at / 2 + i];
        b[i] = mul2(swapped(a[i]), pair(-s, s)), a[i] = mul2(a[i], pair(c, c));
      }
    } else {
      f32x2 other[4];
      weights8<T>(w, f32, partner, other);
      const int k = at < half ? at : partner;
      const float sign = at < half ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = *reinterpret_cast<const float2*>(cs + k + 2 * i), s = *reinterpret_cast<const float2*>(sn + k + 2 * i);
        a[i] = mul2(a[i], pair(c.x, c.y)), b[i] = mul2(other[i], pair(sign * s.x, sign * s.y));
      }
    }
  }

  // y <- (y A + p B) / rms (or without the norm), `times` a factor on top; `piece`: the partner's, `row`: the head in shared memory
  __device__ __forceinline__ void apply(f32x2 (&y)[4], const uint4& piece, const T* row, bool normed, float eps, float inv_dim, float times) const {
    float r = times;
    if (normed) {
      f32x2 s2 = mul2(y[0], y[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) s2 = fma2(y[i], y[i], s2);
      float ss = both(s2).x + both(s2).y;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      r *= rsqrtf(fmaf(ss, inv_dim, eps));
    }
    const f32x2 r2 = pair(r, r);
    if (!turns) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], mul2(a[i], r2));
      return;
    }
    // the partner of an element that stays is 0, not itself: 0 * inf is not 0
    f32x2 p[4];
    if constexpr (PAIRS == PAIRS_ADJACENT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = turns >> i & 1 ? swapped(y[i]) : 0;
    } else if constexpr (PAIRS == PAIRS_HALF) {
      widen8<T>(piece, p);
    } else {
      if (half & 1) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = turns >> e & 1 ? weight<T>(row, 0, mate(at + e)) : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
      } else {  // two neighbours have neighbours for partners
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = turns >> 2 * i & 1 ? *reinterpret_cast<const uint32_t*>(row + mate(at + 2 * i)) : 0u;
        widen8<T>(make_uint4(w[0], w[1], w[2], w[3]), p);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mul2(r2, fma2(p[i], b[i], mul2(y[i], a[i])));
  }
};

template <typename T, int L, int PAIRS, bool SEVERAL>  // SEVERAL: tokens of a CTA
__global__ void __launch_bounds__(QR_THREADS) qk_norm_rope_kernel(const RopeArgs a) {
  constexpr int GROUPS = QR_THREADS / L;
  using std::integral_constant;
  wait_for_predecessor();
  __shared__ __align__(16) float cs[SEVERAL ? GROUPS : 1][L * 4], sn[SEVERAL ? GROUPS : 1][L * 4];  // per token of the CTA
  __shared__ uint4 staged[PAIRS == PAIRS_ANY ? QR_BATCH : 1][PAIRS == PAIRS_ANY ? QR_THREADS : 1];
  // a CTA's groups: `crew` of them on each of its tokens, which take the token's heads in turn
  const int group = threadIdx.x / L, crew = SEVERAL ? 1 << a.crew_log2 : GROUPS, tokens = SEVERAL ? GROUPS >> a.crew_log2 : 1;
  const int member = SEVERAL ? group & (crew - 1) : group, mine = SEVERAL ? group >> a.crew_log2 : 0, half = a.half;
  const int token = blockIdx.x * tokens + mine;
  const int step = crew * gridDim.y, first = blockIdx.y * crew;  // heads first + member, + step, ..
  const bool exists = !SEVERAL || token < a.tokens, live = threadIdx.x % L * 8 < a.dim && exists;
  const int at = threadIdx.x % L * 8 < a.dim ? threadIdx.x % L * 8 : 0;  // lanes past the head count as zeros
  Lane<T, L, PAIRS> ln;
  ln.place(at, half);
  for (int i = threadIdx.x; i < tokens * half; i += QR_THREADS) {
    const int t = SEVERAL ? i / half : 0, f = i - t * half;
    if (SEVERAL && blockIdx.x * tokens + t >= a.tokens) break;
    const double turns = (double)a.positions[blockIdx.x * tokens + t] * a.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[t][f] = c * a.magnitude, sn[t][f] = s * a.magnitude;
  }
  __syncthreads();
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // heads h0 + member, + step, .. (N of them); CHECK: the last ones may not be there
  auto loads = [&](auto n, auto check, const T* x, long long head, int heads, int h0, int from, bool wanted, uint4* v) {
    const T* p = x + (long long)(h0 + member) * head + from;
#pragma unroll
    for (int i = 0; i < decltype(n)::value; ++i, p += step * head)
      v[i] = wanted && (!decltype(check)::value || h0 + member + i * step < heads) ? *reinterpret_cast<const uint4*>(p) : zero;
  };
  // as many whole batches as there are, then one by one
  auto over = [&](int heads, auto batch, auto&& work) {
    constexpr int N = decltype(batch)::value;
    int h = first;
    for (; h + (N - 1) * step + crew <= heads; h += N * step) work(batch, integral_constant<bool, false>{}, h);
    for (; h < heads; h += step) work(integral_constant<int, 1>{}, integral_constant<bool, true>{}, h);
  };
  // PAIRS_ANY: the heads of a batch as they are, for the lanes that have their partners
  auto stage = [&](auto n, const uint4* v) {
    if constexpr (PAIRS == PAIRS_ANY) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < decltype(n)::value; ++i) staged[i][threadIdx.x] = v[i];
      __syncwarp();
    }
  };
  auto row = [&](int i) { return PAIRS == PAIRS_ANY ? reinterpret_cast<const T*>(&staged[i][group * L]) : nullptr; };

  const T* q = static_cast<const T*>(a.q.x) + token * a.q.token;
  T* q_out = static_cast<T*>(a.q_out) + (long long)token * a.heads * a.dim + at;
  ln.set(a.q_weight, a.w_f32, cs[mine], sn[mine]);
  over(a.heads, integral_constant<int, QR_BATCH>{}, [&](auto n, auto check, int h0) {
    constexpr int N = decltype(n)::value;
    uint4 own[N], piece[N];
    loads(n, check, q, a.q.head, a.heads, h0, at, live, own);
    if (PAIRS == PAIRS_HALF) loads(n, check, q, a.q.head, a.heads, h0, ln.partner, live, piece);
    stage(n, own);
    T* out = q_out + (h0 + member) * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i, out += step * a.dim) {
      f32x2 y[4];
      widen8<T>(own[i], y);
      ln.apply(y, piece[i], row(i), a.q_weight != nullptr, a.eps, a.inv_dim, 1.f);
      if (live && (!decltype(check)::value || h0 + member + i * step < a.heads)) *reinterpret_cast<uint4*>(out) = round8<T>(y);
    }
  });

  bool stored = false;
  uint8_t *k_row = nullptr, *v_row = nullptr;
  if (a.cache.k && exists) {
    const int slot = a.slots[token];
    const int n = a.cache.n_pages * a.cache.page_size;
    stored = slot >= 0 && slot < n;
    if (slot >= n && a.status && member == 0 && threadIdx.x % L == 0 && blockIdx.y == 0) atomicOr(a.status, CACHALOT_STATUS_SLOT_RANGE);
    const int page = stored ? slot / a.cache.page_size : 0, off = stored ? slot - page * a.cache.page_size : 0;
    k_row = a.cache.k + page * a.cache.k_page + off * a.cache.k_token;
    v_row = a.cache.v + page * a.cache.v_page + off * a.cache.v_token;
  }
  if (!SEVERAL && !stored && !a.k_out) return;
  const bool f8 = a.cache.dtype == CACHALOT_E4M3, wanted = live && (!SEVERAL || stored || a.k_out);
  const T* k = static_cast<const T*>(a.k.x) + token * a.k.token;
  const T* v = static_cast<const T*>(a.v.x) + token * a.v.token;
  ln.set(a.k_weight, a.w_f32, cs[mine], sn[mine]);
  over(a.kv_heads, integral_constant<int, 2>{}, [&](auto n, auto check, int h0) {
    constexpr int N = decltype(n)::value;
    uint4 own[N], piece[N], value[N];
    loads(n, check, k, a.k.head, a.kv_heads, h0, at, wanted, own);
    if (PAIRS == PAIRS_HALF) loads(n, check, k, a.k.head, a.kv_heads, h0, ln.partner, wanted, piece);
    if (SEVERAL ? a.cache.k != nullptr : stored) loads(n, check, v, a.v.head, a.kv_heads, h0, at, wanted && (!SEVERAL || stored), value);
    stage(n, own);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + member + i * step;
      const bool there = wanted && (!decltype(check)::value || h < a.kv_heads);
      f32x2 y[4];
      widen8<T>(own[i], y);
      // E4M3: times 1 / scale, one more rounding to fp32 than the division, instead of eight divisions
      const float k_times = f8 && a.cache.k_scale && there ? 1.f / a.cache.k_scale[h] : 1.f;
      ln.apply(y, piece[i], row(i), a.k_weight != nullptr, a.eps, a.inv_dim, k_times);
      if (!there) continue;
      if (a.k_out) *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + ((long long)token * a.kv_heads + h) * a.dim + at) = round8<T>(y);
      if (!stored) continue;
      uint8_t *ks = k_row + h * a.cache.k_head, *vs = v_row + h * a.cache.v_head;
      if (f8) {
        *reinterpret_cast<uint2*>(ks + at) = e4m3_8(y);
        widen8<T>(value[i], y);
        const float v_times = a.cache.v_scale ? 1.f / a.cache.v_scale[h] : 1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = mul2(y[j], pair(v_times, v_times));
        *reinterpret_cast<uint2*>(vs + at) = e4m3_8(y);
      } else {
        *reinterpret_cast<uint4*>(ks + at * 2) = round8<T>(y);
        *reinterpret_cast<uint4*>(vs + at * 2) = value[i];
      }
    }
  });
}

int check_rows(const char* name, const void* x, int64_t token, int64_t head) {
  if (!x) return fail(CACHALOT_EINVAL, "qk_norm_rope: null %s", name);
  if (!aligned(x, 16) || token % 8 || head % 8) return fail(CACHALOT_EALIGN, "qk_norm_rope: rows of %s need 16-byte alignment", name);
  return CACHALOT_OK;
}

}  // namespace
}  // namespace cachalot

using namespace cachalot;

extern "C" int cachalot_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                                     int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                     int tokens, int heads, int kv_heads, int head_dim, const void* q_weight, const void* k_weight,
                                     int w_dtype, float eps, const int32_t* positions, const double* inv_freq, int rotary_dim,
                                     int interleaved, float magnitude, void* q_out, void* k_out, const cachalot_paged_kv* cache,
                                     const int32_t* slots, int* status, cachalot_stream_t stream) {
  if (tokens < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return fail(CACHALOT_EINVAL, "qk_norm_rope: bad shape");
  if (dtype != CACHALOT_F16 && dtype != CACHALOT_BF16) return fail(CACHALOT_EINVAL, "qk_norm_rope: activations are float16 or bfloat16");
  if (head_dim > QR_MAX_DIM || head_dim % 8) return fail(CACHALOT_EUNSUPPORTED, "qk_norm_rope: head size %d (multiples of 8 up to %d)", head_dim, QR_MAX_DIM);
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(CACHALOT_EINVAL, "qk_norm_rope: rotary size %d must be even and at most the head size %d", rotary_dim, head_dim);
  if ((q_weight || k_weight) && w_dtype != dtype && w_dtype != CACHALOT_F32)
    return fail(CACHALOT_EINVAL, "qk_norm_rope: norm weights have the activations' type or float32");
  if (tokens == 0) return CACHALOT_OK;
  if (!cache && !k_out) return fail(CACHALOT_EINVAL, "qk_norm_rope: the keys go nowhere (no cache, no output)");
  if (!q_out || !positions || (rotary_dim && !inv_freq)) return fail(CACHALOT_EINVAL, "qk_norm_rope: null pointer");
  RopeArgs a = {};
  if (const int rc = check_rows("q", q, q_token_stride, q_head_stride)) return rc;
  if (const int rc = check_rows("k", k, k_token_stride, k_head_stride)) return rc;
  if (!aligned(q_out, 16) || !aligned(k_out, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16))
    return fail(CACHALOT_EALIGN, "qk_norm_rope: outputs and weights need 16-byte alignment");
  if (cache) {
    if (const int rc = check_rows("v", v, v_token_stride, v_head_stride)) return rc;
    if (const int rc = paged_view("qk_norm_rope", cache, &a.cache)) return rc;
    if (!slots) return fail(CACHALOT_EINVAL, "qk_norm_rope: null slots");
    if (cache->kv_heads != kv_heads || cache->head_dim != head_dim)
      return fail(CACHALOT_EINVAL, "qk_norm_rope: cache holds %d heads of %d, keys have %d of %d", cache->kv_heads, cache->head_dim, kv_heads, head_dim);
    if (cache->dtype != CACHALOT_E4M3 && cache->dtype != dtype) return fail(CACHALOT_EINVAL, "qk_norm_rope: cache and activations differ in type");
  }
  a.q = {q, q_token_stride, q_head_stride}, a.k = {k, k_token_stride, k_head_stride}, a.v = {v, v_token_stride, v_head_stride};
  a.q_weight = q_weight, a.k_weight = k_weight, a.w_f32 = w_dtype == CACHALOT_F32, a.eps = eps, a.magnitude = magnitude;
  a.positions = positions, a.inv_freq = inv_freq, a.half = rotary_dim / 2;
  a.tokens = tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim, a.inv_dim = 1.f / (float)head_dim, a.q_out = q_out, a.k_out = k_out, a.slots = slots, a.status = status;
  const int lanes = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32, groups = QR_THREADS / lanes;
  // Many tokens of few heads: several tokens share a CTA, so that a group has eight heads per setting of its factors (18589
  // tokens of 6 + 2 + 2 heads of 128: 22.6 us; 16384 of 16 + 2 + 2: 40 us, with four heads per setting 52).  Few tokens: their heads go over several CTAs.
  const int sms = device_sms(148);
  int crew = groups;
  while (crew > 1 && heads < 8 * crew && (long long)tokens * crew / groups >= 8 * sms) crew /= 2;
  for (a.crew_log2 = 0; 1 << a.crew_log2 < crew;) ++a.crew_log2;
  const long long parts = ((long long)heads + groups - 1) / groups, want = (4 * sms + (long long)tokens - 1) / tokens;
  const dim3 grid((unsigned)((tokens + (long long)groups / crew - 1) / (groups / crew)), (unsigned)(parts < want ? parts : want));
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  auto run = [&](auto type, auto l) {
    using T = decltype(type);
    constexpr int L = decltype(l)::value;
    auto pick = [&](auto several) {
      constexpr bool SEVERAL = decltype(several)::value;
      return interleaved       ? qk_norm_rope_kernel<T, L, PAIRS_ADJACENT, SEVERAL>
             : rotary_dim % 16 ? qk_norm_rope_kernel<T, L, PAIRS_ANY, SEVERAL>
                               : qk_norm_rope_kernel<T, L, PAIRS_HALF, SEVERAL>;
    };
    e = launch_early(crew < groups ? pick(std::true_type{}) : pick(std::false_type{}), grid, QR_THREADS, 0, s, 1, a);
  };
  auto go = [&](auto type) {
    if (lanes == 8) run(type, std::integral_constant<int, 8>{});
    else if (lanes == 16) run(type, std::integral_constant<int, 16>{});
    else run(type, std::integral_constant<int, 32>{});
  };
  if (dtype == CACHALOT_F16) go(__half{});
  else go(__nv_bfloat16{});
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "qk_norm_rope: %s", cudaGetErrorString(e));
  return check_launch("qk_norm_rope");
}

// Queries, keys and values of new tokens on their way from the projection to attention, one pass: RMS norm of every query
// and key head, position rotation of (part of) the head, write of keys and values into a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          per head, w optional, all in fp32
//   (y_a, y_b) -> m (y_a cos - y_b sin, y_b cos + y_a sin)   pairs (i, i + r/2) or (2i, 2i + 1), i < r/2; the rest stays
//   one rounding at the end, to the activation type or to E4M3 of y / scale (saturated at 448)
//
// HBM-bound: 2 bytes in and 2 (or 1) out per element.  A head is a group of 8, 16 or 32 lanes with 8 elements (16 bytes)
// each, so the norm is a shuffle tree and interleaved pairs sit in one lane; the half layout fetches the partner through
// shared memory.  A CTA works on one token, so its angles are computed once for all of its heads: position * frequency in
// 64 bits, reduced to a fraction of a turn there (a float product is off by 0.06 rad at position 10^6), then sincospif.
#include <cuda_fp8.h>

#include "paged.cuh"

namespace cachalot {
namespace {

constexpr int QR_THREADS = 256;
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
  int half, interleaved;
  int heads, kv_heads, dim;
  void *q_out, *k_out;
  PagedView cache;  // cache.k null: none
  const int32_t* slots;
  int* status;
};

template <typename T>
__device__ __forceinline__ void widen8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 round8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 e4m3_8(const float (&f)[8]) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}
template <typename T>
__device__ __forceinline__ void weights8(const void* w, int f32, int at, bool live, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 1.f;
  if (!w || !live) return;
  if (f32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<const float*>(w)[at + e];
  } else {
    widen8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(w) + at), f);
  }
}

template <typename T, int L>
__global__ void __launch_bounds__(QR_THREADS) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int GROUPS = QR_THREADS / L;
  __shared__ __align__(16) float cs[QR_MAX_DIM / 2], sn[QR_MAX_DIM / 2];
  __shared__ __align__(16) float swap[GROUPS][2][L][4];  // a lane's elements 0-3 and 4-7 apart: no bank conflicts
  const int token = blockIdx.x, group = threadIdx.x / L, lane = threadIdx.x % L;
  const int at = lane * 8, half = a.half;
  const bool in_head = at < a.dim;
  for (int i = threadIdx.x; i < half; i += QR_THREADS) {
    const double turns = (double)a.positions[token] * a.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = c * a.magnitude, sn[i] = s * a.magnitude;
  }
  float wq[8], wk[8];
  weights8<T>(a.q_weight, a.w_f32, at, in_head, wq);
  weights8<T>(a.k_weight, a.w_f32, at, in_head, wk);
  long long page = 0;
  int off = 0;
  bool stored = false;
  if (a.cache.k) {
    const int slot = a.slots[token];
    const int n = a.cache.n_pages * a.cache.page_size;
    stored = slot >= 0 && slot < n;
    if (slot >= n && a.status && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, CACHALOT_STATUS_SLOT_RANGE);
    if (stored) page = slot / a.cache.page_size, off = slot - (int)page * a.cache.page_size;
  }
  const bool f8 = a.cache.dtype == CACHALOT_E4M3;
  const int es = f8 ? 1 : 2;
  const int k_from = a.heads, v_from = a.heads + (stored || a.k_out ? a.kv_heads : 0), items = v_from + (stored ? a.kv_heads : 0);
  __syncthreads();
  for (int base = blockIdx.y * GROUPS; base < items; base += gridDim.y * GROUPS) {
    const int it = base + group;
    const bool live = it < items && in_head;
    const int what = it < k_from ? 0 : it < v_from ? 1 : 2;
    const int h = it - (what == 0 ? 0 : what == 1 ? k_from : v_from);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) {
      const Rows& r = what == 0 ? a.q : what == 1 ? a.k : a.v;
      raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(r.x) + token * r.token + h * r.head + at);
    }
    float y[8];
    widen8<T>(raw, y);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const bool normed = what == 0 ? a.q_weight != nullptr : what == 1 && a.k_weight != nullptr;
    if (normed) {
      const float inv = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (what ? wk[e] : wq[e]);
    }
    if (a.interleaved) {
      if (what < 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = lane * 4 + e;
          if (i < half) {
            const float u = y[2 * e], v = y[2 * e + 1];
            y[2 * e] = u * cs[i] - v * sn[i], y[2 * e + 1] = v * cs[i] + u * sn[i];
          }
        }
      }
    } else {
      float4* mine = reinterpret_cast<float4*>(&swap[group][0][lane][0]);
      mine[0] = make_float4(y[0], y[1], y[2], y[3]);
      mine[L] = make_float4(y[4], y[5], y[6], y[7]);
      __syncwarp();
      if (what < 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = at + e;
          if (i < 2 * half) {
            const int j = i < half ? i + half : i - half, k = i < half ? i : j;
            const float p = swap[group][(j >> 2) & 1][j >> 3][j & 3];
            y[e] = i < half ? y[e] * cs[k] - p * sn[k] : y[e] * cs[k] + p * sn[k];
          }
        }
      }
      __syncwarp();
    }
    if (!live) continue;
    if (what == 0) {
      *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + ((long long)token * a.heads + h) * a.dim + at) = round8<T>(y);
      continue;
    }
    if (what == 1 && a.k_out) *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + ((long long)token * a.kv_heads + h) * a.dim + at) = round8<T>(y);
    if (!stored) continue;
    uint8_t* row = what == 1 ? a.cache.k + page * a.cache.k_page + h * a.cache.k_head + off * a.cache.k_token
                             : a.cache.v + page * a.cache.v_page + h * a.cache.v_head + off * a.cache.v_token;
    row += at * es;
    if (f8) {
      const float* scales = what == 1 ? a.cache.k_scale : a.cache.v_scale;
      if (scales) {
        const float s = scales[h];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] / s;
      }
      *reinterpret_cast<uint2*>(row) = e4m3_8(y);
    } else {
      *reinterpret_cast<uint4*>(row) = what == 1 ? round8<T>(y) : raw;
    }
  }
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
  a.positions = positions, a.inv_freq = inv_freq, a.half = rotary_dim / 2, a.interleaved = interleaved != 0;
  a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim, a.q_out = q_out, a.k_out = k_out, a.slots = slots, a.status = status;
  const int lanes = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32, groups = QR_THREADS / lanes;
  const long long parts = ((long long)heads + 2 * kv_heads + groups - 1) / groups;  // passes of a CTA that takes a whole token
  const long long want = (600 + (long long)tokens - 1) / tokens;                    // few tokens: their heads over more CTAs
  const dim3 grid((unsigned)tokens, (unsigned)(parts < want ? parts : want));
  cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto type) {
    using T = decltype(type);
    if (lanes == 8) qk_norm_rope_kernel<T, 8><<<grid, QR_THREADS, 0, s>>>(a);
    else if (lanes == 16) qk_norm_rope_kernel<T, 16><<<grid, QR_THREADS, 0, s>>>(a);
    else qk_norm_rope_kernel<T, 32><<<grid, QR_THREADS, 0, s>>>(a);
  };
  if (dtype == CACHALOT_F16) go(__half{});
  else go(__nv_bfloat16{});
  return check_launch("qk_norm_rope");
}

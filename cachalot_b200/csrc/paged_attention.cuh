// Attention of one new token per request over a paged key-value cache: the kernel, instantiated per cache type in
// paged_attention_{bf16,f16,e4m3,e4m3_two}.cu.
//
//   s_j = scale * q . k_j   (cap * tanh(s / cap) with a soft cap),  j in [max(0, len - window), len)
//   out = sum_j 2^(s_j log2 e - m) v_j / sum_j 2^(s_j log2 e - m),  m a running maximum
//
// HBM-bound: every visible key and value is read once for the G query heads that share it, 2 G FLOP per byte of a 16-bit
// cache.  On CUDA cores G = 8 would already need the whole fp32 rate; the legacy warp MMA (m16n8k16) has ten times the
// arithmetic this needs and, unlike tcgen05, takes its operands from registers, so nothing is staged:
//   * a warp works on tiles of 16 tokens, 32 where a row is 128 bytes or less.  S^T = K Q^T has the tokens as MMA rows and 8 query
//     heads as columns, O^T = V^T P^T the head's elements as rows and the 8 heads as columns: no row of an MMA is spent on
//     padding for G = 8.
//   * the order of the reduction index is free, so a lane's 16-byte loads of a key row ARE its operand fragments; for the
//     values, whose fragments pair two tokens, one byte permute per register pairs the words of two rows.
//   * keys of the next tile are requested when the scores are done, its values when the products are: 4 to 8 KB in
//     flight per warp, 8 to 16 warps per SM.
//   * S^T fragments become P^T fragments by one movmatrix each.
//   * the running maximum moves only when a score exceeds it by more than 2^8 (one vote per tile instead of six shuffles
//     and a rescaling); P stays below 2^8 in bf16, and is shifted by 2^7 in f16 to use that type's range.
// Work is cut on the device, where the lengths are: the steps (a tile for each of a CTA's warps, of one request and key-value head)
// of the whole batch are laid on a line and every CTA takes an equal run of it, so a batch of very different lengths is balanced
// and one long request fills the GPU.  A unit (request, head) also occupies what it costs to begin one (query, first
// page, empty pipeline, merge: as long as 48 or 96 KB of keys and values, or 384 tokens of E4M3; without that, CTAs with many
// short requests took twice the average and 32 requests of 1 to 8192 tokens 79 us), and a cut that falls near a unit's end is moved there.
// A CTA's warps (four, or one where short requests are many) are merged in shared memory; a unit that lies in one CTA is finished there, a unit that crosses
// CTAs leaves (m, l, O) of each part for the join kernel.
#pragma once
#include <cfloat>

#include "paged.cuh"
#include "pairs.cuh"

namespace cachalot {

constexpr int PA_THREADS = 128, PA_WARPS = 4;  // of a CTA; of one warp where short requests are many

struct AttendArgs {
  const void* q;
  long long q_row, q_head;  // elements
  int q_bf16;
  PagedView c;
  const int32_t* table;
  long long table_stride;
  int room;                        // tokens that a request's row of the table holds
  const int32_t* lens;
  int requests, heads, group;      // group: query heads per key-value head
  int tiles, head_blocks;          // head tiles (of 8 NT heads) a CTA's warps are split over; units per key-value head
  int page_shift;                  // log2(page_size / 8) or -1; tokens one by one where the page size is no multiple of 8
  uint64_t page_magic;             // ceil(2^35 / (page_size / 8)) for page sizes below 1024, else 0
  int one_warp;                    // CTAs of one warp (one head tile, pages of 8 k tokens)
  int unit_cost;                   // what beginning a unit costs, in steps
  float scale, softcap;
  int window;
  float* part_o;                   // [ctas][2][heads of a unit][dim]
  float2* part_ml;                 // [ctas][2][heads of a unit]
  int4* parts;                     // [ctas][2]: request, key-value head * head_blocks + block, first CTA, CTAs (0: none)
  void* out;
  int out_dtype;
  float* lse;
  int* status;
};

constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Soft cap, cap * tanh(z), z = x / cap, of two scores.  1 - 2 / (1 + e^2z) is off by 2^-21 whatever its size, which under a cap far
// above the scores would be more than they are; so up to 0.4 of the cap the Taylor series, five terms: what is left out is
// 0.009 z^10 < 2^-19.9 of the result.  Both forms 2^-18 of the result or better.  (Tiles without a score past the border leave out the second
// form; where most have one, 64 requests of up to 8192 tokens over E4M3 take 110 us instead of 101.)
constexpr float PA_CAP_NEAR = 0.4f;
__device__ __forceinline__ f32x2 capped_near(f32x2 x, f32x2 per_cap) {
  const f32x2 z = mul2(x, per_cap), z2 = mul2(z, z);
  f32x2 s = fma2(pair(62.f / 2835.f, 62.f / 2835.f), z2, pair(-17.f / 315.f, -17.f / 315.f));
  s = fma2(s, z2, pair(2.f / 15.f, 2.f / 15.f)), s = fma2(s, z2, pair(-1.f / 3.f, -1.f / 3.f));
  return fma2(x, mul2(s, z2), x);
}
__device__ __forceinline__ f32x2 capped_far(f32x2 x, f32x2 cap, f32x2 per_cap) {
  const float2 t = both(mul2(mul2(x, per_cap), pair(2.f * PA_LOG2E, 2.f * PA_LOG2E))), from = both(x);
  const float2 d = both(add2(pair(ex2(fabsf(t.x)), ex2(fabsf(t.y))), pair(1.f, 1.f)));
  const float2 y = both(mul2(cap, fma2(pair(-2.f, -2.f), pair(reciprocal(d.x), reciprocal(d.y)), pair(1.f, 1.f))));
  return pair(copysignf(y.x, from.x), copysignf(y.y, from.y));
}

template <typename M>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<M, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename M>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<M, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename M>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (std::is_same<M, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  else return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// two E4M3 codes, the low or the high half of `x` -> two f16
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t x) {
  uint32_t y;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t x) {
  uint32_t y;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(y) : "r"(x));
  return y;
}

// B bytes per load (16, 8 or 4), W words in all, loads STRIDE bytes apart
template <int B, int W, int STRIDE, bool KEEP>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const uint8_t* p) {
#pragma unroll
  for (int c = 0; c < W * 4 / B; ++c) {
    const uint8_t* at = p + c * STRIDE;
    if constexpr (B == 16) {
      const uint4 v = KEEP ? *reinterpret_cast<const uint4*>(at) : ld_once_u4(at);
      r[c * 4] = v.x, r[c * 4 + 1] = v.y, r[c * 4 + 2] = v.z, r[c * 4 + 3] = v.w;
    } else if constexpr (B == 8) {
      const uint2 v = KEEP ? *reinterpret_cast<const uint2*>(at) : ld_once_u2(at);
      r[c * 2] = v.x, r[c * 2 + 1] = v.y;
    } else {
      r[c] = KEEP ? *reinterpret_cast<const uint32_t*>(at) : ld_once_u32(at);
    }
  }
}

// Geometry of one instantiation: what a lane holds of a key row (a quarter of it) and of a value row (an eighth).
template <bool F8, int D, int NT, int W>
struct AttendShape {
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int KBYTES = D * ES / 4, VBYTES = D * ES / 8;
  static constexpr int KB = KBYTES % 16 == 0 ? 16 : 8;
  static constexpr int VB = VBYTES % 16 == 0 ? 16 : VBYTES % 8 == 0 ? 8 : 4;
  static constexpr int KW = KBYTES / 4, VW = VBYTES / 4;
  // MMA tiles of 16 tokens that a warp works on at a time.  (E4M3 with several column tiles: one tile and three CTAs per SM 141 us,
  // two and two 168 us, batch of 64 with 16 heads of 128 to a key-value head.)
  static constexpr int U = D * ES <= 128 && !(F8 && NT > 1 && D > 64) ? 2 : 1;
  static constexpr int TILE = 16 * U, STEP = W * TILE;
  static constexpr int KSTEPS = D / 16;                 // MMAs over the head's elements = MMA row tiles of O^T
  static constexpr int TILE_HEADS = 8 * NT;
  static constexpr int O_PITCH = D + 4;
  // element of the head at which lane quad t's key word w starts / lane row g's value word w
  static constexpr __host__ __device__ int k_dim(int w, int t) { return (w / (KB / 4) * (4 * KB) + t * KB + w % (KB / 4) * 4) / ES; }
  static constexpr __host__ __device__ int v_dim(int w, int g) { return (w / (VB / 4) * (8 * VB) + g * VB + w % (VB / 4) * 4) / ES; }
  static constexpr int Q_BYTES(int tiles) { return tiles * NT * KSTEPS * 32 * 8; }
  static constexpr int SMEM(int tiles) { return Q_BYTES(tiles) + W * TILE_HEADS * (O_PITCH * 4 + 8) + 4 * TILE_HEADS * 4; }
  static constexpr int MAX_TILES = 4;
  // CTAs per SM that the registers are cut for
  static constexpr int CTAS = PA_WARPS / W * (D * NT <= 64 ? 4 : D * NT <= 128 || (F8 && NT > 1 && D * NT <= 256) ? 3 : 2);
};

struct Span {  // what is visible of a request
  int lo, len, first_tile, steps;
};
template <typename S>
__device__ __forceinline__ Span span_of_length(const AttendArgs& a, int length) {
  Span s;
  s.len = min(max(length, 0), a.room);
  s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
  s.first_tile = s.lo / S::TILE;
  s.steps = s.len > 0 ? (s.len - s.first_tile * S::TILE + S::STEP - 1) / S::STEP : 0;
  return s;
}

template <typename S>
__device__ __forceinline__ Span span_of(const AttendArgs& a, int r) { return span_of_length<S>(a, a.lens[r]); }

// Division by a number that stays the same, of dividends below 2^53 (a 64-bit division takes a thousand cycles).
struct Divisor {
  long long d;
  double inverse;
  __device__ __forceinline__ explicit Divisor(long long by) : d(by), inverse(1.0 / (double)by) {}
  __device__ __forceinline__ long long of(long long x) const {
    const long long q = (long long)((double)x * inverse), rest = x - q * d;
    return rest < 0 ? q - 1 : rest >= d ? q + 1 : q;
  }
};

__device__ __forceinline__ void store_out(void* out, int dtype, long long at, float v) {
  if (dtype == CACHALOT_F32) static_cast<float*>(out)[at] = v;
  else if (dtype == CACHALOT_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[at] = __float2half_rn(v);
}
// ... of elements at .. at + 3, at a multiple of 4
__device__ __forceinline__ void store_out4(void* out, int dtype, long long at, float4 v) {
  const bool whole = ((uintptr_t)out & (dtype == CACHALOT_F32 ? 15 : 7)) == 0;
  if (!whole) {
    store_out(out, dtype, at, v.x), store_out(out, dtype, at + 1, v.y), store_out(out, dtype, at + 2, v.z), store_out(out, dtype, at + 3, v.w);
  } else if (dtype == CACHALOT_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
  } else {
    const uint2 w = dtype == CACHALOT_BF16 ? make_uint2(pack2<__nv_bfloat16>(v.x, v.y), pack2<__nv_bfloat16>(v.z, v.w))
                                           : make_uint2(pack2<__half>(v.x, v.y), pack2<__half>(v.z, v.w));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = w;
  }
}

// TERMS of P, of the matrix type: two keep 16 bits of a weight (bf16) or 22 (f16); one f16 term, 11 bits, over an E4M3 cache where
// the result is rounded to bf16 (error against 64 bits 1.67e-3 with one term, 1.66e-3 of the rounding alone; rounded to f16 2.8e-4 and 2.1e-4, so
// that takes two; they cost 64 requests of up to 8192 tokens, 8, 16 and 24 query heads of 128, 128 and 192 to a
// key-value head, 101 us instead of 97, 146 instead of 131, 299 instead of 271).
template <typename M, bool F8, int D, int NT, bool PAGE8, bool KEEP, int W, int TERMS>
__global__ void __launch_bounds__(W * 32, AttendShape<F8, D, NT, W>::CTAS) attend_kernel(const AttendArgs a) {
  using S = AttendShape<F8, D, NT, W>;
  constexpr bool HALF = std::is_same<M, __half>::value;
  constexpr float SHIFT = HALF ? 7.f : 0.f, SLACK = 8.f;
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* sq = reinterpret_cast<uint2*>(smem);                                        // [tiles * NT][KSTEPS][32]
  float* so = reinterpret_cast<float*>(smem + S::Q_BYTES(a.tiles));                  // [warps][TILE_HEADS][O_PITCH]
  float2* sml = reinterpret_cast<float2*>(so + W * S::TILE_HEADS * S::O_PITCH);  // [warps][TILE_HEADS]
  float* sexp = reinterpret_cast<float*>(sml + W * S::TILE_HEADS);            // [tiles * TILE_HEADS] scale of the query
  __shared__ long long sums[W];
  __shared__ long long shared_found_at;
  __shared__ int shared_found;

  wait_for_predecessor();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int per_request = a.c.kv_heads * a.head_blocks;
  int flags = 0;

  // ---- which part of the line is this CTA's ----
  auto cost_of = [&](int n) {  // of a request of n tokens
    if (n < 0 || n > a.room) flags |= CACHALOT_STATUS_LENGTH;
    const int steps = span_of_length<S>(a, n).steps;
    return steps ? (long long)(steps + a.unit_cost) * per_request : 0LL;
  };
  auto scan = [&](long long v) {  // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  int found = -1;  // the request that lies where the run begins, and where that request begins
  long long found_at = 0, total = 0, per, begin;
  auto cut = [&] {
    per = max(Divisor(gridDim.x).of(total + gridDim.x - 1), 1LL);
    begin = per * blockIdx.x;
  };
  if (a.requests <= 32) {  // every warp for itself
    const long long own = cost_of(lane < a.requests ? a.lens[lane] : 0), end = scan(own);
    total = __shfl_sync(0xffffffffu, end, 31);
    cut();
    const unsigned here = __ballot_sync(0xffffffffu, begin >= end - own && begin < end);
    if (here) found = __ffs(here) - 1, found_at = __shfl_sync(0xffffffffu, end - own, found);
  } else {
    // a thread has `each` requests in a row; eight loads at a time
    const int each = (a.requests + W * 32 - 1) / (W * 32), r0 = tid * each;
    long long own = 0;
    for (int i0 = 0; i0 < each; i0 += 8) {
      int n[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) n[i] = i0 + i < each && r0 + i0 + i < a.requests ? a.lens[r0 + i0 + i] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) own += cost_of(n[i]);
    }
    long long end = scan(own);
    if (lane == 31) sums[warp] = end;
    if (tid == 0) shared_found = -1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) total += sums[w], end += w < warp ? sums[w] : 0;
    cut();
    if (begin >= end - own && begin < end) {
      int r = r0;
      long long from = end - own;
      for (long long c; begin >= from + (c = cost_of(a.lens[r])); ++r) from += c;
      shared_found = r, shared_found_at = from;
    }
    __syncthreads();
    found = shared_found, found_at = shared_found_at;
  }
  if (tid < 2) a.parts[blockIdx.x * 2 + tid] = make_int4(0, 0, 0, 0);
  __syncthreads();
  const Divisor by_per(per);
  const int near_end = (int)max(min((long long)a.unit_cost, per / 4), 1LL);  // a cut is at least that many steps inside a unit

  const int mt = W == 1 ? 0 : warp % a.tiles, slice = W == 1 ? 0 : warp / a.tiles, slices = W == 1 ? 1 : W / a.tiles;
  const int unit_heads = a.tiles * S::TILE_HEADS;
  int r = max(found, 0);
  Span sp = span_of<S>(a, r);
  int unit = 0;
  if (found >= 0) unit = (int)Divisor(sp.steps + a.unit_cost).of(begin - found_at);
  long long at = found_at + (long long)unit * (sp.steps + a.unit_cost);  // where the unit begins on the line

  for (; found >= 0; at += sp.steps + a.unit_cost, ++unit) {
    if (unit == per_request) {
      unit = 0;
      do sp = ++r < a.requests ? span_of<S>(a, r) : Span{0, 0, 0, -1};
      while (sp.steps == 0);
      if (sp.steps < 0) break;
    }
    // the unit is cut where multiples of `per` fall among its steps, not within `inside` of either end: CTAs c0 .. c1
    const int inside = min(near_end, sp.steps);
    const long long cta = blockIdx.x, steps_at = at + a.unit_cost;
    const long long c0 = by_per.of(steps_at + inside - 1), c1 = max(c0, by_per.of(steps_at + sp.steps - inside));
    if (c0 > cta) break;
    if (c1 < cta) continue;  // this CTA's run begins so near the unit's end that another one does all of it
    const int step0 = cta == c0 ? 0 : (int)(cta * per - steps_at);
    const int steps = (cta == c1 ? sp.steps : (int)((cta + 1) * per - steps_at)) - step0;
    const int h = a.head_blocks == 1 ? unit : unit / a.head_blocks, block = a.head_blocks == 1 ? 0 : unit % a.head_blocks;
    const int head0 = block * unit_heads, heads = min(unit_heads, a.group - head0);  // within the group
    const long long row0 = (long long)r * a.heads + (long long)h * a.group + head0;  // first output row of the unit

    // ---- this warp's tiles ----
    const uint8_t* kbase = a.c.k + h * a.c.k_head + t4 * S::KB;
    const uint8_t* vbase = a.c.v + h * a.c.v_head + g * S::VB;
    const uint32_t k_page = (uint32_t)a.c.k_page, k_token = (uint32_t)a.c.k_token, v_page = (uint32_t)a.c.v_page, v_token = (uint32_t)a.c.v_token;
    const uint8_t *klane = kbase + (uint64_t)(uint32_t)g * k_token, *vlane = vbase + (uint64_t)(uint32_t)(2 * t4) * v_token;
    const int32_t* pages = a.table + r * a.table_stride;
    const int tile_end = min(sp.first_tile + (step0 + steps) * W, (sp.len + S::TILE - 1) / S::TILE);
    uint32_t kr[S::U][2][S::KW], vr[S::U][4][S::VW];

    // page of a token, -1 where the table names none of the cache's
    auto page_of = [&](int token, int index) {
      if (token >= sp.len) return -1;
      const int p = pages[index];
      if ((unsigned)p < (unsigned)a.c.n_pages) return p;
      flags |= CACHALOT_STATUS_SLOT_RANGE;
      return -1;
    };
    struct Place {  // where a tile lies: page and place in it of its pieces of 8 tokens (pages of 8 k tokens)
      int tile, page[2 * S::U], off[2 * S::U];
      bool full;
    };
    auto locate = [&](int tile) {
      Place p;
      p.tile = tile;
      p.full = tile * S::TILE >= sp.lo && (tile + 1) * S::TILE <= sp.len;
      if constexpr (PAGE8) {
#pragma unroll
        for (int i = 0; i < 2 * S::U; ++i) {
          const int token = tile * S::TILE + 8 * i;
          // token / 8 < 2^28 and page_size / 8 < 2^7, so the magic product is exact and fits 64 bits
          const int index = a.page_shift >= 0 ? (token >> 3) >> a.page_shift
                            : a.page_magic    ? (int)((uint64_t)(uint32_t)(token >> 3) * a.page_magic >> 35)
                                              : token / a.c.page_size;
          p.off[i] = token - index * a.c.page_size;
          p.page[i] = token + 8 <= sp.lo ? -1 : page_of(token, index);
          p.full = p.full && p.page[i] >= 0;
        }
      } else {
        p.full = false;
      }
      return p;
    };
    // place of token i of piece `piece` of a tile: true and its page and offset if it is visible
    auto token_at = [&](const Place& p, int piece, int i, int& page, int& off) {
      const int token = p.tile * S::TILE + piece * 8 + i;
      const bool ok = token >= sp.lo && token < sp.len;
      if constexpr (PAGE8) {
        page = p.page[piece], off = p.off[piece] + i;
        return ok && page >= 0;
      } else {
        if (!ok) return false;
        const int index = token / a.c.page_size;
        page = page_of(token, index), off = token - index * a.c.page_size;
        return page >= 0;
      }
    };
    int seen = 0;  // bit i: key row g of piece i of the tile in `kr` is visible
    auto load_k = [&](const Place& p) {
      seen = (1 << 2 * S::U) - 1;
      if (p.full) {
#pragma unroll
        for (int i = 0; i < 2 * S::U; ++i)
          load_words<S::KB, S::KW, 4 * S::KB, KEEP>(kr[i / 2][i % 2], klane + (uint64_t)(uint32_t)p.page[i] * k_page + (uint64_t)(uint32_t)p.off[i] * k_token);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * S::U; ++i) {
          int page, off;
          if (token_at(p, i, g, page, off)) {
            load_words<S::KB, S::KW, 4 * S::KB, KEEP>(kr[i / 2][i % 2], kbase + (uint64_t)(uint32_t)page * k_page + (uint64_t)(uint32_t)off * k_token);
          } else {
            seen &= ~(1 << i);
#pragma unroll
            for (int w = 0; w < S::KW; ++w) kr[i / 2][i % 2][w] = 0;
          }
        }
      }
    };
    auto load_v = [&](const Place& p) {  // rows 2 t4, 2 t4 + 1 of every piece; what is hidden must be zero, 0 * NaN is not
      if (p.full) {
#pragma unroll
        for (int i = 0; i < 2 * S::U; ++i) {
          const uint8_t* row = vlane + (uint64_t)(uint32_t)p.page[i] * v_page + (uint64_t)(uint32_t)p.off[i] * v_token;
          load_words<S::VB, S::VW, 8 * S::VB, KEEP>(vr[i / 2][i % 2 * 2], row);
          load_words<S::VB, S::VW, 8 * S::VB, KEEP>(vr[i / 2][i % 2 * 2 + 1], row + v_token);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4 * S::U; ++i) {
          int page, off;
          if (token_at(p, i / 2, 2 * t4 + i % 2, page, off)) {
            load_words<S::VB, S::VW, 8 * S::VB, KEEP>(vr[i / 4][i % 4], vbase + (uint64_t)(uint32_t)page * v_page + (uint64_t)(uint32_t)off * v_token);
          } else {
#pragma unroll
            for (int w = 0; w < S::VW; ++w) vr[i / 4][i % 4][w] = 0;
          }
        }
      }
    };

    int tile = sp.first_tile + step0 * W + slice;
    Place next;
    if (tile < tile_end) {  // on their way while the queries are laid out
      const Place p = locate(tile);
      load_k(p), load_v(p);
      if (tile + slices < tile_end) next = locate(tile + slices);
    }

    // ---- the query heads as MMA fragments ----
    if constexpr (F8) {  // f16 from here on: a bf16 head is brought into range by a power of two
      for (int i0 = warp; i0 < unit_heads; i0 += 4 * W) {  // four heads' loads at a time
        float top[4] = {};
        if (a.q_bf16) {
          uint32_t x[4][(D + 63) / 64];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = min(i0 + j * W, heads - 1);
            const uint16_t* q = static_cast<const uint16_t*>(a.q) + r * a.q_row + (long long)(h * a.group + head0 + i) * a.q_head;
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c) {
              const int d = c * 64 + 2 * lane;
              x[j][c] = d < D ? *reinterpret_cast<const uint32_t*>(q + d) : 0;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c)
              top[j] = fmaxf(top[j], fmaxf(fabsf(__uint_as_float(x[j][c] << 16)), fabsf(__uint_as_float(x[j][c] & 0xffff0000u))));
            top[j] = warp_max(top[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = (int)((__float_as_uint(top[j]) >> 23) & 255) - 127;
          if (lane == 0 && i0 + j * W < unit_heads) sexp[i0 + j * W] = top[j] > 0.f ? pow2f(max(-126, min(126, e))) : 1.f;
        }
      }
      __syncthreads();
    }
    // Several loads of a thread in flight: one at a time, 161 requests of 2 tokens with 52 heads took 25.8 us, not 20.8.
    constexpr int BATCH = NT * S::KSTEPS * PA_WARPS / W >= 16 ? 8 : (NT * S::KSTEPS + 1) / 2;
    for (int i0 = tid; i0 < a.tiles * NT * S::KSTEPS * 32; i0 += BATCH * W * 32) {
      uint2 f[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = i0 + j * W * 32, l = i & 31, ks = (i >> 5) % S::KSTEPS, head = (i >> 5) / S::KSTEPS * 8 + (l >> 2);
        const int d0 = F8 ? S::k_dim(ks, l & 3) : S::k_dim(2 * ks, l & 3), d1 = F8 ? d0 + 2 : S::k_dim(2 * ks + 1, l & 3);
        f[j] = make_uint2(0, 0);
        if (head < heads) {
          const uint16_t* q = static_cast<const uint16_t*>(a.q) + r * a.q_row + (long long)(h * a.group + head0 + head) * a.q_head;
          f[j].x = *reinterpret_cast<const uint32_t*>(q + d0), f[j].y = *reinterpret_cast<const uint32_t*>(q + d1);
        }
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = i0 + j * W * 32, head = (i >> 5) / S::KSTEPS * 8 + ((i & 31) >> 2);
        if (i >= a.tiles * NT * S::KSTEPS * 32) break;
        if (F8 && a.q_bf16) {
          const float inv = 1.f / sexp[head];  // a power of two
          f[j].x = pack2<__half>(__uint_as_float(f[j].x << 16) * inv, __uint_as_float(f[j].x & 0xffff0000u) * inv);
          f[j].y = pack2<__half>(__uint_as_float(f[j].y << 16) * inv, __uint_as_float(f[j].y & 0xffff0000u) * inv);
        }
        sq[i] = f[j];
      }
    }
    __syncthreads();

    // scores in units of log2
    float hs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float f = a.scale * PA_LOG2E;
        if constexpr (F8) f *= sexp[(mt * NT + n) * 8 + 2 * t4 + c] * (a.c.k_scale ? a.c.k_scale[h] : 1.f);
        hs[n][c] = f;
      }

    float o[S::KSTEPS][NT][4];
    float m[NT][2], base[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) m[n][c] = -INFINITY, base[n][c] = 0.f, l[n][c] = 0.f;
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[k][n][c] = 0.f;
    }
    const uint2* q = sq + mt * NT * S::KSTEPS * 32 + lane;
    for (; tile < tile_end; tile += slices) {
      const bool more = tile + slices < tile_end;
      float s[S::U][NT][4];
#pragma unroll
      for (int u = 0; u < S::U; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][n][c] = 0.f;
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k) {
        uint2 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = q[(n * S::KSTEPS + k) * 32];
#pragma unroll
        for (int u = 0; u < S::U; ++u) {
          uint32_t a0, a1, a2, a3;
          if constexpr (F8) {
            a0 = e4m3_lo(kr[u][0][k]), a1 = e4m3_lo(kr[u][1][k]), a2 = e4m3_hi(kr[u][0][k]), a3 = e4m3_hi(kr[u][1][k]);
          } else {
            a0 = kr[u][0][2 * k], a1 = kr[u][1][2 * k], a2 = kr[u][0][2 * k + 1], a3 = kr[u][1][2 * k + 1];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<M>(s[u][n], a0, a1, a2, a3, b[n].x, b[n].y);
        }
      }
      const int visible = seen;
      if (more) load_k(next);
#pragma unroll
      for (int u = 0; u < S::U; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][n][c] *= hs[n][c & 1];
      if (a.softcap > 0.f) {
        const float cap = fminf(a.softcap * PA_LOG2E, FLT_MAX), border = PA_CAP_NEAR * cap;
        float inverse;  // volatile: worked out here, not kept in a register from before the loop
        asm volatile("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(cap));
        inverse = fminf(inverse, FLT_MAX);
        const f32x2 per_cap = pair(inverse, inverse);
        bool far = false;
#pragma unroll
        for (int u = 0; u < S::U; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) far = far || !(fabsf(s[u][n][c]) < border);
        const bool both_forms = __any_sync(0xffffffffu, far);
        auto each = [&](auto also_far) {
#pragma unroll
          for (int u = 0; u < S::U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 4; c += 2) {
                const f32x2 x = pair(s[u][n][c], s[u][n][c + 1]);
                float2 y = both(capped_near(x, per_cap));
                if constexpr (decltype(also_far)::value) {
                  const float2 z = both(capped_far(x, pair(cap, cap), per_cap));
                  y.x = fabsf(s[u][n][c]) < border ? y.x : z.x, y.y = fabsf(s[u][n][c + 1]) < border ? y.y : z.y;
                }
                s[u][n][c] = y.x, s[u][n][c + 1] = y.y;
              }
        };
        if (both_forms) each(std::true_type{});
        else each(std::false_type{});
      }
      if (visible != (1 << 2 * S::U) - 1) {
#pragma unroll
        for (int u = 0; u < S::U; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[u][n][c] = visible >> (2 * u + (c >> 1)) & 1 ? s[u][n][c] : -INFINITY;
      }
      bool higher = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < S::U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) top[c & 1] = fmaxf(top[c & 1], s[u][n][c]);
        higher = higher || top[0] > m[n][0] + SLACK || top[1] > m[n][1] + SLACK;
      }
      if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < S::U; ++u) top = fmaxf(top, fmaxf(s[u][n][c], s[u][n][c + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(m[n][c], top);
            const float keep = now == -INFINITY ? 1.f : ex2(m[n][c] - now);  // m still -inf: 0
            m[n][c] = now, base[n][c] = now == -INFINITY ? 0.f : now - SHIFT;
            l[n][c] *= keep;
#pragma unroll
            for (int k = 0; k < S::KSTEPS; ++k) o[k][n][c] *= keep, o[k][n][c + 2] *= keep;
          }
      }
      uint32_t pb[S::U][NT][TERMS][2];
#pragma unroll
      for (int u = 0; u < S::U; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = ex2(s[u][n][c] - base[n][c & 1]);
          l[n][0] += p[0] + p[2], l[n][1] += p[1] + p[3];
#pragma unroll
          for (int i = 0; i < TERMS; ++i) {
            const uint32_t lo = pack2<M>(p[0], p[1]), hi = pack2<M>(p[2], p[3]);
            pb[u][n][i][0] = movmatrix(lo), pb[u][n][i][1] = movmatrix(hi);
            const float2 x = unpack2<M>(lo), y = unpack2<M>(hi);
            p[0] -= x.x, p[1] -= x.y, p[2] -= y.x, p[3] -= y.y;
          }
        }
#pragma unroll
      for (int u = 0; u < S::U; ++u)
#pragma unroll
        for (int w = 0; w < S::VW; ++w) {
          if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = __byte_perm(vr[u][0][w], vr[u][1][w], i ? 0x7362 : 0x5140), y = __byte_perm(vr[u][2][w], vr[u][3][w], i ? 0x7362 : 0x5140);
              const uint32_t a0 = e4m3_lo(x), a1 = e4m3_hi(x), a2 = e4m3_lo(y), a3 = e4m3_hi(y);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < TERMS; ++j) mma16816<M>(o[2 * w + i][n], a0, a1, a2, a3, pb[u][n][j][0], pb[u][n][j][1]);
            }
          } else {
            const uint32_t a0 = __byte_perm(vr[u][0][w], vr[u][1][w], 0x5410), a1 = __byte_perm(vr[u][0][w], vr[u][1][w], 0x7632);
            const uint32_t a2 = __byte_perm(vr[u][2][w], vr[u][3][w], 0x5410), a3 = __byte_perm(vr[u][2][w], vr[u][3][w], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < TERMS; ++i) mma16816<M>(o[w][n], a0, a1, a2, a3, pb[u][n][i][0], pb[u][n][i][1]);
          }
        }
      if (more) {
        load_v(next);
        if (tile + 2 * slices < tile_end) next = locate(tile + 2 * slices);
      }
    }

    // ---- the four warps' parts of this run ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
        if (g == 0) sml[warp * S::TILE_HEADS + n * 8 + 2 * t4 + c] = make_float2(m[n][c], l[n][c]);
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = n * 8 + 2 * t4 + c;
        float top = -INFINITY;
        for (int w = mt; w < W; w += a.tiles) top = fmaxf(top, sml[w * S::TILE_HEADS + row].x);
        const float f = m[n][c] == -INFINITY ? 0.f : ex2(m[n][c] - top);
        float* dst = so + (warp * S::TILE_HEADS + row) * S::O_PITCH;
#pragma unroll
        for (int w = 0; w < S::VW; ++w) {
          if constexpr (F8)
            *reinterpret_cast<float4*>(dst + S::v_dim(w, g)) =
                make_float4(o[2 * w][n][c] * f, o[2 * w][n][c + 2] * f, o[2 * w + 1][n][c] * f, o[2 * w + 1][n][c + 2] * f);
          else
            *reinterpret_cast<float2*>(dst + S::v_dim(w, g)) = make_float2(o[w][n][c] * f, o[w][n][c + 2] * f);
        }
      }
    __syncthreads();
    const bool whole = c0 == c1;
    const int which = cta == c0 ? 1 : 0;
    const long long slot = (long long)blockIdx.x * 2 + which;
    const float v_scale = F8 && a.c.v_scale ? a.c.v_scale[h] : 1.f;
    for (int i = tid; i < heads * (D / 4); i += W * 32) {
      const int head = i / (D / 4), d = i % (D / 4) * 4;
      const int row = head % S::TILE_HEADS, from = head / S::TILE_HEADS;
      float top = -INFINITY, sum = 0.f;
      for (int w = from; w < W; w += a.tiles) top = fmaxf(top, sml[w * S::TILE_HEADS + row].x);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = from; w < W; w += a.tiles) {
        const float2 ml = sml[w * S::TILE_HEADS + row];
        sum += ml.x == -INFINITY ? ml.y : ml.y * ex2(ml.x - top);  // no maximum: 0, or NaN where all its scores are
        const float4 x = *reinterpret_cast<const float4*>(so + (w * S::TILE_HEADS + row) * S::O_PITCH + d);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : v_scale / sum;
        const long long to = (row0 + head) * D + d;
        store_out4(a.out, a.out_dtype, to, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        if (d == 0 && a.lse) a.lse[row0 + head] = sum == 0.f ? -INFINITY : (top - SHIFT + log2f(sum)) * PA_LN2;
      } else {
        *reinterpret_cast<float4*>(a.part_o + (slot * unit_heads + head) * D + d) = v;
        if (d == 0) a.part_ml[slot * unit_heads + head] = make_float2(top, sum);
      }
    }
    if (!whole && tid == 0) a.parts[slot] = make_int4(r, unit, (int)c0, (int)(c1 - c0) + 1);
    __syncthreads();
  }

  // ---- rows without a visible key ----
  for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
    if (span_of<S>(a, r).steps) continue;
    for (int i = tid; i < a.heads * D; i += W * 32) store_out(a.out, a.out_dtype, (long long)r * a.heads * D + i, 0.f);
    if (a.lse)
      for (int i = tid; i < a.heads; i += W * 32) a.lse[(long long)r * a.heads + i] = -INFINITY;
  }
  if (a.status && flags) atomicOr(a.status, flags);
}

struct AttendLaunch {
  int unit_heads, tiles, head_blocks, ctas_per_sm, step;
};
// head tiles and units of a group of query heads
template <bool F8, int D, int NT>
AttendLaunch attend_shape(int group) {
  AttendLaunch l;
  const int need = (group + 8 * NT - 1) / (8 * NT);
  l.tiles = need >= 3 ? 4 : need;
  l.unit_heads = l.tiles * 8 * NT;
  l.head_blocks = (group + l.unit_heads - 1) / l.unit_heads;
  l.ctas_per_sm = AttendShape<F8, D, NT, PA_WARPS>::CTAS, l.step = AttendShape<F8, D, NT, PA_WARPS>::STEP;
  return l;
}
// Column tiles of 8 query heads per warp: as few warps as possible read the same keys, up to three tiles where the registers hold
// their sums; wider heads have fewer.  Each with both sides measured when it was chosen (loads of the queries have since been
// batched, which took 5 to 17 % off), E4M3, 64 requests of up to 8192 tokens, 8 key-value heads: 24 heads to each, of 192: 321 us with three
// tiles, 405 with two, 604 with one; of 256: 720, 471, 691.  16 heads to each, of 192: 225 with two, 323 with one; of 256: 244, 356.
// bf16, 32 requests, 16 heads to each, of 192: 181 with two, 205 with one; of 256: 390, 268.  24 heads of 128 to each of 2, up to 16384
// tokens: 121 with three in one warp, 178 with two in two.
template <bool F8, typename Fn>
bool attend_dispatch(int dim, int group, Fn&& fn) {
  auto go = [&](auto d, auto nt) { fn(d, nt, attend_shape<F8, decltype(d)::value, decltype(nt)::value>(group)); };
  using std::integral_constant;
  auto nt = [&](auto d) {
    if constexpr (decltype(d)::value <= 192 || F8) {
      const int two = (group + 15) / 16, three = (group + 23) / 24;  // warps
      if constexpr (decltype(d)::value <= (F8 ? 192 : 128))
        if (group > 16 && (three == 1 || (two > 2 && three == 2))) return go(d, integral_constant<int, 3>{});
      if (group > 8) return go(d, integral_constant<int, 2>{});
    }
    go(d, integral_constant<int, 1>{});
  };
  switch (dim) {
    case 64: nt(integral_constant<int, 64>{}); return true;
    case 96: nt(integral_constant<int, 96>{}); return true;
    case 128: nt(integral_constant<int, 128>{}); return true;
    case 192: nt(integral_constant<int, 192>{}); return true;
    case 256: nt(integral_constant<int, 256>{}); return true;
    default: return false;
  }
}

template <typename M, bool F8, int TERMS>
int launch_attend(AttendArgs& a, int dim, int ctas, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  attend_dispatch<F8>(dim, a.group, [&](auto d, auto nt, const AttendLaunch& l) {
    constexpr int D = decltype(d)::value, NT = decltype(nt)::value;
    auto run = [&](auto kern, auto warps) {
      constexpr int W = decltype(warps)::value;
      using S = AttendShape<F8, D, NT, W>;
      e = smem_optin_once(kern, S::SMEM(W == 1 ? 1 : S::MAX_TILES));
      if (e == cudaSuccess) e = launch_early(kern, dim3(ctas), W * 32, S::SMEM(l.tiles), stream, 1, a);
    };
    using std::integral_constant;
    constexpr auto all = integral_constant<int, PA_WARPS>{};
    const bool page8 = a.c.page_size % 8 == 0;
    if constexpr (NT <= 2)
      if (a.one_warp) return run(attend_kernel<M, F8, D, NT, true, false, 1, TERMS>, integral_constant<int, 1>{});
    if (page8 && l.tiles == 1) run(attend_kernel<M, F8, D, NT, true, false, PA_WARPS, TERMS>, all);
    else if (page8) run(attend_kernel<M, F8, D, NT, true, true, PA_WARPS, TERMS>, all);
    else run(attend_kernel<M, F8, D, NT, false, true, PA_WARPS, TERMS>, all);
  });
  if (e != cudaSuccess) return fail(CACHALOT_ECUDA, "paged_attention: %s", cudaGetErrorString(e));
  return check_launch("paged_attention");
}

int launch_attend_bf16(AttendArgs& a, int dim, int ctas, cudaStream_t stream);
int launch_attend_f16(AttendArgs& a, int dim, int ctas, cudaStream_t stream);
int launch_attend_e4m3(AttendArgs& a, int dim, int ctas, cudaStream_t stream);
int launch_attend_e4m3_two(AttendArgs& a, int dim, int ctas, cudaStream_t stream);

}  // namespace cachalot

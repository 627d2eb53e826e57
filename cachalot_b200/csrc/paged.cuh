// The paged key-value cache as the kernels see it, and the checks every entry point makes of a caller's descriptor.
#pragma once
#include "common.cuh"

namespace cachalot {

struct PagedView {
  uint8_t* k;
  uint8_t* v;
  const float* k_scale;  // null: 1
  const float* v_scale;
  long long k_page, k_head, k_token, v_page, v_head, v_token;  // strides in bytes
  int n_pages, page_size, kv_heads, head_dim, dtype;
};

inline int paged_elem_bytes(int dtype) { return dtype == CACHALOT_E4M3 ? 1 : 2; }

// Rows are read and written 16 bytes at a time: base, strides and rows are multiples of that.
inline int paged_view(const char* who, const cachalot_paged_kv* c, PagedView* p) {
  if (!c || !c->k || !c->v) return fail(CACHALOT_EINVAL, "%s: null cache", who);
  if (c->dtype != CACHALOT_F16 && c->dtype != CACHALOT_BF16 && c->dtype != CACHALOT_E4M3)
    return fail(CACHALOT_EINVAL, "%s: a cache holds float16, bfloat16 or E4M3", who);
  if (c->n_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0) return fail(CACHALOT_EINVAL, "%s: empty cache", who);
  if ((long long)c->n_pages * c->page_size > 0x7fffffffLL)
    return fail(CACHALOT_EUNSUPPORTED, "%s: %d pages of %d tokens are more than int32 slots can name", who, c->n_pages, c->page_size);
  const long long es = paged_elem_bytes(c->dtype);
  const int64_t strides[6] = {c->k_page_stride, c->k_head_stride, c->k_token_stride, c->v_page_stride, c->v_head_stride, c->v_token_stride};
  for (int64_t s : strides)
    if (s < 0 || (s * es) % 16) return fail(CACHALOT_EALIGN, "%s: cache strides must be non-negative multiples of 16 bytes", who);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || (c->head_dim * es) % 16) return fail(CACHALOT_EALIGN, "%s: cache rows need 16-byte alignment", who);
  p->k = static_cast<uint8_t*>(c->k), p->v = static_cast<uint8_t*>(c->v);
  p->k_scale = c->k_scale, p->v_scale = c->v_scale;
  p->k_page = c->k_page_stride * es, p->k_head = c->k_head_stride * es, p->k_token = c->k_token_stride * es;
  p->v_page = c->v_page_stride * es, p->v_head = c->v_head_stride * es, p->v_token = c->v_token_stride * es;
  p->n_pages = c->n_pages, p->page_size = c->page_size, p->kv_heads = c->kv_heads, p->head_dim = c->head_dim, p->dtype = c->dtype;
  return CACHALOT_OK;
}

}  // namespace cachalot

// The paged key-value cache as its kernels see it, and the host checks of a cache and of rows given by strides.
#pragma once
#include "common.h"

namespace lsattn {

struct CacheArgs {
  const uint16_t *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  const int32_t* table;
  int64_t table_stride;
  int num_pages, max_pages, page_log2;
};

inline int check_cache(const char* what, const lsurge_kv_cache* c, CacheArgs* a) {
  LSURGE_REQUIRE(c, "%s: null cache", what);
  LSURGE_REQUIRE(c->d == 64 || c->d == 128 || c->d == 256, "%s: head_dim %lld (64, 128 or 256)", what, (long long)c->d);
  LSURGE_REQUIRE(c->heads >= 1 && c->heads <= 65535, "%s: %lld key heads", what, (long long)c->heads);
  LSURGE_REQUIRE(c->num_pages >= 1 && c->num_pages < (1ll << 31) && c->max_pages >= 1 && c->max_pages < (1ll << 31) &&
                     c->table_stride >= c->max_pages,
                 "%s: num_pages=%lld max_pages=%lld table_stride=%lld", what, (long long)c->num_pages,
                 (long long)c->max_pages, (long long)c->table_stride);
  int lg = 3;
  while (lg < 12 && (1ll << lg) < c->page_size) ++lg;
  LSURGE_REQUIRE((1ll << lg) == c->page_size, "%s: page_size %lld (a power of two from 8 to 4096)", what,
                 (long long)c->page_size);
  LSURGE_REQUIRE(c->k && c->v && c->page_table && c->seq_lens, "%s: null pointer", what);
  LSURGE_REQUIRE(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0, "%s: the caches must be 16-byte aligned", what);
  for (const int64_t st : {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride, c->v_slot_stride,
                           c->v_head_stride})
    LSURGE_REQUIRE(st >= 0 && st < (1ll << 40) && st % 8 == 0,
                   "%s: cache stride %lld (elements; a multiple of 8 in [0, 2^40))", what, (long long)st);
  if (c->dtype != LSURGE_BF16 && c->dtype != LSURGE_F16) return lsurge::set_error(LSURGE_ERR_DTYPE, "%s: bf16 or f16", what);
  a->k = (const uint16_t*)c->k, a->v = (const uint16_t*)c->v;
  a->k_page = c->k_page_stride, a->k_slot = c->k_slot_stride, a->k_head = c->k_head_stride;
  a->v_page = c->v_page_stride, a->v_slot = c->v_slot_stride, a->v_head = c->v_head_stride;
  a->table = c->page_table, a->table_stride = c->table_stride;
  a->num_pages = (int)c->num_pages, a->max_pages = (int)c->max_pages, a->page_log2 = lg;
  return LSURGE_OK;
}
inline int check_new_rows(const char* what, const lsurge_attn_rows* r) {
  LSURGE_REQUIRE(r && r->data && (uintptr_t)r->data % 16 == 0, "%s: null or misaligned rows", what);
  LSURGE_REQUIRE(r->row_stride >= 0 && r->row_stride < (1ll << 40) && r->head_stride >= 0 && r->head_stride < (1ll << 40) &&
                     r->row_stride % 8 == 0 && r->head_stride % 8 == 0,
                 "%s: row and head strides (%lld, %lld elements) must be multiples of 8 in [0, 2^40)", what,
                 (long long)r->row_stride, (long long)r->head_stride);
  return LSURGE_OK;
}

}  // namespace lsattn

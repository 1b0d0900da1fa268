// The 4-bit paged cache as kernels see it; argument checks shared by its entry points.
#ifndef ITEXB_CSRC_KV4_H_
#define ITEXB_CSRC_KV4_H_

#include "decoder.h"

namespace itexb {

struct Kv4View {
  uint8_t* k_codes; __half2* k_params;
  uint8_t* v_codes; __half2* v_params;
  int64_t cp, ch, ct;   // bytes
  int64_t pp, ph, pt;   // pairs
  int num_pages, page_size, kv_heads, head_dim, group;
  FastDiv div_page;
};

inline int CheckKv4(const itexb_kv4_cache_t& c, const char* what, Kv4View* v) {
  ITEXB_REQUIRE(c.num_pages > 0 && c.page_size > 0 && c.kv_heads > 0, ITEXB_INVALID_ARGUMENT, "%s: bad cache shape", what);
  ITEXB_REQUIRE(int64_t(c.num_pages) * c.page_size < (int64_t(1) << 31), ITEXB_INVALID_ARGUMENT, "%s: 2^31 cache rows or more", what);
  ITEXB_REQUIRE(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, ITEXB_INVALID_ARGUMENT,
                "%s: head_dim must be 64, 128 or 256, got %d", what, c.head_dim);
  ITEXB_REQUIRE((c.group == 32 || c.group == 64 || c.group == 128) && c.group <= c.head_dim, ITEXB_INVALID_ARGUMENT,
                "%s: group must be 32, 64 or 128 and at most head_dim, got %d", what, c.group);
  ITEXB_REQUIRE(c.k_codes && c.k_params && c.v_codes && c.v_params, ITEXB_INVALID_ARGUMENT, "%s: NULL cache tensor", what);
  const uintptr_t codes = reinterpret_cast<uintptr_t>(c.k_codes) | reinterpret_cast<uintptr_t>(c.v_codes);
  ITEXB_REQUIRE(codes % 16 == 0 && c.codes_page_stride % 16 == 0 && c.codes_head_stride % 16 == 0 && c.codes_token_stride % 16 == 0,
                ITEXB_INVALID_ARGUMENT, "%s: the codes' rows must be 16-byte aligned", what);
  const int pairs = c.head_dim / c.group, align = pairs < 4 ? pairs : 4;
  const uintptr_t params = reinterpret_cast<uintptr_t>(c.k_params) | reinterpret_cast<uintptr_t>(c.v_params);
  ITEXB_REQUIRE(params % (4 * align) == 0 && c.params_page_stride % align == 0 && c.params_head_stride % align == 0 &&
                    c.params_token_stride % align == 0,
                ITEXB_INVALID_ARGUMENT, "%s: the params' rows must be aligned to %d bytes", what, 4 * align);
  v->k_codes = static_cast<uint8_t*>(c.k_codes);
  v->v_codes = static_cast<uint8_t*>(c.v_codes);
  v->k_params = static_cast<__half2*>(c.k_params);
  v->v_params = static_cast<__half2*>(c.v_params);
  v->cp = c.codes_page_stride; v->ch = c.codes_head_stride; v->ct = c.codes_token_stride;
  v->pp = c.params_page_stride; v->ph = c.params_head_stride; v->pt = c.params_token_stride;
  v->num_pages = c.num_pages; v->page_size = c.page_size; v->kv_heads = c.kv_heads;
  v->head_dim = c.head_dim; v->group = c.group;
  v->div_page = MakeFastDiv(uint32_t(c.page_size));
  return ITEXB_OK;
}

}  // namespace itexb

#endif  // ITEXB_CSRC_KV4_H_

// Host checks that the serving entry points share.
#pragma once
#include <cstdint>

#include "htree.h"

namespace htree {

struct Range {
  const void* at;
  int64_t bytes;
};
inline bool overlap(const Range& a, const Range& b) {
  const char *x = (const char*)a.at, *y = (const char*)b.at;
  return a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}
inline int cache_es(const htree_cache* c) { return c->dtype == HTREE_F32 ? 4 : 2; }

// sizes, types and alignment of the cache
inline int cache_check(const htree_cache* c) {
  if (!c) return HTREE_ENULL;
  if (c->dtype != HTREE_F32 && c->dtype != HTREE_BF16 && c->dtype != HTREE_F16) return HTREE_ESHAPE;
  if (c->H_kv <= 0 || c->Dk <= 0 || c->Dv <= 0 || c->num_pages <= 0) return HTREE_ESHAPE;
  if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1))) return HTREE_EUNSUPPORTED;
  const int es = cache_es(c);
  if (c->Dk > 256 || c->Dv > 256 || c->Dk * es % 16 || c->Dv * es % 16) return HTREE_EUNSUPPORTED;
  const int64_t st[6] = {c->k_page, c->k_token, c->k_head, c->v_page, c->v_token, c->v_head};
  for (int64_t s : st)
    if (s < 0 || s * es % 16) return HTREE_EUNSUPPORTED;
  // lanes hold 32-bit offsets into 16 tokens
  if (c->k_token * es > (1 << 26) || c->v_token * es > (1 << 26)) return HTREE_EUNSUPPORTED;
  return HTREE_OK;
}
inline bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }
inline int log2i(int x) { return __builtin_ctz((unsigned)x); }

}  // namespace htree

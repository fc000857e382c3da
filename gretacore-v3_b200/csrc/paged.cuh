// What the operators on paged caches share: where a sequence's rows and keys lie, and the checks of their arguments.
#pragma once
#include <cuda_bf16.h>

#include "greta_common.cuh"

namespace greta {

constexpr uint32_t PAGED_MAX_BATCH = 1024;

inline bool paged_float(int fmt) { return fmt == GRETA_FMT_F32 || fmt == GRETA_FMT_F16 || fmt == GRETA_FMT_BF16; }
inline uint32_t paged_size(int fmt) { return fmt == GRETA_FMT_F32 ? 4 : 2; }

inline int paged_check(const greta_paged_cache *c, const greta_ragged *r, const char *name) {
  GRETA_REQUIRE(c && r, "%s: null pointer", name);
  GRETA_REQUIRE(c->fmt == GRETA_FMT_F16 || c->fmt == GRETA_FMT_BF16, "%s: cache of format %d, not fp16 or bf16", name, c->fmt);
  GRETA_REQUIRE(c->k && c->v && c->table && r->start && r->len, "%s: null pointer", name);
  GRETA_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: the cache is not 16-byte aligned", name);
  GRETA_REQUIRE(c->dim >= 8 && c->dim <= 128 && c->dim % 8 == 0, "%s: heads of %u, not a multiple of 8 up to 128", name, c->dim);
  GRETA_REQUIRE(c->page >= 8 && c->page <= 256 && (c->page & (c->page - 1)) == 0, "%s: pages of %u rows, not a power of two from 8 to 256", name, c->page);
  GRETA_REQUIRE(c->pages && c->kv_heads && c->kv_heads <= 65535 && (uint64_t)c->pages * c->kv_heads * c->page < (1ull << 31),
                "%s: %u pages of %u heads and %u rows", name, c->pages, c->kv_heads, c->page);
  GRETA_REQUIRE(c->ld_table && (uint64_t)c->ld_table * c->page < (1ull << 31), "%s: tables of %u pages", name, c->ld_table);
  GRETA_REQUIRE(r->batch >= 1 && r->batch <= PAGED_MAX_BATCH, "%s: %u sequences, not 1 to %u", name, r->batch, PAGED_MAX_BATCH);
  GRETA_REQUIRE(r->tokens < (1u << 24), "%s: %u rows", name, r->tokens);
  return GRETA_OK;
}

// One sequence: `rows` rows of the token buffers from `first` on, the first of them at position pos0 (negative: it has none), `len` positions.
struct PagedSeq {
  uint32_t first, rows, len;
  int pos0;
};
__device__ __forceinline__ PagedSeq paged_seq(const greta_ragged &r, uint32_t max_len, uint32_t b) {
  PagedSeq s;
  s.first = min(__ldcg(r.start + b), r.tokens);
  const uint32_t end = min(__ldcg(r.start + b + 1), r.tokens);
  s.rows = end > s.first ? end - s.first : 0;
  s.len = min(__ldcg(r.len + b), max_len);
  s.pos0 = (int)s.len - (int)s.rows;
  if (r.max_rows) s.rows = min(s.rows, r.max_rows);
  return s;
}

}  // namespace greta

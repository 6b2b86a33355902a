// The paged key / value cache as the kernels that write and read it see it.
#pragma once

#include "capi.hpp"

namespace logo {

// Refuses what neither kernel takes.
inline int paged_check(const logo_paged_cache* c, int d) {
  LOGO_REQUIRE(c != nullptr, "null cache");
  LOGO_REQUIRE(d == 64 || d == 128, "head dim %d unsupported (64 or 128)", d);
  LOGO_REQUIRE(c->heads >= 1 && c->heads <= 65535, "bad head count");
  LOGO_REQUIRE(c->page_size >= 16 && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0,
               "page_size (%d) must be a power of two in [16, 65536]", c->page_size);
  LOGO_REQUIRE(c->nseq >= 0 && c->table_width >= 0 && c->pages >= 0 && c->table_row >= c->table_width,
               "bad sequence, table or page counts");
  LOGO_REQUIRE((int64_t)c->table_width * c->page_size < ((int64_t)1 << 31), "a sequence must stay below 2^31 keys");
  const int64_t strides[6] = {c->k_page, c->k_head, c->k_slot, c->v_page, c->v_head, c->v_slot};
  for (int64_t s : strides) LOGO_REQUIRE(s % 8 == 0 && s >= 0, "page strides must be multiples of 8 elements");
  // a page's rows are addressed by 32-bit byte offsets
  LOGO_REQUIRE(c->k_slot >= d && c->v_slot >= d && c->k_slot * c->page_size < ((int64_t)1 << 30) &&
                   c->v_slot * c->page_size < ((int64_t)1 << 30),
               "slots must hold a row, and a page stay below 2 GB");
  LOGO_REQUIRE(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0, "pages must be 16-byte aligned");
  LOGO_REQUIRE(c->pages == 0 || (c->k && c->v), "null pages");
  LOGO_REQUIRE(c->nseq == 0 || (c->cu && c->lens && (c->table || c->table_width == 0)), "null table, cu or lens");
  return LOGO_OK;
}

}  // namespace logo

// The paged 4-bit cache as kernels address it.
#pragma once

#include "types.cuh"

namespace modiff {

struct Kv4Pages {
  uint8_t *k_codes, *v_codes;      // [page][head][offset][dim / 2]
  uint16_t *k_params, *v_params;   // fp16 [page][head][offset][2]
  int pages, heads, page_size, dim;
  FastDiv by_page;
};

int kv4_check(const modiff_kv4_cache* c, const int32_t* table, const int32_t* lengths, int batch, int max_pages);
Kv4Pages kv4_pages(const modiff_kv4_cache* c);

#ifdef __CUDACC__
// Row of a token in the cache's arrays, or -1: a position outside the table or a page number outside
// the cache is never followed.
__device__ inline int64_t kv4_place(const Kv4Pages& c, const int32_t* table_row, int max_pages, int at, int head) {
  if (at < 0) return -1;
  int offset;
  const int slot = c.by_page.divmod(at, offset);
  if (slot >= max_pages) return -1;
  const int page = __ldg(table_row + slot);
  if (page < 0 || page >= c.pages) return -1;
  return ((int64_t)page * c.heads + head) * c.page_size + offset;
}
#endif

}  // namespace modiff

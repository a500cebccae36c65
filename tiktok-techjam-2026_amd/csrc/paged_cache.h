// Shared definitions of the kernels that read and write the paged cache of
// keys and values.
//
// Keys and values lie in pages: row r (of page_size, a power of two), head h of
// page p at p page_stride + h head_stride + r row_stride elements, the same for
// both.  Position x of a sequence is row x % page_size of the page that the
// sequence's block table names at x / page_size.
#pragma once

#include "f8_common.h"
#include "strided_rows.h"

namespace tjk {

struct Paged {
  char* k;
  char* v;
  int64_t page_bytes, head_bytes;
  uint32_t row_bytes;
  int pages;
  int shift;  // log2 page_size
};

inline Paged paged(const tjk_paged_cache& c) {
  int shift = 0;
  while ((1 << shift) < c.page_size) ++shift;
  return {static_cast<char*>(c.k), static_cast<char*>(c.v), 2 * c.page_stride, 2 * c.head_stride,
          (uint32_t)(2 * c.row_stride), (int)c.pages, shift};
}

// Status of a cache that an entry point `who` is given.
int check_cache(const char* who, const tjk_paged_cache* c, bool writes);
// Status of one that it writes, `layers` of them, besides: no two rows in one place.
int check_written(const char* who, const tjk_paged_cache* c, int layers, int64_t layer_stride);

// A page that a block table names, -1 if the cache holds no such page.
__device__ __forceinline__ int page_of(const int32_t* table_row, int at, int pages) {
  const int p = table_row[at];
  return (uint32_t)p < (uint32_t)pages ? p : -1;
}

}  // namespace tjk

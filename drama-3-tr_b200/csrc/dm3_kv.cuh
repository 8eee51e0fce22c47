// The paged key-value cache as the kernels see it (kv_cache.cu, attention.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace dm3 {

enum : uint32_t {
  STATUS_BAD_PAGE = 4u,  // a page id, row or position outside the cache or table was skipped
};

namespace kv {

struct Cache {
  void *k, *v;            // [pages][kv_heads][page_size][dim] bf16, or e4m3 codes
  int8_t *k_exp, *v_exp;  // [pages][kv_heads][page_size] exponents of an e4m3 cache, else null
  int64_t page_stride;    // elements from one page to the next
  int64_t exp_stride;
  int pages, page_size;
  const int32_t* table;   // [rows][per_row] page ids
  int64_t table_stride;
  int rows, per_row;
  uint32_t* status;       // one word, STATUS_BAD_PAGE
};

__device__ __forceinline__ void set_status(uint32_t* word, uint32_t bit) { atomicOr(word, bit); }

}  // namespace kv

// Whether the host arguments describe a cache that the kernels take; false with the error set.
bool kv_cache_ok(const kv::Cache& c, int kv_heads, int dim);

}  // namespace dm3

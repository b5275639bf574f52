// Where a position of a paged cache lies.
#pragma once

#include <stdint.h>

namespace i4 {

// A row of one kv head in the pool, from the page's number `id` as the table has it.
struct PageRows {
  int64_t at;  // of the row in k and v, in bytes
  bool bad;    // no such page: `at` is then that row of page 0, which there always is
};
// position j's, head g: pages of 2^shift rows of `row` bytes, strides in bytes
__host__ __device__ inline PageRows page_rows_of(int32_t id, int32_t pages, int64_t page_stride,
                                                 int64_t head_stride, int shift, int row, int g,
                                                 int j) {
  const bool bad = (uint32_t)id >= (uint32_t)pages;
  const int64_t page = bad ? 0 : id;
  return PageRows{page * page_stride + g * head_stride + (int64_t)(j & ((1 << shift) - 1)) * row,
                  bad};
}

}  // namespace i4

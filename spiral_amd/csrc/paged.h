// Where the rows of a sequence lie in a paged cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace spiral {

// Division of 32-bit numbers by a divisor known on the host: the high half of a
// product with floor((2^32 - 1) / d) is the quotient or one less.
struct Divisor {
  uint32_t d, inverse;
  __host__ __device__ explicit Divisor(uint32_t divisor) : d(divisor), inverse(0xffffffffu / divisor) {}
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    const uint32_t q = __umulhi(x, inverse);
    return x - q * d >= d ? q + 1 : q;
  }
};

struct PagedRows {
  const int32_t* table;  // the sequence's page ids
  uint32_t cols, pages;
  Divisor page;

  // Whether the table has an entry for position pos; the entry (a page id, valid below
  // `pages`), and the row of the page.
  __device__ __forceinline__ bool in_table(int64_t pos) const {
    return pos >= 0 && pos <= 0x7fffffff && page.quotient(static_cast<uint32_t>(pos)) < cols;
  }
  __device__ __forceinline__ uint32_t entry(int64_t pos) const {
    return static_cast<uint32_t>(table[page.quotient(static_cast<uint32_t>(pos))]);
  }
  __device__ __forceinline__ uint32_t row(int64_t pos) const {
    const uint32_t p = static_cast<uint32_t>(pos);
    return p - page.quotient(p) * page.d;
  }
};

}  // namespace spiral

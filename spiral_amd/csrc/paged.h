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

struct Place {
  bool ok;
  uint32_t page, row;
};

struct PagedRows {
  const int32_t* table;  // the sequence's page ids
  uint32_t cols, pages;
  Divisor page;

  // Position pos; ok is false where no row lies.
  __device__ __forceinline__ Place at(int64_t pos) const {
    Place p{pos >= 0 && pos <= 0x7fffffff, 0u, 0u};
    const uint32_t i = static_cast<uint32_t>(pos), col = page.quotient(i);
    p.ok = p.ok && col < cols;
    if (p.ok) p.page = static_cast<uint32_t>(table[col]);
    p.row = i - col * page.d;
    p.ok = p.ok && p.page < pages;  // a negative id is past every page
    return p;
  }
};

}  // namespace spiral

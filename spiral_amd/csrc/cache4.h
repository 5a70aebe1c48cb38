// Where things lie in a page of a cache in 4 bits (spiral_cache.h), and its codes.
#pragma once

#include "common.h"

namespace spiral {

// A cached head's block of a page: the codes of its rows, dim / 2 bytes a row, the even
// element of a pair in the low half of the byte, then the scale bytes of every 32
// elements, [dim / 32][page]. A page is a whole number of tiles of 16 rows, so a tile
// lies in one piece, rows and blocks at multiples of 16 bytes.
struct Block4 {
  uint32_t page, dim;
  __host__ __device__ uint32_t scales() const { return page * (dim / 2); }
  __host__ __device__ int64_t bytes() const { return static_cast<int64_t>(page) * (dim / 32) * 17; }
};

// Codes to pairs of a 16-bit type. The conversions take nothing but the exponent bits of
// their scale (every exponent checked under eight patterns of the other bits), so byte K
// of a word of scale bytes is in place after one shift; exponent 0 is 2^-127, 255 NaN.
template <int K>
__device__ __forceinline__ float scale_byte(uint32_t w) {
  return __uint_as_float(K == 0 ? w << 23 : K == 1 ? w << 15 : K == 2 ? w << 7 : w >> 1);
}

// The two codes of byte SEL of w times the scale, as a pair of E's type (tree.h).
template <typename E, int SEL>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  if constexpr (E::kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
  else
    return fp4_bf16x2<SEL>(w, scale);
}

// Magnitude codes from this one on are past the 16-bit type, which makes them infinities (8:
// none are, 0: the scale is NaN).
__device__ __forceinline__ uint32_t first_odd_code(uint32_t scale, bool f16) {
  if (scale == 255u) return 0u;
  const int32_t past = static_cast<int32_t>(scale) - (f16 ? 141 : 253);
  return past < 0 ? 8u : past == 0 ? 6u : past == 1 ? 4u : past == 2 ? 2u : 1u;
}

// Sizes that every call over a cache in 4 bits checks.
inline bool sizes4_ok(int64_t pages, int64_t page, int64_t kv_heads, int64_t dim, int64_t page_stride) {
  return pages >= 0 && pages <= INT32_MAX && page > 0 && page % 16 == 0 && page <= (1 << 20) && kv_heads > 0 &&
         kv_heads <= 65536 && dim > 0 && dim % 32 == 0 && dim <= 256 && page_stride % 16 == 0 &&
         page_stride >= kv_heads * Block4{static_cast<uint32_t>(page), static_cast<uint32_t>(dim)}.bytes() &&
         page_stride <= (int64_t(1) << 40);
}

}  // namespace spiral

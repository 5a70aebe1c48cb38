// MXFP4 (OCP microscaling, ggml's block_mxfp4): quantization of rows, and the
// products whose operands the hardware takes as they are.
//
// A block is 32 E2M1 codes under one E8M0 scale, value = code * 2^(e - 127).
//
// mxfp4_quantize_kernel: e = clamp(floor(log2(max |x|)) - 2, -127, 127), the
// largest scale at which the block's largest value still reaches the code range
// [4, 8); code = nearest E2M1 of x / 2^e, ties to the even code, magnitudes past
// 6 to 6. A block with a NaN or an infinity gets the scale byte 255 (NaN) and
// zero codes. Reads the rows once and writes 17 bytes a block; four lanes a
// block, lane p with elements 4p .. 4p + 3 and 16 + 4p .. + 3, so that a lane's
// four bytes of nibble pairs (j, 16 + j) are its own.
//
// mxfp4_stream_kernel: y[t][n] = sum_k x[t][k] W[n][k] for few rows t, x in bf16
// or MXFP4. Bound by the weight bytes. A wave owns 16 RF weight rows and a range
// of k: lane (r, g) = (l % 16, l / 16) loads block 4 st + g of row r, 16 bytes,
// which are its MFMA operand as they lie:
//  - x in MXFP4: v_mfma_scale_f32_16x16x128_f8f6f4 takes both blocks and scales.
//  - x in bf16: v_cvt_scalef32_pk_bf16_fp4 makes two exact bf16 weights of a
//    byte, four v_mfma_f32_16x16x32_bf16 a step; the byte's two nibbles are
//    elements 16 apart, so x is zipped to match (four v_perm_b32).
// The waves of a workgroup that share rows split k and join their sums through
// LDS in a fixed order.
// Measured, 14336 x 4096 (31 MB): one bf16 row 11.9 us, 2.6 TB/s, bound by the loads of
// x beside a single batch of the wave's weight loads; one MXFP4 row 9.0 us, 3.5 TB/s.
// Quantization of 2047 x 14336 F32: 22.8 us, 5.8 TB/s.
#include <algorithm>

#include "common.h"
#include "dequant_impl.h"

namespace spiral {

// The product of many rows (gemm_mxfp4.hip).
bool mxfp4_gemm_fits(int64_t m, int64_t n_rows, int64_t nb);
int64_t mxfp4_gemm_workspace(int64_t m, int64_t n_rows, int64_t nb);
int mxfp4_gemm(const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int y_type, int64_t ldy,
               void* workspace, int64_t workspace_bytes, hipStream_t s);

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;

// ---- quantization -------------------------------------------------------------

// Maximum over the four lanes of a quad.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, false)));
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, false)));
}

template <int TYPE>
__device__ __forceinline__ f32x4_t load4(const void* p) {
  if constexpr (TYPE == SPIRAL_TYPE_F32) {
    return *static_cast<const f32x4_t*>(p);
  } else if constexpr (TYPE == SPIRAL_TYPE_BF16) {
    const uint2 v = *static_cast<const uint2*>(p);
    return f32x4_t{bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)};
  } else {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 v = *static_cast<const h4*>(p);
    return f32x4_t{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]),
                   static_cast<float>(v[3])};
  }
}

// Thread i: lane p = i % 4 of block i / 4 (blocks row after row).
template <int TYPE>
__global__ void __launch_bounds__(256) mxfp4_quantize_kernel(const uint8_t* __restrict__ x, int64_t row_bytes,
                                                             int64_t blocks, uint32_t nb, uint8_t* __restrict__ out) {
  constexpr int kSize = TYPE == SPIRAL_TYPE_F32 ? 4 : 2;
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x >> 2);
  if (b >= blocks) return;  // whole quads
  const uint32_t p = threadIdx.x & 3u;
  const int64_t row = b / nb;
  const uint8_t* src = x + row * row_bytes + ((b - row * nb) * 32 + 4 * p) * kSize;
  const f32x4_t lo = load4<TYPE>(src), hi = load4<TYPE>(src + 16 * kSize);
  // Magnitudes order as their bits do, NaN and infinity above every number.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = max(top, max(__float_as_uint(lo[i]) & 0x7fffffffu, __float_as_uint(hi[i]) & 0x7fffffffu));
  top = quad_max(top) >> 23;  // exponent field: floor(log2) + 127
  const uint32_t e = top == 255u ? 255u : top < 2u ? 0u : top - 2u;
  const float s = e8m0_scale(e);
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, lo[0], hi[0], s, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, lo[1], hi[1], s, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, lo[2], hi[2], s, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, lo[3], hi[3], s, 3);
  reinterpret_cast<uint32_t*>(out)[4 * b + p] = e == 255u ? 0u : q;
  if (p == 0) out[16 * blocks + b] = static_cast<uint8_t>(e);
}

// ---- few rows -------------------------------------------------------------------

constexpr int kWaves = 8;

// Rows of x as the kernel takes them: bf16 rows of stride ld elements, or the
// code and scale planes of an MXFP4 matrix.
struct Rows {
  const uint8_t* p;
  const uint8_t* scale;
  int64_t ld;
};

// One step (128 elements) of 16 rows of x.
template <bool X4>
struct XStep;
template <>
struct XStep<true> {
  uint4 q;
  __device__ __forceinline__ void load(const Rows& x, int64_t t, uint32_t nb, uint32_t b) {
    q = *reinterpret_cast<const uint4*>(x.p + (t * nb + b) * 16);
  }
  __device__ __forceinline__ void zero() { q = make_uint4(0u, 0u, 0u, 0u); }
};
template <>
struct XStep<false> {
  uint4 v[4];
  __device__ __forceinline__ void load(const Rows& x, int64_t t, uint32_t, uint32_t b) {
    const uint4* src = reinterpret_cast<const uint4*>(x.p + (t * x.ld + 32 * static_cast<int64_t>(b)) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = src[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // MFMA s: elements 4s + i and 16 + 4s + i, zipped.
  __device__ __forceinline__ bf16x8_t zip(int s) const {
    const uint4 a = v[s >> 1], b = v[2 + (s >> 1)];
    const uint32_t a0 = s & 1 ? a.z : a.x, a1 = s & 1 ? a.w : a.y, b0 = s & 1 ? b.z : b.x, b1 = s & 1 ? b.w : b.y;
    return __builtin_bit_cast(
        bf16x8_t, make_uint4(__builtin_amdgcn_perm(b0, a0, 0x05040100u), __builtin_amdgcn_perm(b0, a0, 0x07060302u),
                             __builtin_amdgcn_perm(b1, a1, 0x05040100u), __builtin_amdgcn_perm(b1, a1, 0x07060302u)));
  }
};

// Scale bytes of 16 consecutive blocks of a row, from block b0 on (16 bytes at any
// alignment, one load instead of one a step: a step's load of single bytes asks for as
// many cache lines as its codes). Near the end of a row the 16 bytes end with it, and
// blocks past it get any of them. SHORT: rows of fewer blocks, byte by byte.
template <bool SHORT>
struct Scales16 {
  u32x4_t v;
  uint32_t skip;  // block b0's place among them
  __device__ __forceinline__ void load(const uint8_t* row, uint32_t b0, uint32_t nb) {
    if constexpr (SHORT) {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        w[i / 4] |= static_cast<uint32_t>(row[min(b0 + i, nb - 1)]) << (8 * (i % 4));
      v = u32x4_t{w[0], w[1], w[2], w[3]};
      skip = 0;
    } else {
      const uint32_t at = min(b0, nb - 16);
      __builtin_memcpy(&v, row + at, 16);
      skip = b0 - at;
    }
  }
  // Byte of block b0 + 4 u + g.
  __device__ __forceinline__ uint32_t at(uint32_t u, uint32_t g) const {
    if (skip == 0) return v[u] >> (8 * g) & 0xffu;
    const uint32_t i = min(skip + 4 * u + g, 15u), w = i < 8 ? (i < 4 ? v[0] : v[1]) : (i < 12 ? v[2] : v[3]);
    return w >> (8 * (i & 3u)) & 0xffu;
  }
};

__device__ __forceinline__ f32x4_t mfma_fp4(const uint4& a, uint32_t ea, const uint4& b, uint32_t eb, f32x4_t c) {
  const i32x8_t av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w)};
  const i32x8_t bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w)};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, static_cast<int>(ea), 0,
                                                          static_cast<int>(eb));
}

// Four consecutive outputs v of row t of y, from column n on (those past n_rows dropped).
template <bool F32_OUT>
__device__ __forceinline__ void store4(void* y, int64_t ldy, int64_t t, int64_t n, int64_t n_rows, const f32x4_t& v) {
  if constexpr (F32_OUT) {
    float* dst = static_cast<float*>(y) + t * ldy + n;
    if (n + 4 <= n_rows && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
      *reinterpret_cast<f32x4_t*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < n_rows) dst[e] = v[e];
    }
  } else {
    uint16_t* dst = static_cast<uint16_t*>(y) + t * ldy + n;
    const uint32_t w[2] = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    if (n + 4 <= n_rows && (reinterpret_cast<uintptr_t>(dst) & 7u) == 0) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < n_rows) dst[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// kw waves share a row group and split its k steps; blockIdx.y takes 16 TB rows
// of x. Rows of x past m and blocks past the end of a row multiply as zeros, weight
// rows past n_rows repeat the last one.
template <bool X4, int RF, int TB, bool F32_OUT, bool SHORT>
__global__ void __launch_bounds__(64 * kWaves)
    mxfp4_stream_kernel(const uint8_t* __restrict__ w, int64_t n_rows, uint32_t nb, Rows x, int64_t m,
                        void* __restrict__ y, int64_t ldy, uint32_t kw) {
  __shared__ f32x4_t part[kWaves * RF * TB * 64];
  constexpr int U = 4;  // steps whose loads are in flight together
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t kp = wave % kw, groups = kWaves / kw;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * groups + wave / kw) * (16 * RF);
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * (16 * TB);
  const uint32_t steps = (nb + 3) / 4;
  const uint32_t s0 = steps * kp / kw, s1 = steps * (kp + 1) / kw;
  const uint8_t* scales = w + n_rows * nb * 16;
  int64_t wrow[RF], t[TB];
#pragma unroll
  for (int i = 0; i < RF; ++i) wrow[i] = min(n0 + 16 * i + r, n_rows - 1) * nb;
#pragma unroll
  for (int j = 0; j < TB; ++j) t[j] = min(t0 + 16 * j + r, m - 1);

  f32x4_t acc[RF][TB];
#pragma unroll
  for (int i = 0; i < RF; ++i)
#pragma unroll
    for (int j = 0; j < TB; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  for (uint32_t s = s0; s < s1; s += U) {
    uint4 wq[U][RF];
    XStep<X4> xs[U][TB];
    Scales16<SHORT> we[RF], xe[X4 ? TB : 1];
#pragma unroll
    for (int i = 0; i < RF; ++i) we[i].load(scales + wrow[i], 4 * s, nb);
    if constexpr (X4) {
#pragma unroll
      for (int j = 0; j < TB; ++j) xe[j].load(x.scale + t[j] * nb, 4 * s, nb);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t b = min(4 * min(s + u, s1 - 1) + g, nb - 1);
#pragma unroll
      for (int i = 0; i < RF; ++i) wq[u][i] = load_stream16(w + (wrow[i] + b) * 16);
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        if (t0 + 16 * j + r < m)
          xs[u][j].load(x, t[j], nb, b);
        else
          xs[u][j].zero();
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) break;
      uint32_t ew[RF], ex[TB];
#pragma unroll
      for (int i = 0; i < RF; ++i) ew[i] = we[i].at(u, g);
#pragma unroll
      for (int j = 0; j < TB; ++j) ex[j] = X4 ? xe[X4 ? j : 0].at(u, g) : 127u;
      if (4 * (s + u) + 4 > nb && 4 * (s + u) + g >= nb) {  // the last step's blocks past the row
#pragma unroll
        for (int i = 0; i < RF; ++i) wq[u][i] = make_uint4(0u, 0u, 0u, 0u), ew[i] = 127u;
#pragma unroll
        for (int j = 0; j < TB; ++j) xs[u][j].zero(), ex[j] = 127u;
      }
      if constexpr (X4) {
#pragma unroll
        for (int i = 0; i < RF; ++i)
#pragma unroll
          for (int j = 0; j < TB; ++j)
            acc[i][j] = mfma_fp4(wq[u][i], ew[i], xs[u][j].q, ex[j], acc[i][j]);
      } else {
        float sc[RF];
#pragma unroll
        for (int i = 0; i < RF; ++i) sc[i] = e8m0_scale(ew[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          bf16x8_t xb[TB];
#pragma unroll
          for (int j = 0; j < TB; ++j) xb[j] = xs[u][j].zip(q);
#pragma unroll
          for (int i = 0; i < RF; ++i) {
            const uint4& c = wq[u][i];
            const uint32_t v = q == 0 ? c.x : q == 1 ? c.y : q == 2 ? c.z : c.w;
            const bf16x8_t wb = __builtin_bit_cast(
                bf16x8_t, make_uint4(fp4_bf16x2<0>(v, sc[i]), fp4_bf16x2<1>(v, sc[i]), fp4_bf16x2<2>(v, sc[i]),
                                     fp4_bf16x2<3>(v, sc[i])));
#pragma unroll
            for (int j = 0; j < TB; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, xb[j], acc[i][j], 0, 0, 0);
          }
        }
      }
    }
  }

  // Lane (r, g) holds row t0 + 16 j + r of y, columns n0 + 16 i + 4 g .. + 3.
#pragma unroll
  for (int i = 0; i < RF; ++i)
#pragma unroll
    for (int j = 0; j < TB; ++j) part[(wave * RF * TB + i * TB + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (uint32_t f = wave; f < groups * RF * TB; f += kWaves) {
    const uint32_t grp = f / (RF * TB), ij = f % (RF * TB), i = ij / TB, j = ij % TB;
    f32x4_t sum = part[(grp * kw * RF * TB + ij) * 64 + lane];
    for (uint32_t q = 1; q < kw; ++q) sum += part[((grp * kw + q) * RF * TB + ij) * 64 + lane];
    const int64_t row = t0 + 16 * j + r;
    const int64_t n = (static_cast<int64_t>(blockIdx.x) * groups + grp) * (16 * RF) + 16 * i + 4 * g;
    if (row < m && n < n_rows) store4<F32_OUT>(y, ldy, row, n, n_rows, sum);
  }
}

// Waves that share the k steps of a row: two steps each at least.
uint32_t waves_of_a_row(int64_t nb) {
  const int64_t steps = ceil_div(nb, 4);
  uint32_t kw = kWaves;
  while (kw > 1 && kw * 2 > steps) kw /= 2;
  return kw;
}

template <bool X4, int RF, int TB>
int launch_stream(const void* w, int64_t n_rows, int64_t nb, const Rows& x, int64_t m, void* y, int y_type,
                  int64_t ldy, hipStream_t s) {
  const uint32_t kw = waves_of_a_row(nb);
  const int64_t bx = ceil_div(n_rows, 16 * RF * (kWaves / kw)), by = ceil_div(m, 16 * TB);
  if (bx > INT32_MAX || by > 65535) return SPIRAL_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  const uint8_t* W = static_cast<const uint8_t*>(w);
  const bool f32 = y_type == SPIRAL_TYPE_F32;
#define SPIRAL_STREAM(F32, SHORT)                                                                                 \
  hipLaunchKernelGGL((mxfp4_stream_kernel<X4, RF, TB, F32, SHORT>), grid, dim3(64 * kWaves), 0, s, W, n_rows,      \
                     static_cast<uint32_t>(nb), x, m, y, ldy, kw)
  if (nb < 16) {
    if (f32)
      SPIRAL_STREAM(true, true);
    else
      SPIRAL_STREAM(false, true);
  } else if (f32) {
    SPIRAL_STREAM(true, false);
  } else {
    SPIRAL_STREAM(false, false);
  }
#undef SPIRAL_STREAM
  return launch_status();
}

// Up to 16 rows. A wave's x serves two groups of weight rows where these still give
// every CU one and a half workgroups: 14336 x 4096, five bf16 rows 14.6 -> 12.9 us;
// 4096 x 14336, half a workgroup a CU, 12.3 -> 18.9 for one row.
template <bool X4>
int launch_few(const void* w, int64_t n_rows, int64_t nb, const Rows& x, int64_t m, void* y, int y_type, int64_t ldy,
               hipStream_t s) {
  if (ceil_div(n_rows, 32 * (kWaves / waves_of_a_row(nb))) * 2 >= 3 * device_cu_count())
    return launch_stream<X4, 2, 1>(w, n_rows, nb, x, m, y, y_type, ldy, s);
  return launch_stream<X4, 1, 1>(w, n_rows, nb, x, m, y, y_type, ldy, s);
}

}  // namespace

// The weight-only product of up to 16 rows; arguments validated by the caller.
bool mxfp4_stream_fits(int64_t m) { return m <= 16; }

int mxfp4_stream(const void* w, int64_t n_rows, int64_t k, const uint16_t* x, int64_t ldx, int64_t m, void* y,
                 int y_type, int64_t ldy, hipStream_t s) {
  const Rows rows{reinterpret_cast<const uint8_t*>(x), nullptr, ldx};
  return launch_few<false>(w, n_rows, k / 32, rows, m, y, y_type, ldy, s);
}

static bool mul_mat_sizes_ok(int64_t n_rows, int64_t k, int64_t m, int64_t ldy) {
  int64_t span = 0;
  return n_rows > 0 && m > 0 && k > 0 && k % kMXFP4Elems == 0 && k / kMXFP4Elems <= INT32_MAX / 4 && ldy >= n_rows &&
         !__builtin_mul_overflow(m, ldy, &span) && span <= INT64_MAX / 4 &&
         spiral_tensor_bytes(SPIRAL_TYPE_MXFP4, n_rows, k) != 0 && spiral_tensor_bytes(SPIRAL_TYPE_MXFP4, m, k) != 0;
}

}  // namespace spiral

using namespace spiral;

extern "C" {

int spiral_mxfp4_quantize(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t k, void* out, void* stream) {
  if (x_type != SPIRAL_TYPE_F32 && x_type != SPIRAL_TYPE_F16 && x_type != SPIRAL_TYPE_BF16) return SPIRAL_ERR_TYPE;
  int64_t span = 0;
  if (rows < 0 || k <= 0 || k % kMXFP4Elems != 0 || ldx < k || __builtin_mul_overflow(rows, ldx, &span) ||
      span > INT64_MAX / 8)
    return SPIRAL_ERR_SHAPE;
  if (rows == 0) return SPIRAL_OK;
  if (x == nullptr || out == nullptr) return SPIRAL_ERR_NULL;
  if (!aligned16(x) || !aligned16(out) || ldx % 8 != 0) return SPIRAL_ERR_ALIGN;
  const int64_t nb = k / kMXFP4Elems, blocks = rows * nb, wgs = ceil_div(blocks, 64);
  if (wgs > INT32_MAX || nb > UINT32_MAX) return SPIRAL_ERR_SHAPE;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const dim3 grid(static_cast<unsigned>(wgs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint8_t* X = static_cast<const uint8_t*>(x);
  uint8_t* o = static_cast<uint8_t*>(out);
#define SPIRAL_QUANTIZE(T, SIZE)                                                                            \
  hipLaunchKernelGGL(mxfp4_quantize_kernel<T>, grid, dim3(256), 0, s, X, ldx * SIZE, blocks, \
                     static_cast<uint32_t>(nb), o)
  if (x_type == SPIRAL_TYPE_F32)
    SPIRAL_QUANTIZE(SPIRAL_TYPE_F32, 4);
  else if (x_type == SPIRAL_TYPE_F16)
    SPIRAL_QUANTIZE(SPIRAL_TYPE_F16, 2);
  else
    SPIRAL_QUANTIZE(SPIRAL_TYPE_BF16, 2);
#undef SPIRAL_QUANTIZE
  return launch_status();
}

int64_t spiral_mxfp4_mul_mat_workspace_bytes(int64_t n_rows, int64_t k, int64_t m) {
  if (!mul_mat_sizes_ok(n_rows, k, m, n_rows) || !mxfp4_gemm_fits(m, n_rows, k / kMXFP4Elems)) return 0;
  return mxfp4_gemm_workspace(m, n_rows, k / kMXFP4Elems);
}

int spiral_mxfp4_mul_mat(const void* w, int64_t n_rows, int64_t k, const void* x, int64_t m, void* y, int y_type,
                         int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream) {
  if (y_type != SPIRAL_TYPE_BF16 && y_type != SPIRAL_TYPE_F32) return SPIRAL_ERR_TYPE;
  if (w == nullptr || x == nullptr || y == nullptr) return SPIRAL_ERR_NULL;
  if (!mul_mat_sizes_ok(n_rows, k, m, ldy) || workspace_bytes < 0) return SPIRAL_ERR_SHAPE;
  if (!aligned16(w) || !aligned16(x) || !aligned16(workspace)) return SPIRAL_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(y) & (y_type == SPIRAL_TYPE_F32 ? 3u : 1u)) != 0) return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t nb = k / kMXFP4Elems;
  const uint8_t* X = static_cast<const uint8_t*>(x);
  const Rows rows{X, X + m * nb * 16, 0};
  if (m <= 16) return launch_few<true>(w, n_rows, nb, rows, m, y, y_type, ldy, s);
  if (mxfp4_gemm_fits(m, n_rows, nb))
    return mxfp4_gemm(X, m, static_cast<const uint8_t*>(w), n_rows, nb, y, y_type, ldy, workspace,
                      workspace == nullptr ? 0 : workspace_bytes, s);
  return launch_stream<true, 2, 4>(w, n_rows, nb, rows, m, y, y_type, ldy, s);
}

}  // extern "C"

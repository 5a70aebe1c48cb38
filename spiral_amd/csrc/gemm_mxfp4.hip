// Products of two MXFP4 matrices with many rows: Y[m][n] = sum_k X[m][k] W[n][k],
// codes and scales as they lie in the planar layout.
//
// One workgroup of 8 waves per BM x BN tile (BM = 64 MF, BN = 32 NF), k steps of 256
// (8 blocks, 128 bytes of codes a row). v_mfma_scale_f32_16x16x128_f8f6f4 multiplies
// four blocks of 16 rows of W and 16 rows of X: lane (r, g) gives block g of row r,
// its 16 code bytes and its scale byte, so that operands need no decoding.
//  - Codes go straight to LDS (buffer loads, 1 KiB an instruction: 8 rows of 128
//    bytes). The 16-byte chunks of a row are stored permuted (chunk c of row r at
//    c ^ (r / 2 % 8)) so that the operand reads, 16 rows x one chunk, touch every
//    bank once.
//  - Scales, 8 bytes a row and step at any alignment (a row has k / 32 of them),
//    pass through a register of the thread that owns the row, a step ahead.
//    Blocks past the end of a row get scale bytes 0 on both sides: whatever codes
//    the loads brought for them, 2^-127 times 2^-127 times 36 is no fp32 number.
//  - A step's two halves have an operand register set each: one is read from LDS
//    while the other multiplies. The barrier lies between them, when a wave holds
//    all of the step's operands, and both publishes the next stage and frees this one.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "dequant_impl.h"

namespace spiral {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;

constexpr int kThreads = 512;
constexpr int kStepBlocks = 8, kRowBytes = kStepBlocks * 16;
constexpr int kWaitLds = 0xC07F;  // s_waitcnt lgkmcnt(0)

// Tile index for workgroup b: consecutive workgroups go to consecutive XCDs, so
// XCD x gets a contiguous range of the tile order (the first `grid % 8` one more).
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t grid) {
  const uint32_t x = b & 7u, q = grid >> 3, r = grid & 7u;
  return x * q + (x < r ? x : r) + (b >> 3);
}

// Bytes of an X and a W stage of codes, how many of each LDS holds, and two stages
// of scales.
constexpr int kLdsBytes = 160 * 1024;
template <int MF, int NF>
struct Stages {
  static constexpr int kX = 64 * MF * kRowBytes, kW = 64 * ((NF + 1) / 2) * kRowBytes;
  static constexpr int kS = (64 * MF + 32 * NF) * kStepBlocks;
  static constexpr int kRoom = kLdsBytes - 2 * kS;
  static constexpr int kNX = 3 * (kX + kW) <= kRoom ? 3 : 2;
  static constexpr int kNW = kNX * kX + 3 * kW <= kRoom ? 3 : 2;
  static constexpr int kScales = kNX * kX + kNW * kW;
  static constexpr int kBytes = kScales + 2 * kS;
};

// Scheduling of one half: the loads, then the LDS reads, spread over the MFMAs, so
// that neither queue blocks the wave's issue while the matrix core idles.
template <int MFMAS, int READS, int LOADS>
__device__ __forceinline__ void interleave() {
  constexpr int kMfma = 0x8, kVmem = 0x10, kDsRead = 0x100, kAll = LOADS + READS;
#pragma unroll
  for (int i = 0; i < kAll; ++i) {
    if ((i + 1) * MFMAS / kAll > i * MFMAS / kAll) __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    if (i < LOADS)
      __builtin_amdgcn_sched_group_barrier(kVmem, 1, 0);
    else
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, MFMAS, 0);
  __builtin_amdgcn_sched_barrier(0);
}

template <int MF, int NF, bool F32_OUT>
__global__ void __launch_bounds__(kThreads, 2)
    mxfp4_gemm_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ xe, uint32_t m,
                      const uint8_t* __restrict__ w, const uint8_t* __restrict__ we, uint32_t n, uint32_t nb,
                      void* __restrict__ y, int64_t ldy, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int BM = 64 * MF, BN = 32 * NF;
  using S = Stages<MF, NF>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = wave >> 1, wn = wave & 1u;

  // Tiles in column blocks of 8 n-tiles, m fastest inside a block: the tiles an XCD
  // runs together share X and W rows in its L2.
  const uint32_t t = xcd_order(blockIdx.x, gridDim.x);
  const uint32_t per = 8 * tiles_m, blk = t / per, in = t - blk * per;
  const uint32_t bw = min(8u, tiles_n - 8 * blk);
  const uint32_t tm = in / bw, tn = 8 * blk + (in - tm * bw);
  const uint32_t m0 = tm * BM, n0 = tn * BN;

  // Codes past the last row read as zeros (the buffers' ends); scales of rows past it
  // are the last row's. Their products are not stored.
  const uint32_t row = nb * 16;
  const uint32_t xr = min(m - 1 - m0, BM - 1u), wr = min(n - 1 - n0, BN - 1u);  // last rows of the tile
  const __amdgpu_buffer_rsrc_t X = buffer_rsrc(x + static_cast<int64_t>(m0) * row, (xr + 1) * row);
  const __amdgpu_buffer_rsrc_t W = buffer_rsrc(w + static_cast<int64_t>(n0) * row, (wr + 1) * row);
  // The wave's i-th X (W) instruction brings rows 64 i + 8 wave .. + 7 of the tile's
  // X (W) rows (with an odd NF, rows past the tile that nobody reads).
  constexpr int kWi = (NF + 1) / 2;
  const uint32_t r0 = 8 * wave + (lane >> 3), off0 = r0 * row + ((lane & 7u) ^ ((r0 >> 1) & 7u)) * 16;
  auto load_x = [&](uint32_t at, uint32_t step) {
#pragma unroll
    for (int i = 0; i < MF; ++i)
      dma16(X, smem + at + wave * 1024 + i * 8192, off0 + (step * kRowBytes + i * 64 * row), 0);
  };
  auto load_w = [&](uint32_t at, uint32_t step) {
#pragma unroll
    for (int i = 0; i < kWi; ++i)
      dma16(W, smem + S::kNX * S::kX + at + wave * 1024 + i * 8192, off0 + (step * kRowBytes + i * 64 * row), 0);
  };
  // Thread's row of scales (X rows, then W rows; threads past them repeat the last).
  const uint32_t srow = min(tid, BM + BN - 1u);
  const uint8_t* se = srow < BM ? xe + static_cast<int64_t>(m0 + min(srow, xr)) * nb
                                : we + static_cast<int64_t>(n0 + min(srow - BM, wr)) * nb;
  // The last step's bytes past the row shift in as zeros.
  auto load_scales = [&](uint32_t step) {
    const uint32_t at = min(step * kStepBlocks, nb - kStepBlocks);
    uint64_t v;
    __builtin_memcpy(&v, se + at, 8);
    return v;
  };
  auto keep_scales = [&](uint64_t v, uint32_t step) {
    v >>= 8 * (step * kStepBlocks - min(step * kStepBlocks, nb - kStepBlocks));
    *reinterpret_cast<u32x2_t*>(smem + S::kScales + (step & 1u) * S::kS + srow * kStepBlocks) =
        u32x2_t{static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32)};
  };

  // Operand reads: fragment row l % 16, chunk 4 h + l / 16 of half h. Rows are 16
  // apart from fragment to fragment, so the permutation is the lane's.
  const uint32_t fr = lane & 15u, g = lane >> 4;
  const uint32_t rd = fr * kRowBytes + ((g ^ ((fr >> 1) & 7u)) * 16);
  const uint32_t rx = (wm * 16 * MF) * kRowBytes + rd, rw = S::kNX * S::kX + (wn * 16 * NF) * kRowBytes + rd;
  const uint32_t sx = S::kScales + (wm * 16 * MF + fr) * kStepBlocks + g;
  const uint32_t sw = S::kScales + (BM + wn * 16 * NF + fr) * kStepBlocks + g;
  struct Frags {
    u32x4_t x[MF], w[NF];
    uint32_t ex[MF], ew[NF];
  };
  auto read = [&](Frags& f, uint32_t xat, uint32_t wat, uint32_t step, int h) {
    const uint32_t sat = (step & 1u) * S::kS + 4 * h;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      f.w[j] = *reinterpret_cast<const u32x4_t*>(smem + wat + ((rw ^ (h * 64)) + j * 16 * kRowBytes));
      f.ew[j] = smem[sw + sat + j * 16 * kStepBlocks];
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      f.x[i] = *reinterpret_cast<const u32x4_t*>(smem + xat + ((rx ^ (h * 64)) + i * 16 * kRowBytes));
      f.ex[i] = smem[sx + sat + i * 16 * kStepBlocks];
    }
  };
  f32x4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const i32x8_t a = {static_cast<int>(f.w[j].x), static_cast<int>(f.w[j].y), static_cast<int>(f.w[j].z),
                           static_cast<int>(f.w[j].w)};
        const i32x8_t b = {static_cast<int>(f.x[i].x), static_cast<int>(f.x[i].y), static_cast<int>(f.x[i].z),
                           static_cast<int>(f.x[i].w)};
        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[j][i], 4, 4, 0,
                                                                     static_cast<int>(f.ew[j]), 0,
                                                                     static_cast<int>(f.ex[i]));
      }
  };
  // The wave's loads up to the next step's have landed (they retire in order;
  // `newer` later ones may be in flight) and its LDS work is done, then the same of
  // every wave.
  auto publish = [&](auto newer) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(newer)::value) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Loads behind the next step's at a publish: the whole of the steps after it, or
  // the W of the one after it, which is requested last.
  constexpr int kNewer = (S::kNX - 2) * MF + (S::kNW - 2) * kWi;
  auto wrap = [](uint32_t at, uint32_t by, uint32_t end) { return at + by == end ? 0u : at + by; };

  const uint32_t steps = (nb + kStepBlocks - 1) / kStepBlocks;
  Frags f0, f1;
  keep_scales(load_scales(0), 0);
  uint64_t next = load_scales(min(1u, steps - 1));
#pragma unroll
  for (int i = 0; i < S::kNW; ++i) {
    if (i < S::kNX) load_x(i * S::kX, min(static_cast<uint32_t>(i), steps - 1));
    load_w(i * S::kW, min(static_cast<uint32_t>(i), steps - 1));
  }
  publish(std::integral_constant<int, MF + kWi + kNewer>());
  read(f0, 0, 0, 0, 0);
  uint32_t xat = 0, wat = 0;
#pragma unroll 1
  for (uint32_t s = 0; s + 1 < steps; ++s) {
    const uint32_t xn = wrap(xat, S::kX, S::kNX * S::kX), wn_ = wrap(wat, S::kW, S::kNW * S::kW);
    // f0's reads ran under the multiplies of f1: waiting for them here, before f1's
    // reads are issued, keeps the compiler from waiting for both below.
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    read(f1, xat, wat, s, 1);
    multiply(f0);
    interleave<MF * NF, 2 * (MF + NF), 0>();
    keep_scales(next, s + 1);
    publish(std::integral_constant<int, kNewer>());
    // Past the last step the last one is loaded again, which keeps the counts.
    next = load_scales(min(s + 2, steps - 1));
    load_x(xat, min(s + S::kNX, steps - 1));
    load_w(wat, min(s + S::kNW, steps - 1));
    xat = xn, wat = wn_;
    read(f0, xat, wat, s + 1, 0);
    multiply(f1);
    interleave<MF * NF, 2 * (MF + NF), MF + kWi + 1>();
  }
  read(f1, xat, wat, steps - 1, 1);
  multiply(f0);
  multiply(f1);
  publish(std::integral_constant<int, 0>());  // no load may be in flight when the workgroup's LDS is given back

  // Lane l holds Y[.. + l % 16][.. + 4 (l / 16) + e] of each fragment.
  using OutT = typename std::conditional<F32_OUT, float, uint16_t>::type;
  OutT* Y = static_cast<OutT*>(y);
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const uint32_t gm = m0 + (wm * MF + i) * 16 + fr;
    if (gm >= m) continue;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const uint32_t gn = n0 + (wn * NF + j) * 16 + 4 * g;
      if (gn >= n) continue;
      OutT* dst = Y + gm * ldy + gn;
      const f32x4_t a = acc[j][i];
      if constexpr (F32_OUT) {
        if (gn + 4 <= n && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
          *reinterpret_cast<f32x4_t*>(dst) = a;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (gn + e < n) dst[e] = a[e];
        }
      } else {
        const uint32_t v[2] = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])};
        if (gn + 4 <= n && (reinterpret_cast<uintptr_t>(dst) & 7u) == 0) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (gn + e < n) dst[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1)));
        }
      }
    }
  }
}

template <int MF, int NF>
int launch(const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int y_type, int64_t ldy,
           hipStream_t s) {
  const bool f32 = y_type == SPIRAL_TYPE_F32;
  const void* fn = f32 ? reinterpret_cast<const void*>(&mxfp4_gemm_kernel<MF, NF, true>)
                       : reinterpret_cast<const void*>(&mxfp4_gemm_kernel<MF, NF, false>);
  constexpr int lds = Stages<MF, NF>::kBytes;
  const int rc = allow_dynamic_lds(fn, lds);
  if (rc != SPIRAL_OK) return rc;
  const int64_t tm = ceil_div(m, 64 * MF), tn = ceil_div(n, 32 * NF);
  const dim3 grid(static_cast<unsigned>(tm * tn));
  const uint8_t *xe = x + m * nb * 16, *we = w + n * nb * 16;
#define SPIRAL_GEMM(F32)                                                                                        \
  hipLaunchKernelGGL((mxfp4_gemm_kernel<MF, NF, F32>), grid, dim3(kThreads), lds, s, x, xe, static_cast<uint32_t>(m), \
                     w, we, static_cast<uint32_t>(n), static_cast<uint32_t>(nb), y, ldy, static_cast<uint32_t>(tm),   \
                     static_cast<uint32_t>(tn))
  if (f32)
    SPIRAL_GEMM(true);
  else
    SPIRAL_GEMM(false);
#undef SPIRAL_GEMM
  return launch_status();
}

// Tiles (64 MF rows of X x 32 NF rows of W) and their average k step, ns.
struct Tile {
  int mf, nf, step_ns;
};
constexpr Tile kTiles[] = {{4, 8, 1330}, {4, 4, 730}, {2, 4, 510}, {1, 4, 380}};

int64_t tile_ns(const Tile& t, int64_t m, int64_t n, int64_t nb) {
  const int64_t rounds = ceil_div(ceil_div(m, 64 * t.mf) * ceil_div(n, 32 * t.nf), device_cu_count());
  return rounds * (ceil_div(nb, kStepBlocks) * t.step_ns + 2000);
}

}  // namespace

// Whether the tiled form takes this product: at least a step of k, 32-bit offsets
// inside a tile and 32-bit tile counts.
bool mxfp4_gemm_fits(int64_t m, int64_t n_rows, int64_t nb) {
  return m > 16 && nb >= kStepBlocks && nb < (1 << 18) && m <= (1 << 24) && n_rows <= (1 << 24) &&
         ceil_div(m, 64) * ceil_div(n_rows, 128) <= INT32_MAX;
}

int mxfp4_gemm(const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int y_type, int64_t ldy,
               hipStream_t s) {
  Tile best = kTiles[0];
  for (const Tile& t : kTiles)
    if (tile_ns(t, m, n, nb) < tile_ns(best, m, n, nb)) best = t;
  if (best.mf == 1) return launch<1, 4>(x, m, w, n, nb, y, y_type, ldy, s);
  if (best.mf == 2) return launch<2, 4>(x, m, w, n, nb, y, y_type, ldy, s);
  return best.nf == 4 ? launch<4, 4>(x, m, w, n, nb, y, y_type, ldy, s)
                      : launch<4, 8>(x, m, w, n, nb, y, y_type, ldy, s);
}

}  // namespace spiral

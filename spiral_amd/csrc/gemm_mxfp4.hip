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
//  - Scales (a row has k / 32 of them, at any alignment) are loaded by the thread
//    that owns the row, 32 bytes for four steps at a time: 8 bytes a step would ask
//    for as many cache lines as the codes do. They are turned (4 x 4 bytes) into a
//    dword a lane group, whose bytes are the four halves of two steps, and go to LDS
//    for two steps at a time; the instruction selects the byte. Blocks past the end
//    of a row get scale bytes 0 on both sides: whatever codes the loads brought for
//    them, 2^-127 times 2^-127 times 36 is no fp32 number.
//  - A step's two halves have an operand register set each: one is read from LDS
//    while the other multiplies. The barrier lies between them, when a wave holds
//    all of the step's operands, and both publishes the next stage and frees this one.
//
// Measured, 2048 x 14336 x 4096, bf16 out: 80 us, 3.0 PFLOP/s (256 x 160 tiles, three
// rounds of 16 steps of about a microsecond). Without the stores 53 us: a tile's 80 KiB
// go out when the CU does nothing else, its LDS and registers holding one workgroup.
// Within a tile the loads bound it, 50 bytes a nanosecond and CU; the matrix cores are
// busy a third of the time. 777 x 4096 x 4096: 15.6 us, 224 tiles of 128 x 128.
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
// of scales, two steps each.
constexpr int kLdsBytes = 160 * 1024;
template <int MF, int NF>
struct Stages {
  static constexpr int kBM = 64 * MF, kBN = 32 * NF;
  static constexpr int kX = kBM * kRowBytes, kW = 64 * ((NF + 1) / 2) * kRowBytes;
  static constexpr int kS = (kBM + kBN) * 2 * kStepBlocks;
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
                      void* __restrict__ y, int64_t ldy, uint32_t tiles_m, uint32_t tiles_n, uint32_t range) {
  using S = Stages<MF, NF>;
  constexpr int BM = S::kBM, BN = S::kBN;
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
  // X (W) rows (with an odd NF, at the end, rows past the tile that nobody reads).
  constexpr int kWi = (NF + 1) / 2, kStride = 64 * kRowBytes;
  const uint32_t r0 = 8 * wave + (lane >> 3), off0 = r0 * row + ((lane & 7u) ^ ((r0 >> 1) & 7u)) * 16;
  auto load_x = [&](uint32_t at, uint32_t step) {
#pragma unroll
    for (int i = 0; i < MF; ++i)
      dma16(X, smem + at + wave * 1024 + i * kStride, off0 + (step * kRowBytes + i * 64 * row), 0);
  };
  auto load_w = [&](uint32_t at, uint32_t step) {
#pragma unroll
    for (int i = 0; i < kWi; ++i)
      dma16(W, smem + S::kNX * S::kX + at + wave * 1024 + i * kStride, off0 + (step * kRowBytes + i * 64 * row), 0);
  };
  // Thread's rows of scales (X rows, then W rows; past them the last one again).
  constexpr int kSr = (BM + BN + kThreads - 1) / kThreads;
  const uint8_t* se[kSr];
  uint32_t s_lds[kSr];
#pragma unroll
  for (int j = 0; j < kSr; ++j) {
    const uint32_t r = min(tid + j * kThreads, BM + BN - 1u);
    se[j] = r < BM ? xe + static_cast<int64_t>(m0 + min(r, xr)) * nb
                   : we + static_cast<int64_t>(n0 + min(r - BM, wr)) * nb;
    s_lds[j] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)smem)) +
               S::kScales + r * (2 * kStepBlocks);
  }
  // Steps 4 q .. + 3, eight bytes a step; bytes past the row are shifted out when used.
  u32x2_t lo[kSr][2], hi[kSr][2];
  auto load_scales = [&](uint32_t q) {
#pragma unroll
    for (int j = 0; j < kSr; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        __builtin_memcpy(&lo[j][i], se[j] + min((4 * q + i) * kStepBlocks, nb - kStepBlocks), 8);
        __builtin_memcpy(&hi[j][i], se[j] + min((4 * q + 2 + i) * kStepBlocks, nb - kStepBlocks), 8);
      }
  };
  // Steps s and s + 1 (the first or second two of four) to the stage of s / 2. The
  // write is in assembly because the compiler lets an ordinary one wait for every
  // direct load in flight.
  auto keep_scales = [&](uint32_t s) {
#pragma unroll
    for (int j = 0; j < kSr; ++j) {
      uint32_t d[4];
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t at = (s + i) * kStepBlocks, past = at - min(at, nb - kStepBlocks);
        const u32x2_t r = s & 2 ? hi[j][i] : lo[j][i];
        const uint64_t v = past >= 8 ? 0 : (r.x | static_cast<uint64_t>(r.y) << 32) >> (8 * past);
        d[2 * i] = static_cast<uint32_t>(v), d[2 * i + 1] = static_cast<uint32_t>(v >> 32);
      }
      const uint32_t t0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u);  // bytes 0 and 1 of d0 and d1
      const uint32_t t1 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u);
      const uint32_t t2 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
      const uint32_t t3 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
      const u32x4_t out{__builtin_amdgcn_perm(t1, t0, 0x05040100u), __builtin_amdgcn_perm(t1, t0, 0x07060302u),
                        __builtin_amdgcn_perm(t3, t2, 0x05040100u), __builtin_amdgcn_perm(t3, t2, 0x07060302u)};
      asm volatile("ds_write_b128 %0, %1" ::"v"(s_lds[j] + (s / 2 & 1u) * S::kS), "v"(out) : "memory");
    }
  };

  // Operand reads: fragment row l % 16, chunk 4 h + l / 16 of half h. Rows are 16
  // apart from fragment to fragment, so the permutation is the lane's.
  const uint32_t fr = lane & 15u, g = lane >> 4;
  const uint32_t rd = fr * kRowBytes + ((g ^ ((fr >> 1) & 7u)) * 16);
  const uint32_t rx = (wm * 16 * MF) * kRowBytes + rd, rw = S::kNX * S::kX + (wn * 16 * NF) * kRowBytes + rd;
  const uint32_t sx = S::kScales + (wm * 16 * MF + fr) * (2 * kStepBlocks) + 4 * g;
  const uint32_t sw = S::kScales + (BM + wn * 16 * NF + fr) * (2 * kStepBlocks) + 4 * g;
  struct Frags {
    u32x4_t x[MF], w[NF];
  };
  struct Scales {
    uint32_t x[MF], w[NF];
  };
  auto read = [&](Frags& f, uint32_t xat, uint32_t wat, int h) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
      f.w[j] = *reinterpret_cast<const u32x4_t*>(smem + wat + ((rw ^ (h * 64)) + j * 16 * kRowBytes));
#pragma unroll
    for (int i = 0; i < MF; ++i)
      f.x[i] = *reinterpret_cast<const u32x4_t*>(smem + xat + ((rx ^ (h * 64)) + i * 16 * kRowBytes));
  };
  auto read_scales = [&](Scales& e, uint32_t s) {
    const uint32_t at = (s / 2 & 1u) * S::kS;
#pragma unroll
    for (int j = 0; j < NF; ++j)
      e.w[j] = *reinterpret_cast<const uint32_t*>(smem + sw + at + j * 32 * kStepBlocks);
#pragma unroll
    for (int i = 0; i < MF; ++i)
      e.x[i] = *reinterpret_cast<const uint32_t*>(smem + sx + at + i * 32 * kStepBlocks);
  };
  auto shift_scales = [](Scales& e) {  // to the second of the two steps
#pragma unroll
    for (int j = 0; j < NF; ++j) e.w[j] >>= 16;
#pragma unroll
    for (int i = 0; i < MF; ++i) e.x[i] >>= 16;
  };
  f32x4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Frags& f, const Scales& e, auto byte) {
    constexpr int B = decltype(byte)::value;
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const i32x8_t a = {static_cast<int>(f.w[j].x), static_cast<int>(f.w[j].y), static_cast<int>(f.w[j].z),
                           static_cast<int>(f.w[j].w)};
        const i32x8_t b = {static_cast<int>(f.x[i].x), static_cast<int>(f.x[i].y), static_cast<int>(f.x[i].z),
                           static_cast<int>(f.x[i].w)};
        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[j][i], 4, 4, B,
                                                                     static_cast<int>(e.w[j]), B,
                                                                     static_cast<int>(e.x[i]));
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

  // This workgroup's steps of k: `range` of them, a multiple of four.
  const uint32_t first = blockIdx.y * range;
  const uint32_t steps = min((nb + kStepBlocks - 1) / kStepBlocks, first + range);
  if constexpr (F32_OUT) y = static_cast<float*>(y) + static_cast<int64_t>(blockIdx.y) * m * ldy;
  Frags f0, f1;
  Scales e;
  load_scales(first / 4);
  keep_scales(first);
#pragma unroll
  for (int i = 0; i < S::kNW; ++i) {
    if (i < S::kNX) load_x(i * S::kX, min(first + i, steps - 1));
    load_w(i * S::kW, min(first + i, steps - 1));
  }
  publish(std::integral_constant<int, MF + kWi + kNewer>());
  read(f0, 0, 0, 0);
  read_scales(e, first);
  uint32_t xat = 0, wat = 0;
  // The scales of two steps are written a step ahead, and read when those of the two
  // before have been used: a second register set would cost the wider tile.
#pragma unroll 1
  for (uint32_t s = first; s + 1 < steps; ++s) {
    const uint32_t xn = wrap(xat, S::kX, S::kNX * S::kX), wn_ = wrap(wat, S::kW, S::kNW * S::kW);
    // f0's reads ran under the multiplies of f1: waiting for them here, before f1's
    // reads are issued, keeps the compiler from waiting for both below.
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    read(f1, xat, wat, 1);
    multiply(f0, e, std::integral_constant<int, 0>());
    interleave<MF * NF, MF + NF, 0>();
    if ((s & 1) == 0) keep_scales(s + 2);
    publish(std::integral_constant<int, kNewer>());
    if ((s & 3) == 0) load_scales(s / 4 + 1);
    // Past the last step the last one is loaded again, which keeps the counts.
    load_x(xat, min(s + S::kNX, steps - 1));
    load_w(wat, min(s + S::kNW, steps - 1));
    xat = xn, wat = wn_;
    read(f0, xat, wat, 0);
    multiply(f1, e, std::integral_constant<int, 1>());
    interleave<MF * NF, MF + NF, MF + kWi>();
    if (s & 1)
      read_scales(e, s + 1);
    else
      shift_scales(e);
  }
  read(f1, xat, wat, 1);
  multiply(f0, e, std::integral_constant<int, 0>());
  multiply(f1, e, std::integral_constant<int, 1>());
  publish(std::integral_constant<int, 0>());  // no load may be in flight when the workgroup's LDS is given back

  // Lane l holds Y[.. + l % 16][.. + 4 (l / 16) + e] of each fragment: 32 bytes of a
  // row of bf16 for four lanes. The tile's fragments go through LDS, 16 rows of each
  // wave or as many as it holds at a time, and are stored in whole rows, 16 bytes a
  // lane, past the caches.
  using OutT = typename std::conditional<F32_OUT, float, uint16_t>::type;
  constexpr uint32_t kSize = sizeof(OutT), kLine = BN * kSize + 16, kChunks = BN * kSize / 16;
  constexpr int kPass = 64 * MF * kLine <= S::kBytes ? MF : 64 * (MF / 2) * kLine <= S::kBytes ? MF / 2 : 1;
  static_assert(64 * kPass * kLine <= S::kBytes && MF % kPass == 0, "the rows of a pass in LDS");
  OutT* Y = static_cast<OutT*>(y);
#pragma unroll
  for (int i0 = 0; i0 < MF; i0 += kPass) {
    if (i0 > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      uint8_t* line = smem + ((wm * kPass + i) * 16 + fr) * kLine + (wn * NF * 16 + 4 * g) * kSize;
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const f32x4_t a = acc[j][i0 + i];
        if constexpr (F32_OUT)
          *reinterpret_cast<f32x4_t*>(line + j * 64) = a;
        else
          *reinterpret_cast<u32x2_t*>(line + j * 32) = u32x2_t{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])};
      }
    }
    __syncthreads();
    for (uint32_t c = tid; c < 64 * kPass * kChunks; c += kThreads) {
      const uint32_t r = c / kChunks, col = (c - r * kChunks) * (16 / kSize);
      const uint32_t gm = m0 + (r / (16 * kPass) * MF + i0) * 16 + r % (16 * kPass), gn = n0 + col;
      if (gm >= m || gn >= n) continue;
      OutT* dst = Y + gm * ldy + gn;
      const uint8_t* src = smem + r * kLine + col * kSize;
      if (gn + 16 / kSize <= n && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
        __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(src), reinterpret_cast<u32x4_t*>(dst));
      } else {
        for (uint32_t e = 0; e < 16 / kSize && gn + e < n; ++e) dst[e] = reinterpret_cast<const OutT*>(src)[e];
      }
    }
  }
}

// Y = the sum of `parts` F32 results of m rows of `line` floats (n rounded up to
// four), in order. Four columns a thread.
template <bool F32_OUT>
__global__ void __launch_bounds__(256) mxfp4_join_kernel(const float* __restrict__ part, uint32_t parts, uint32_t m,
                                                         uint32_t n, uint32_t line, void* __restrict__ y,
                                                         int64_t ldy) {
  using OutT = typename std::conditional<F32_OUT, float, uint16_t>::type;
  const uint32_t i = (blockIdx.x * 256 + threadIdx.x) * 4, row = i / line, col = i - row * line;
  if (row >= m) return;
  const int64_t all = static_cast<int64_t>(m) * line;
  f32x4_t sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t p = 0; p < parts; ++p) sum += *reinterpret_cast<const f32x4_t*>(part + p * all + i);
  OutT* dst = static_cast<OutT*>(y) + row * ldy + col;
  const uint32_t v[2] = {pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  if (col + 4 <= n && (reinterpret_cast<uintptr_t>(dst) & (4 * sizeof(OutT) - 1)) == 0) {
    if constexpr (F32_OUT)
      *reinterpret_cast<f32x4_t*>(dst) = sum;
    else
      *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{v[0], v[1]};
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    if (col + e >= n) break;
    if constexpr (F32_OUT)
      dst[e] = sum[e];
    else
      dst[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1)));
  }
}

template <int MF, int NF, bool F32_OUT>
int launch(const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int64_t ldy, int64_t splits,
           int64_t range, hipStream_t s) {
  using S = Stages<MF, NF>;
  const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&mxfp4_gemm_kernel<MF, NF, F32_OUT>), S::kBytes);
  if (rc != SPIRAL_OK) return rc;
  const int64_t tm = ceil_div(m, S::kBM), tn = ceil_div(n, S::kBN);
  hipLaunchKernelGGL((mxfp4_gemm_kernel<MF, NF, F32_OUT>),
                     dim3(static_cast<unsigned>(tm * tn), static_cast<unsigned>(splits)), dim3(kThreads), S::kBytes, s,
                     x, x + m * nb * 16, static_cast<uint32_t>(m), w, w + n * nb * 16, static_cast<uint32_t>(n),
                     static_cast<uint32_t>(nb), y, ldy, static_cast<uint32_t>(tm), static_cast<uint32_t>(tn),
                     static_cast<uint32_t>(range));
  return launch_status();
}

template <bool F32_OUT>
int launch_tile(int tile, const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int64_t ldy,
                int64_t splits, int64_t range, hipStream_t s) {
  switch (tile) {
    case 0: return launch<4, 5, F32_OUT>(x, m, w, n, nb, y, ldy, splits, range, s);
    case 1: return launch<4, 4, F32_OUT>(x, m, w, n, nb, y, ldy, splits, range, s);
    case 2: return launch<2, 4, F32_OUT>(x, m, w, n, nb, y, ldy, splits, range, s);
    default: return launch<1, 4, F32_OUT>(x, m, w, n, nb, y, ldy, splits, range, s);
  }
}

// Tiles (64 mf rows of X x 32 nf rows of W), the workgroups a CU has room for, and
// nanoseconds of a step of one of them and of a round besides its steps (first
// loads, stores). Two on a CU take 1.7 times as long a step.
struct Tile {
  int mf, nf, per_cu, step_ns, round_ns;
};
constexpr Tile kTiles[] = {{4, 5, 1, 1350, 5000}, {4, 4, 1, 1200, 4000}, {2, 4, 1, 800, 2500}, {1, 4, 2, 620, 2500}};

// Floats of a row of a part.
int64_t part_line(int64_t n) { return ceil_div(n, 4) * 4; }

struct Plan {
  int tile;
  int64_t splits, range;  // ranges of k, steps each
};

// The tile and ranges of k that are estimated fastest. A join costs a launch and
// the F32 parts' way to memory and back.
Plan make_plan(int64_t m, int64_t n, int64_t nb, int64_t most_splits) {
  const int64_t steps = ceil_div(nb, kStepBlocks);
  if (m * part_line(n) > INT32_MAX - 1024) most_splits = 1;  // 32-bit indexes in the join
  Plan best{0, 1, 0};
  int64_t best_ns = INT64_MAX;
  for (int t = 0; t < 4; ++t) {
    const Tile& c = kTiles[t];
    const int64_t tiles = ceil_div(m, 64 * c.mf) * ceil_div(n, 32 * c.nf);
    for (int64_t want = 1; want <= std::min<int64_t>(16, most_splits); ++want) {
      const int64_t range = ceil_div(ceil_div(steps, want), 4) * 4, splits = ceil_div(steps, range);
      if (splits != want) continue;
      const int64_t on_cu = std::min<int64_t>(c.per_cu, ceil_div(tiles * splits, device_cu_count()));
      const int64_t rounds = ceil_div(tiles * splits, on_cu * device_cu_count());
      const int64_t step = on_cu == 2 ? c.step_ns * 17 / 10 : c.step_ns;
      const int64_t ns = rounds * (std::min(range, steps) * step + c.round_ns) +
                         (splits > 1 ? 3500 + splits * m * n / 450 : 0);
      if (ns < best_ns) best_ns = ns, best = Plan{t, splits, range};
    }
  }
  return best;
}

}  // namespace

// Whether the tiled form takes this product: at least a step of k, 32-bit offsets
// inside a tile and 32-bit tile counts.
bool mxfp4_gemm_fits(int64_t m, int64_t n_rows, int64_t nb) {
  return m > 16 && nb >= kStepBlocks && nb < (1 << 18) && m <= (1 << 24) && n_rows <= (1 << 24) &&
         ceil_div(m, 64) * ceil_div(n_rows, 128) <= INT32_MAX;
}

int64_t mxfp4_gemm_workspace(int64_t m, int64_t n_rows, int64_t nb) {
  const Plan p = make_plan(m, n_rows, nb, INT64_MAX);
  return p.splits > 1 ? p.splits * m * part_line(n_rows) * 4 : 0;
}

int mxfp4_gemm(const uint8_t* x, int64_t m, const uint8_t* w, int64_t n, int64_t nb, void* y, int y_type, int64_t ldy,
               void* workspace, int64_t workspace_bytes, hipStream_t s) {
  const Plan p = make_plan(m, n, nb, std::max<int64_t>(1, workspace_bytes / (m * part_line(n) * 4)));
  const bool f32 = y_type == SPIRAL_TYPE_F32;
  if (p.splits == 1)
    return f32 ? launch_tile<true>(p.tile, x, m, w, n, nb, y, ldy, 1, p.range, s)
               : launch_tile<false>(p.tile, x, m, w, n, nb, y, ldy, 1, p.range, s);
  const int rc = launch_tile<true>(p.tile, x, m, w, n, nb, workspace, part_line(n), p.splits, p.range, s);
  if (rc != SPIRAL_OK) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(m * part_line(n), 1024)));
  const float* part = static_cast<const float*>(workspace);
  if (f32)
    hipLaunchKernelGGL(mxfp4_join_kernel<true>, grid, dim3(256), 0, s, part, static_cast<uint32_t>(p.splits),
                       static_cast<uint32_t>(m), static_cast<uint32_t>(n), static_cast<uint32_t>(part_line(n)), y, ldy);
  else
    hipLaunchKernelGGL(mxfp4_join_kernel<false>, grid, dim3(256), 0, s, part, static_cast<uint32_t>(p.splits),
                       static_cast<uint32_t>(m), static_cast<uint32_t>(n), static_cast<uint32_t>(part_line(n)), y, ldy);
  return launch_status();
}

}  // namespace spiral

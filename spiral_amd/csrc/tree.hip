// Attention of drafted trees over a paged cache (spiral_cache.h).
//
// out_i = sum_r p_ir V_r / sum_r p_ir,  p_ir = exp(scale q_i . K_r - m_i), in one
// pass over the rows with a running maximum m_i and sum.
//
// The query rows of one cached head (its group of heads times the tree's nodes) are
// the columns of every matrix product, so they share each loaded row:
//   S^T = K Q^T   v_mfma_f32_16x16x32: 16 cached rows x 16 queries, over dim
//   O^T += V^T P^T  the same: 16 dims x 16 queries, over 32 cached rows
// A lane's four results of S^T are four cached rows of one query. Taken from two
// tiles of 16 rows they are the eight elements of the lane's second operand of
// O^T, for the order of the product's 32 rows in which lane group g has rows
// 4g .. 4g + 3 and 16 + 4g .. + 3: P^T never leaves its registers.
//
// Up to two tiles of 16 queries (QB = 1): every wave has them all and takes every
// fourth chunk of 32 rows, loaded straight to registers, K in operand order. A lane
// has 8 consecutive dims (4 where dim <= 64) of the eight rows of V of its group, so
// the lanes of a group read a whole row, and turns them by one v_perm_b32 a dword;
// product d of the eight covers dim 8 r + d of every lane r.
// More queries (QB = 2, 4, 8): the waves of a workgroup share rows. A stage (a chunk
// of 32 rows of K and of V for each of the KW waves of a query block) is brought to LDS
// by direct loads, kStages of them in flight: loaded by each wave for itself, a chunk at a time, a CU had 16 KiB in flight and waited for it (16
// sequences of up to 8192 rows, 25 nodes x 4 heads, dim 128: 169 us). V's operands
// are read with ds_read_b64_tr_b16, which turns 4 rows x 16 dims.
// The waves of a block join their sums through LDS, and where a sequence's rows are
// split over workgroups, tree_join_kernel joins these from the workspace, in order
// of the rows. The host does not know the lengths: workgroups deal the rows of all
// sequences out themselves, in shares of one length (Share). Split evenly by the
// longest sequence, half the workgroups of a ragged batch had nothing to do.
//
// A new maximum below 2^kSlack of the old one is not taken: p then stays below
// 2^kSlack (F16: 2^kLift times that), which fp32 sums and both 16-bit types hold, and the
// sums are rarely rescaled. p is rounded to the cache's type for the matrix instruction, by
// at most half a step (bf16 2^-8 of p, as much as the output is rounded by: outputs are 1.1
// to 1.4 times as far from float64 as with an unrounded p); its sum is of the values before
// rounding.
//
// What bounds it: decoding (48 sequences of up to 4096 rows, 8 cached heads, dim 128: 99 to
// 102 us, 4.4 to 4.6 TB/s) the bytes; the smallest calls (one of 4096 rows: 13.2 us) chains
// of dependent loads and the second launch; many queries (two sequences of 65536 rows, 512
// queries, dim 256: 73 to 74 us, 0.47 PFLOP/s) latencies within a stage, with two waves a
// SIMD to hide them: registers hold no more. The matrix cores are busy 20 to 25 %.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "tree.h"

namespace spiral {
namespace {

// Elements at .. + 7 of a row of dim elements, zeros past it (FULL: there is nothing past it).
template <bool FULL>
__device__ __forceinline__ u32x4_t load_dims(const uint8_t* row, uint32_t at, uint32_t dim) {
  const bool on = FULL || at < dim;
  const u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + (on ? 2 * at : 0u));
  return on ? w : u32x4_t{0, 0, 0, 0};
}

// 16 bytes a lane from memory straight to LDS, in lane order from the wave's `lds` on.
__device__ __forceinline__ void load_to_lds(const uint8_t* src, uint8_t* lds) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(
                                       reinterpret_cast<uintptr_t>(src)),
                                   (__attribute__((address_space(3))) uint32_t*)lds, 16, 0, 0);
}

__device__ __forceinline__ uint32_t lds_offset(const uint8_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint8_t*)p));
}

// Operands of V for four (eight) tiles of 16 dims: of each 16 lanes, lane r gives at[d]
// + LO (HI), where 4 dims of row r / 4 lie, and gets dim r of the four rows, for LO
// and for HI. In assembly, with its wait: in front of the builtin the compiler waits
// for every direct load in flight.
template <int LO, int HI>
__device__ __forceinline__ void read_turned4(u32x4_t* v, const uint32_t* at) {
  u32x2_t a[4], b[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(LO), "n"(HI)
      : "memory");
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] = u32x4_t{a[d].x, a[d].y, b[d].x, b[d].y};
}
template <int LO, int HI>
__device__ __forceinline__ void read_turned8(u32x4_t* v, const uint32_t* at) {
  u32x2_t a[8], b[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %8, %16 offset:%25\n\t"
      "ds_read_b64_tr_b16 %1, %17 offset:%24\n\tds_read_b64_tr_b16 %9, %17 offset:%25\n\t"
      "ds_read_b64_tr_b16 %2, %18 offset:%24\n\tds_read_b64_tr_b16 %10, %18 offset:%25\n\t"
      "ds_read_b64_tr_b16 %3, %19 offset:%24\n\tds_read_b64_tr_b16 %11, %19 offset:%25\n\t"
      "ds_read_b64_tr_b16 %4, %20 offset:%24\n\tds_read_b64_tr_b16 %12, %20 offset:%25\n\t"
      "ds_read_b64_tr_b16 %5, %21 offset:%24\n\tds_read_b64_tr_b16 %13, %21 offset:%25\n\t"
      "ds_read_b64_tr_b16 %6, %22 offset:%24\n\tds_read_b64_tr_b16 %14, %22 offset:%25\n\t"
      "ds_read_b64_tr_b16 %7, %23 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7]),
        "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(b[4]), "=&v"(b[5]), "=&v"(b[6]), "=&v"(b[7])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7]), "n"(LO),
        "n"(HI)
      : "memory");
#pragma unroll
  for (int d = 0; d < 8; ++d) v[d] = u32x4_t{a[d].x, a[d].y, b[d].x, b[d].y};
}

// Of two elements of V, those of rows that are not there (clear in `on`), infinities
// and NaN to zeros; whether there were any of the latter.
template <typename E>
__device__ __forceinline__ bool clean(uint32_t& v, uint32_t on) {
  const uint32_t w = v & on;
  const bool lo = (w & E::kExp) == E::kExp, hi = (w >> 16 & E::kExp) == E::kExp;
  v = w & (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
  return lo || hi;
}

// How a workgroup is made up: rows of up to 16 DV dims (DV = 4, 8, 16), QT tiles of
// queries a wave, QB query blocks.
template <int DV, int QT, int QB>
struct Shape {
  static constexpr int kWaves = QB == 8 ? 8 : 4;
  static constexpr int KW = kWaves / QB;  // waves that share a query block
  static constexpr int kDims = 16 * DV, kQueries = 16 * QT;
  static constexpr int kRow = 2 * kDims;                 // bytes of a row in LDS
  static constexpr int kHalf = kChunk * kRow;            // a chunk's K or V
  static constexpr int kStage = QB > 1 ? 2 * KW * kHalf : 0;
  // Stages in LDS: four, or as many as leave room for a second workgroup on the CU.
  static constexpr int kRoom = (QB == 8 ? 152 : 80) * 1024;
  static constexpr int kStages = QB == 1 ? 0 : 4 * kStage <= kRoom ? 4 : 3 * kStage <= kRoom ? 3 : 2;
  static constexpr int kJoin = kWaves * kQueries * (kDims + 4 + 2) * 4;
  static constexpr int kRing = kStages * (kStage + kWaves * 256);  // and the table entries of each stage
  static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
  // Waves a SIMD that registers (and LDS) allow.
  static constexpr int kOccupancy = DV == 16 && QB < 4 ? 1 : DV * QT <= 4 ? 3 : 2;
};

// FULL: dim is 16 DV.
template <typename E, int DV, bool FULL, int QT, int QB>
__global__ void __launch_bounds__(QB == 8 ? 512 : 256, (Shape<DV, QT, QB>::kOccupancy)) tree_kernel(TreeArgs a) {
  using S = Shape<DV, QT, QB>;
  constexpr int KS = DV / 2;  // steps of 32 dims
  constexpr int kWaves = S::kWaves, KW = S::KW, kDims = S::kDims, kQueries = S::kQueries;
  extern __shared__ __align__(1024) uint8_t lds[];
  float* smem = reinterpret_cast<float*>(lds);
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t qb = wave % QB, kp = wave / QB;

  // Workgroups of the same rows and other queries run on the same XCD, one after
  // the other: the second finds its rows in the L2.
  const uint32_t unit = (blockIdx.x / 8 / a.query_groups) * 8 + blockIdx.x % 8;
  const uint32_t qg0 = blockIdx.x / 8 % a.query_groups;
  // Heads turn with the shares: eight heads would else be one on each XCD, whose rows,
  // 256 bytes of every 2 KiB, lie in two of its L2's sixteen channels.
  const uint32_t index = unit / a.kv_heads, h = (unit + index) % a.kv_heads;
  if (index >= a.shares) return;
  Share share(a, lane);
  if (!share.find(a, index, lane)) return;
  const uint32_t s = share.seq;
  const Tree tree(a, s);
  const uint32_t row0 = share.split * share.span;
  const uint32_t row1 = min(tree.rows, row0 + share.span);
  const uint32_t queries = tree.count * a.group;
  const PagedRows place{a.table + s * a.table_stride, a.table_cols, a.pages, a.page};
  const uint8_t* kbase = a.k + h * a.head_bytes;
  const uint8_t* vbase = a.v + h * a.head_bytes;

  // Lanes l and l + 32 look up row l of a chunk: the entry of its page (any entry
  // for rows past the end), then the row's offset in units of 16 bytes (of the
  // cache's first row, which every cache has, where there is none), and a bit for
  // each of the 32 rows that there is.
  auto entry = [&](uint32_t pos) { return place.table + place.page.quotient(min(pos + (lane & 31u), row1 - 1)); };
  auto resolve = [&](uint32_t pos, uint32_t page, uint32_t& off, uint32_t& there) {
    const uint32_t p = pos + (lane & 31u);
    const bool ok = p < row1 && page < a.pages;  // a negative id is past every page
    off = ok ? page * a.page_step + (p - place.page.quotient(p) * place.page.d) * a.row_step : 0u;
    there = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok));
  };
  auto row_offset = [&](uint32_t off, uint32_t row) {
    return static_cast<uint64_t>(static_cast<uint32_t>(
               __builtin_amdgcn_ds_bpermute(static_cast<int>(row * 4), static_cast<int>(off)))) * 16;
  };

  for (uint32_t qg = qg0; qg * (QB * kQueries) < queries; qg += a.query_groups) {
    const uint32_t q0 = (qg * QB + qb) * kQueries;
    // Q^T: lane (r, g) has dims 32 j + 8 g .. + 7 of query r.
    u32x4_t qf[QT][KS];
    uint32_t node[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const uint32_t i = min(q0 + 16 * t + r, queries - 1);
      node[t] = tree.first + i / a.group;
      const uint8_t* src = a.q + node[t] * a.q_node + (h * a.group + i % a.group) * a.q_head;
#pragma unroll
      for (int j = 0; j < KS; ++j) qf[t][j] = load_dims<FULL>(src, 32 * j + 8 * g, a.dim);
    }
    // Waits for Q in front of a loop: left to its first use in there, the wait would be
    // for every load in flight.
    auto have_q = [&]() {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int j = 0; j < KS; ++j) asm volatile("" : "+v"(qf[t][j]));
    };
    Sums<E, DV, QT> sums;
    sums.clear();
    bool odd_values = false;  // a masked chunk had infinities or NaN

    // Chunks that reach past the cached rows, or miss rows, are masked.
    auto is_masked = [&](uint32_t pos, uint32_t there) { return there != ~0u || pos + kChunk > tree.cached; };
    auto mask = [&](f32x4_t(&sc)[QT][2], uint32_t pos, uint32_t there) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const uint32_t seen =
            there & seen_bits(a.mask + static_cast<int64_t>(node[t]) * a.mask_words, a.mask_words, tree.cached, pos);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(seen >> row_of(g, e) & 1u)) sc[t][e / 4][e % 4] = -INFINITY;
      }
    };

    if constexpr (QB == 1) {
      u32x4_t kf[2][KS];
      auto load_k = [&](uint32_t off) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint8_t* src = kbase + row_offset(off, 16 * t + r);
#pragma unroll
          for (int j = 0; j < KS; ++j) kf[t][j] = load_dims<FULL>(src, 32 * j + 8 * g, a.dim);
        }
      };
      // Table entries are asked for a chunk before its K, and only looked at when that
      // is loaded: loads return in order, so looking at one waits for all before it.
      uint32_t pos = row0 + kp * kChunk, off = 0, there = 0, page = 0;
      if (pos < row1) {
        resolve(pos, *entry(pos), off, there);
        load_k(off);
        page = *entry(pos + KW * kChunk);
      }
      have_q();
      for (; pos < row1; pos += KW * kChunk) {
        uint32_t vr[8][DV / 2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint8_t* src = vbase + row_offset(off, row_of(g, e));
          if constexpr (DV == 4) {
            const bool on = FULL || 4 * r < a.dim;
            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(src + (on ? 8 * r : 0u));
            vr[e][0] = on ? w.x : 0u, vr[e][1] = on ? w.y : 0u;
          } else {
#pragma unroll
            for (int i = 0; i < DV / 8; ++i) {
              const u32x4_t w = load_dims<FULL>(src, 128 * i + 8 * r, a.dim);
              vr[e][4 * i] = w.x, vr[e][4 * i + 1] = w.y, vr[e][4 * i + 2] = w.z, vr[e][4 * i + 3] = w.w;
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t sc[QT][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][0] = sc[t][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KS; ++j)
          if (FULL || 32u * j < a.dim) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              sc[t][0] = E::mfma(kf[0][j], qf[t][j], sc[t][0]);
              sc[t][1] = E::mfma(kf[1][j], qf[t][j], sc[t][1]);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t there_now = there;
        resolve(pos + KW * kChunk, page, off, there);
        load_k(off);
        page = *entry(pos + 2 * KW * kChunk);
        if (is_masked(pos, there_now)) {
          mask(sc, pos, there_now);
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < DV / 2; ++i)
              bad = clean<E>(vr[e][i], there_now >> row_of(g, e) & 1u ? ~0u : 0u) || bad;
          odd_values = __builtin_amdgcn_ballot_w64(bad) != 0 || odd_values;
        }
        u32x4_t pf[QT];
        sums.soften(sc, a.scale, pf);
#pragma unroll
        for (int d = 0; d < DV; ++d) {
          u32x4_t v;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = __builtin_amdgcn_perm(vr[2 * i + 1][d / 2], vr[2 * i][d / 2], d % 2 ? 0x07060302u : 0x05040100u);
          sums.add(v, pf, d);
        }
      }
    } else {
      // Pieces of a chunk's K (and V) that a load of a wave brings: 1 KiB, kLines rows
      // of kSlots pieces of 16 bytes. Slot c of row i holds piece c ^ turn(i), which
      // spreads over all banks what 16 rows read at one piece.
      constexpr int kSlots = S::kRow / 16, kLines = 64 / kSlots, kLoads = S::kHalf / 1024 / QB;
      auto turn = [](uint32_t row) { return kSlots == 8 ? row >> 1 & 7u : row & 15u; };
      auto load_stage = [&](uint32_t slot, uint32_t off) {
        uint8_t* to = lds + slot * S::kStage + kp * (2 * S::kHalf);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const uint32_t p = i * QB + qb, row = p * kLines + lane / kSlots;
          const uint32_t piece = lane % kSlots ^ turn(row);
          const uint64_t at = row_offset(off, row) + 16 * piece;
          if (FULL || 8 * piece < a.dim) {
            load_to_lds(kbase + at, to + p * 1024);
            load_to_lds(vbase + at, to + S::kHalf + p * 1024);
          }
        }
      };
      // The table entries of a stage come to LDS too, kAhead stages before its rows are
      // asked for: an entry in a register would be waited for with all loads before it.
      constexpr int kAhead = S::kStages - 1;
      uint8_t* entries = lds + S::kStages * S::kStage + wave * (S::kStages * 256);
      auto load_entries = [&](uint32_t slot, uint32_t pos) {
        __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(
                                             reinterpret_cast<uintptr_t>(entry(pos))),
                                         (__attribute__((address_space(3))) uint32_t*)(entries + slot * 256), 4, 0, 0);
      };
      // Newer loads than a stage's own when it is waited for.
      constexpr int kNewer = (kAhead - 1) * (2 * kLoads + 1);
      __syncthreads();  // the previous query group has been written out
      constexpr uint32_t kStep = KW * kChunk;
      uint32_t pos = row0 + kp * kChunk, there[S::kStages];
      if (row0 < row1) {
        uint32_t page[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) page[i] = *entry(pos + i * kStep);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          uint32_t off;
          resolve(pos + i * kStep, page[i], off, there[i]);
          load_stage(i, off);
          load_entries((i + kAhead) % S::kStages, pos + (i + kAhead) * kStep);
        }
      }
      have_q();
      uint32_t slot = 0, slot_next = kAhead;
      for (uint32_t stage0 = row0; stage0 < row1; stage0 += kStep, pos += kStep) {
        // This wave's pieces of the stage have landed, then every wave's; and every
        // wave has left the stage in front, whose place the next loads take.
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kNewer) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        uint32_t off;
        resolve(pos + kAhead * kStep, reinterpret_cast<const uint32_t*>(entries + slot_next * 256)[lane], off,
                there[kAhead]);
        load_stage(slot_next, off);
        load_entries(slot == 0 ? S::kStages - 2 : slot == 1 ? S::kStages - 1 : slot - 2, pos + 2 * kAhead * kStep);
        const uint8_t* ks = lds + slot * S::kStage + kp * (2 * S::kHalf);
        const uint8_t* vs = ks + S::kHalf;
        slot = slot + 1 == S::kStages ? 0 : slot + 1;
        slot_next = slot_next + 1 == S::kStages ? 0 : slot_next + 1;

        // K at once, V while the products with K run.
        u32x4_t kf[2][KS];
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const uint32_t at = r * S::kRow + (((4 * j + g) ^ turn(r)) * 16);
          kf[0][j] = *reinterpret_cast<const u32x4_t*>(ks + at);
          kf[1][j] = *reinterpret_cast<const u32x4_t*>(ks + at + 16 * S::kRow);
          // Pieces past dim are not loaded: whatever lies there counts as zeros in K, and
          // in V goes to dims that are not stored.
          if (!FULL && 32 * j + 8 * g >= a.dim) kf[0][j] = kf[1][j] = u32x4_t{0, 0, 0, 0};
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t sc[QT][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][0] = sc[t][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KS; ++j)
          if (FULL || 32u * j < a.dim) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              sc[t][0] = E::mfma(kf[0][j], qf[t][j], sc[t][0]);
              sc[t][1] = E::mfma(kf[1][j], qf[t][j], sc[t][1]);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
        u32x4_t vf[DV];
        const uint32_t v_at = lds_offset(vs) + (4 * g + r / 4) * S::kRow + r % 2 * 8;
        const uint32_t v_piece = r % 4 / 2, v_turn = turn(4 * g + r / 4);
        uint32_t at[DV < 8 ? DV : 8];
#pragma unroll
        for (int d = 0; d < DV && d < 8; ++d) at[d] = v_at + ((2 * d + v_piece) ^ v_turn) * 16;
        if constexpr (DV == 4) {
          read_turned4<0, 16 * S::kRow>(vf, at);
        } else {
          read_turned8<0, 16 * S::kRow>(vf, at);
          if constexpr (DV == 16) read_turned8<256, 256 + 16 * S::kRow>(vf + 8, at);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (is_masked(pos, there[0])) {
          mask(sc, pos, there[0]);
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bits = there[0] >> row_of(g, 2 * i);
            const uint32_t on = (bits & 1u ? 0x0000ffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
#pragma unroll
            for (int d = 0; d < DV; ++d) {
              uint32_t w = vf[d][i];
              bad = clean<E>(w, FULL || 16 * d + r < a.dim ? on : 0u) || bad;
              vf[d][i] = w;
            }
          }
          odd_values = __builtin_amdgcn_ballot_w64(bad) != 0 || odd_values;
        }
        u32x4_t pf[QT];
        sums.soften(sc, a.scale, pf);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DV; ++d)
          if (FULL || 16u * d < a.dim) sums.add(vf[d], pf, d);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) there[i] = there[i + 1];
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may land in what follows
    }

    // Join the waves of a query block: a common maximum, then the sums in order.
    // smem: maximum and sum [waves][kQueries] each, then sums of V [waves][kQueries][kDims].
    float* s_top = smem;
    float* s_sum = smem + kWaves * kQueries;
    float* s_o = smem + 2 * kWaves * kQueries;
    __syncthreads();  // the stages, or the previous query group, are done with
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float total = across_groups_sum(sums.sum[t]);
      if (g == 0) {
        s_top[wave * kQueries + 16 * t + r] = sums.top[t];
        s_sum[wave * kQueries + 16 * t + r] = total;
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float m = sums.top[t];
#pragma unroll
      for (int w = 0; w < KW; ++w) m = fmaxf(m, s_top[(w * QB + qb) * kQueries + 16 * t + r]);
      const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sums.top[t] - m);
      // Lines of a query are shifted by four floats a query to spread the banks.
      float* dst = s_o + (wave * kQueries + 16 * t + r) * (kDims + 4);
      if constexpr (QB == 1) {  // element i of product d: dim 8 (4 g + i) + d of every 128, or 4 (4 g + i) + d
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DV; d += 4)
            *reinterpret_cast<f32x4_t*>(dst + (DV == 4 ? 4 * (4 * g + i) : 128 * (d / 8) + 8 * (4 * g + i) + d % 8)) =
                f32x4_t{sums.o[t][d][i] * f, sums.o[t][d + 1][i] * f, sums.o[t][d + 2][i] * f, sums.o[t][d + 3][i] * f};
      } else {  // dim 16 d + 4 g + i
#pragma unroll
        for (int d = 0; d < DV; ++d) *reinterpret_cast<f32x4_t*>(dst + 16 * d + 4 * g) = sums.o[t][d] * f;
      }
    }
    if (odd_values) {
      // Rare: the masked chunks' infinities and NaN, added to the sums of the
      // queries that see their rows, a query and a row at a time.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (uint32_t pos = row0 + kp * kChunk; pos < row1; pos += KW * kChunk) {
        uint32_t off, there;
        resolve(pos, *entry(pos), off, there);
        if (!is_masked(pos, there)) continue;
        for (uint32_t q = 0; q < kQueries && q0 + q < queries; ++q) {
          const int64_t n = tree.first + (q0 + q) / a.group;
          const uint32_t seen = there & seen_bits(a.mask + n * a.mask_words, a.mask_words, tree.cached, pos);
          for (uint32_t i = 0; i < kChunk; ++i) {
            const uint8_t* src = vbase + row_offset(off, i);
            for (uint32_t d = lane; d < a.dim; d += 64) {
              const uint32_t x = reinterpret_cast<const uint16_t*>(src)[d];
              if ((seen >> i & 1u) && (x & E::kExp) == E::kExp)
                s_o[(wave * kQueries + q) * (kDims + 4) + d] += E::value(x);
            }
          }
        }
      }
    }
    __syncthreads();
    // Thread: four dims of a query of the workgroup's QB * kQueries.
    constexpr int kPer = kDims / 4;
    for (uint32_t i = threadIdx.x; i < QB * kQueries * kPer; i += 64 * kWaves) {
      const uint32_t query = i / kPer, d = i % kPer * 4, b = query / kQueries, q = query % kQueries;
      const uint32_t at = qg * (QB * kQueries) + query;
      if (at >= queries || d >= a.dim) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < KW; ++w) m = fmaxf(m, s_top[(w * QB + b) * kQueries + q]);
      float total = 0.0f;
      f32x4_t v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t line = (w * QB + b) * kQueries + q;
        const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s_top[line] - m);
        total += s_sum[line] * f;
        v += *reinterpret_cast<const f32x4_t*>(s_o + line * (kDims + 4) + d);
      }
      const int64_t row = static_cast<int64_t>(tree.first + at / a.group) * a.heads + h * a.group + at % a.group;
      if (share.parts > 1) {
        const int64_t line = static_cast<int64_t>(share.line + share.split * tree.count) * a.heads +
                             (row - static_cast<int64_t>(tree.first) * a.heads);
        *reinterpret_cast<f32x4_t*>(a.part + line * a.dim + d) = v;
        if (d == 0) a.part_ml[line] = make_float2(m, total);
      } else {
        write<E>(a, row, d, v, m, total);
      }
    }
    if constexpr (QB == 1) __syncthreads();  // smem is read to its end before the next group's sums
  }
}

// ---- host ---------------------------------------------------------------------------

// How the queries and rows of a call are divided.
struct Plan {
  int dv, qt, qb;
  int64_t query_groups, step, least, want, shares, lines;
  bool by_work;
};

// `lines`: what the workspace holds. Wide rows take one tile of queries a wave:
// with two a SIMD has registers for one wave, which waits more than the two tiles
// save (two sequences of 65536 rows, 512 queries: 150 us against 109), and from five
// tiles on eight waves on the same rows, which halve what L2 gives out (82 us against
// 74; at dim 128, where two tiles a wave share rows already, no change).
Plan make_plan(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, int64_t max_len, int64_t max_tree,
               int64_t lines) {
  Plan p;
  p.dv = dim <= 64 ? 4 : dim <= 128 ? 8 : 16;
  const int64_t tiles = std::max<int64_t>(1, ceil_div(max_tree * (heads / kv_heads), 16));
  p.qt = tiles == 1 || p.dv == 16 ? 1 : 2;
  const int64_t blocks = ceil_div(tiles, p.qt);
  p.qb = blocks == 1 ? 1 : blocks == 2 ? 2 : blocks <= 4 || p.dv < 16 ? 4 : 8;
  p.query_groups = ceil_div(blocks, p.qb);
  p.step = kChunk * (p.qb == 8 ? 1 : 4 / p.qb);  // rows the workgroup takes at a time
  p.least = p.qb == 1 ? 1 : 4;
  // Shares for the workgroups that the CUs hold, or for a few rounds of them where the
  // sequences alone are more. A join costs as much as a few steps, so short sequences
  // stay whole, and so does one whose queries are a workgroup for every place (4096 nodes
  // over 16384 rows: 1949 us, split 2034).
  // From three rounds of whole sequences on a share is a place's part of all work: parts
  // are written and read again for little where lengths differ by a few times only, and
  // one sequence much longer than the others is all that waits in the end. Us with shares
  // as below three rounds, all whole, and so (32 heads, dim 128): 256 sequences of up to
  // 4096 rows, 25 nodes 794, 504, 540; 96 of 8192, 64 nodes 749, 611, 621; 200 of up to
  // 1000, one of 131072, a node each 224, 1660, 189; a chunk of 2048 nodes beside 30 of up
  // to 2000, one of 131072 1608, 4195, 723.
  p.want = 0, p.shares = seqs, p.lines = 0, p.by_work = false;
  const int64_t all = ((p.dv == 16 && p.qb < 4) || p.qb == 8 ? 1 : 2) * device_cu_count();
  const int64_t group = kv_heads * p.query_groups;  // workgroups of a share
  if (max_len <= 4 * p.step || seqs > kMostDealt || (seqs == 1 && group >= all)) return p;
  p.by_work = seqs * group >= 3 * all;
  const int64_t places = std::max<int64_t>(1, all / (p.by_work ? kv_heads : group));
  const int64_t want = p.by_work ? places : places * ceil_div(3 * seqs, 2 * places);
  const int64_t most =
      std::min({std::min(want + seqs, 2 * want) * max_tree, lines, kMostBytes / line_bytes(heads, dim)});
  if (want > 1 && most > 1) p.want = want, p.shares = want + seqs, p.lines = most;
  return p;
}

template <typename E, int DV, bool FULL, int QT, int QB>
int launch(const TreeArgs& a, const Plan& p, hipStream_t s) {
  const void* fn = reinterpret_cast<const void*>(&tree_kernel<E, DV, FULL, QT, QB>);
  constexpr int lds = Shape<DV, QT, QB>::kBytes;
  const int rc = allow_dynamic_lds(fn, lds);
  if (rc != SPIRAL_OK) return rc;
  const int64_t units = ceil_div(p.shares * a.kv_heads, 8) * 8;
  if (units * p.query_groups > INT32_MAX) return SPIRAL_ERR_SHAPE;
  hipLaunchKernelGGL((tree_kernel<E, DV, FULL, QT, QB>), dim3(static_cast<unsigned>(units * p.query_groups)),
                     dim3(64 * Shape<DV, QT, QB>::kWaves), lds, s, a);
  return launch_status();
}

template <typename E, int DV, bool FULL>
int launch_tiles(const TreeArgs& a, const Plan& p, hipStream_t s) {
  constexpr int QT = DV == 16 ? 1 : 2;
  if (p.qt == 1 && p.qb == 1) return launch<E, DV, FULL, 1, 1>(a, p, s);
  if constexpr (DV != 16) {
    if (p.qb == 1) return launch<E, DV, FULL, QT, 1>(a, p, s);
  }
  if constexpr (DV == 16) {
    if (p.qb == 8) return launch<E, DV, FULL, QT, 8>(a, p, s);
  }
  return p.qb == 2 ? launch<E, DV, FULL, QT, 2>(a, p, s) : launch<E, DV, FULL, QT, 4>(a, p, s);
}

template <typename E>
int run_tree(const TreeArgs& a, const Plan& p, int64_t max_tree, hipStream_t s) {
  const bool full = static_cast<int>(a.dim) == 16 * p.dv;
#define SPIRAL_TREE(DV) (full ? launch_tiles<E, DV, true>(a, p, s) : launch_tiles<E, DV, false>(a, p, s))
  const int rc = p.dv == 4 ? SPIRAL_TREE(4) : p.dv == 8 ? SPIRAL_TREE(8) : SPIRAL_TREE(16);
#undef SPIRAL_TREE
  if (rc != SPIRAL_OK || p.want == 0) return rc;
  return launch_join<E>(a, static_cast<uint32_t>(p.want), max_tree, s);
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int64_t spiral_tree_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs,
                                              int64_t max_len, int64_t max_tree) {
  if (!sizes_ok(0, heads, kv_heads, dim, seqs, max_len, max_tree)) return 0;
  const Plan p = make_plan(heads, kv_heads, dim, seqs, max_len, max_tree, INT64_MAX);
  return p.lines * line_bytes(heads, dim);
}

int spiral_tree_attention(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                          int64_t heads, const void* k, const void* v, int64_t pages, int64_t page, int64_t kv_heads,
                          int64_t dim, int64_t page_stride, int64_t row_stride, int64_t head_stride,
                          const int32_t* table, int64_t table_stride, int64_t table_cols, const int32_t* lens,
                          const int32_t* cu, int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len,
                          int64_t max_tree, float scale, void* out, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  if (type != SPIRAL_TYPE_BF16 && type != SPIRAL_TYPE_F16) return SPIRAL_ERR_TYPE;
  if (!sizes_ok(nodes, heads, kv_heads, dim, seqs, max_len, max_tree) || pages <= 0 || pages > INT32_MAX || page <= 0 ||
      page > INT32_MAX || table_cols < 0 || table_cols > INT32_MAX || table_stride < table_cols ||
      table_stride > INT32_MAX || mask_words < 0 || mask_words > (1 << 18) || !std::isfinite(scale) || scale <= 0.0f)
    return SPIRAL_ERR_SHAPE;
  const int64_t strides[] = {q_node_stride, q_head_stride, page_stride, row_stride, head_stride};
  for (int64_t v8 : strides)
    if (v8 < 0 || v8 > (int64_t(1) << 40)) return SPIRAL_ERR_SHAPE;
  for (int64_t v8 : strides)
    if (v8 % 8 != 0) return SPIRAL_ERR_ALIGN;
  // Rows are addressed in 32 bits of 16-byte units (64 GiB of keys or of values).
  int64_t a0 = 0, a1 = 0;
  if (__builtin_mul_overflow(pages, page_stride / 8, &a0) || __builtin_mul_overflow(page, row_stride / 8, &a1) ||
      a0 > UINT32_MAX || a1 > UINT32_MAX || a0 + a1 > UINT32_MAX)
    return SPIRAL_ERR_SHAPE;
  if (nodes == 0 || seqs == 0 || max_tree == 0) return SPIRAL_OK;
  if (q == nullptr || k == nullptr || v == nullptr || (table == nullptr && table_cols > 0) || lens == nullptr ||
      cu == nullptr || (mask == nullptr && mask_words > 0) || out == nullptr)
    return SPIRAL_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(mask) & 7u) != 0 ||
      ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(cu) |
        reinterpret_cast<uintptr_t>(lse)) & 3u) != 0)
    return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const int64_t lines = workspace == nullptr || workspace_bytes < 0 ? 0 : workspace_bytes / line_bytes(heads, dim);
  const Plan p = make_plan(heads, kv_heads, dim, seqs, max_len, max_tree, lines);
  TreeArgs a{static_cast<const uint8_t*>(q), q_node_stride * 2, q_head_stride * 2, static_cast<uint32_t>(nodes),
             static_cast<uint32_t>(heads), static_cast<uint32_t>(heads / kv_heads), static_cast<const uint8_t*>(k),
             static_cast<const uint8_t*>(v), static_cast<uint32_t>(pages), static_cast<uint32_t>(kv_heads),
             static_cast<uint32_t>(dim), static_cast<uint32_t>(page_stride / 8), static_cast<uint32_t>(row_stride / 8),
             head_stride * 2, Divisor(static_cast<uint32_t>(page)), table, table_stride,
             static_cast<uint32_t>(table_cols), lens, cu, static_cast<uint32_t>(seqs), mask,
             static_cast<uint32_t>(mask_words), scale * kLog2e, static_cast<uint8_t*>(out), lse, nullptr, nullptr,
             static_cast<uint32_t>(p.lines), static_cast<uint32_t>(max_tree), static_cast<uint32_t>(p.query_groups),
             static_cast<uint32_t>(p.shares), static_cast<uint32_t>(p.want), static_cast<uint32_t>(p.step),
             static_cast<uint32_t>(p.least), p.by_work, Divisor(static_cast<uint32_t>(16 * p.qt * p.qb))};
  if (p.want > 0) {
    a.part = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part + p.lines * heads * dim);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return type == SPIRAL_TYPE_BF16 ? run_tree<Bf16>(a, p, max_tree, s) : run_tree<F16>(a, p, max_tree, s);
}

}  // extern "C"

// Which cached rows stay (spiral_cache.h): the first, the latest, and of the others those
// of most weight.
//
// Weights are compared as numbers that order as they do, the first and
// the latest rows as the largest number there is, so that all that is left is the `budget`
// largest. The smallest that stays is found digit by digit from the top (11, 11 and 10 bits): a
// histogram in LDS of the rows that share the digits found so far, and from its upper end
// the digit in which the wanted count falls. Then every wave counts what stays of its
// stretch of rows, and writes it behind what the waves in front of it keep: rows come out in
// order, and of equal weights the first ones stay.
//
// A workgroup a sequence, its rows in registers: barriers bound the short ones (4096 rows: 9 us),
// and one CU's 12 bytes a clock the long ones (65536: 38 us, 10 of them the first load). Few long
// ones are divided over workgroups, which find each digit in a launch of their own, up to the
// 983040 rows that their parts can count; longer ones are a workgroup's again, 1.4 ms a million rows.
#include "common.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;
constexpr int kCopies = 4;  // of the histogram, for lanes that count the same digit
constexpr int kSteps = 64;  // rows a thread keeps in registers: 65536 of a sequence

struct EvictArgs {
  const float* mass;
  int64_t mass_stride;
  uint32_t cols;
  const int32_t* lens;
  uint32_t budget, sinks, recent;
  int32_t* keep;
  int64_t keep_stride;
  int32_t* kept;
  float* new_mass;
  int64_t new_stride;
  uint8_t* work;  // of divided sequences, kWorkBytes each
};

// A divided sequence's workspace: of each part, how many rows have each digit, two counts a
// word, in three passes; the rows above the first two digits; what the passes have found.
constexpr uint32_t kParts = 16, kMostRows = 60 * 1024;  // of a part: counts of 16 bits
struct Work {
  uint32_t counts[3][kParts][kBins / 2];
  uint32_t above[kParts];
  uint32_t prefix[2], want[2];
};

// Weights as numbers that order as they do: NaN on top, -0 as +0. No weight is 0 or ~0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return ~1u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 is +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over this lane and those below it.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROW_MASK, 0xF, false));
}
__device__ __forceinline__ uint32_t sum_upto(uint32_t v) {
  v += moved<0x111, 0xF>(v);  // row_shr 1
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15: row 0 into row 1, row 2 into row 3
  v += moved<0x143, 0xC>(v);  // row_bcast 31: rows 0-1 into rows 2 and 3
  return v;
}

// Bits of m below this lane's.
__device__ __forceinline__ uint32_t below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(m >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(m), 0u));
}

// Thread t has c0 and c1 rows in the bins kBins - 1 - 2 t and the next lower: the bin in which `want`
// rows from the upper end on are reached, and how many of its rows are among them.
__device__ __forceinline__ uint2 pick(uint32_t c0, uint32_t c1, uint32_t want, uint32_t* s_wave, uint32_t* s_found) {
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t hi = kBins - 1 - 2 * threadIdx.x, x = sum_upto(c0 + c1);
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  // The wave sums in front of this wave, a wave a lane.
  const uint32_t upto = sum_upto(lane < kWaves ? s_wave[lane] : 0u);
  const uint32_t before = x - c0 - c1 + (wave > 0 ? __builtin_amdgcn_readlane(upto, (wave - 1) & 63) : 0u);
  if (before < want && want <= before + c0) s_found[0] = hi, s_found[1] = want - before;
  if (before + c0 < want && want <= before + c0 + c1) s_found[0] = hi - 1, s_found[1] = want - before - c0;
  __syncthreads();
  return make_uint2(s_found[0], s_found[1]);
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
  __shared__ __align__(16) uint32_t s_bins[kBins][kCopies];
  __shared__ uint32_t s_wave[2][kWaves];
  __shared__ uint32_t s_found[2];  // the digit, and how many of it are wanted
  const uint32_t s = blockIdx.x, lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n = static_cast<uint32_t>(min(max(a.lens[s], 0), static_cast<int32_t>(a.cols)));
  const float* mass = a.mass + s * a.mass_stride;
  int32_t* keep = a.keep + s * a.keep_stride;
  float* out = a.new_mass == nullptr ? nullptr : a.new_mass + s * a.new_stride;
  const uint32_t kept = min(n, a.budget);
  if (threadIdx.x == 0) a.kept[s] = static_cast<int32_t>(kept);
  for (uint32_t i = kept + threadIdx.x; i < a.budget; i += kThreads) keep[i] = -1;
  if (out != nullptr)
    for (uint32_t i = kept + threadIdx.x; i < a.cols; i += kThreads) out[i] = 0.0f;
  if (n <= a.budget) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      keep[i] = static_cast<int32_t>(i);
      if (out != nullptr) out[i] = mass[i];
    }
    return;
  }
  // Wave w has rows w * per .. + per - 1, 64 at a time, and keeps those of its first kSteps steps
  // in registers. Lanes past them have 0, below every weight.
  const uint32_t per = (n + kThreads - 1) / kThreads * 64, from = min(n, wave * per), to = min(n, from + per);
  auto key_at = [&](uint32_t i, float x) {
    const uint32_t key = i < a.sinks || i >= n - a.recent ? ~0u : key_of(x);
    return i < to ? key : 0u;
  };
  uint32_t held[kSteps];
#pragma unroll
  for (int b = 0; b < kSteps; b += 8) {
    if (b * 64u < per) {
#pragma unroll
      for (int j = b; j < b + 8; ++j) held[j] = __float_as_uint(mass[min(from + j * 64 + lane, n - 1)]);
    }
  }
#pragma unroll
  for (int b = 0; b < kSteps; b += 8) {
    if (b * 64u < per) {
#pragma unroll
      for (int j = b; j < b + 8; ++j) held[j] = key_at(from + j * 64 + lane, __uint_as_float(held[j]));
    }
  }
  // Calls f(first row of a step, this lane's key) for every step of the wave.
  auto each = [&](auto f) {
#pragma unroll
    for (int b = 0; b < kSteps; b += 8) {
      if (b * 64u < per) {
#pragma unroll
        for (int j = b; j < b + 8; ++j) f(from + j * 64, held[j]);
      }
    }
    for (uint32_t i0 = from + kSteps * 64; i0 < to; i0 += 64) f(i0, key_at(i0 + lane, mass[min(i0 + lane, n - 1)]));
  };

  uint32_t prefix = 0, known = 0, want = a.budget;  // the digits found, their bits, rows wanted of them
  if (want > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      constexpr uint32_t kBits[] = {11, 11, 10};
      const uint32_t bits = kBits[pass], shift = 32 - known - bits;
      for (uint32_t i = threadIdx.x; i < kBins * kCopies / 4; i += kThreads)
        reinterpret_cast<u32x4_t*>(s_bins)[i] = u32x4_t{0, 0, 0, 0};
      __syncthreads();
      each([&](uint32_t, uint32_t key) {
        if (pass == 0 || key >> (shift + bits) == prefix)
          atomicAdd(&s_bins[key >> shift & ((1u << bits) - 1)][lane % kCopies], 1u);
      });
      __syncthreads();
      // Thread t has the bins 2 t and 2 t + 1 from the upper end.
      const uint32_t hi = kBins - 1 - 2 * threadIdx.x;
      uint32_t c0 = 0, c1 = 0;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) c0 += s_bins[hi][c], c1 += s_bins[hi - 1][c];
      const uint2 found = pick(c0, c1, want, s_wave[0], s_found);
      prefix = prefix << bits | found.x, want = found.y, known += bits;
    }
  } else {
    prefix = ~0u;  // above every row: a budget of none has neither first nor latest ones
  }
  // Above `prefix` rows stay, and of those equal to it the first `want`.
  uint32_t n_more = 0, n_same = 0;
  each([&](uint32_t, uint32_t key) {
    n_more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > prefix));
    n_same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key == prefix));
  });
  __syncthreads();  // s_wave has been read
  if (lane == 0) s_wave[0][wave] = n_more, s_wave[1][wave] = n_same;
  __syncthreads();
  const uint32_t all_more = sum_upto(lane < kWaves ? s_wave[0][lane] : 0u);
  const uint32_t all_same = sum_upto(lane < kWaves ? s_wave[1][lane] : 0u);
  uint32_t at_more = wave > 0 ? __builtin_amdgcn_readlane(all_more, (wave - 1) & 63) : 0u;
  uint32_t at_same = wave > 0 ? __builtin_amdgcn_readlane(all_same, (wave - 1) & 63) : 0u;
  each([&](uint32_t i0, uint32_t key) {
    const uint64_t more = __builtin_amdgcn_ballot_w64(key > prefix), same = __builtin_amdgcn_ballot_w64(key == prefix);
    const uint32_t q = at_same + below(same);
    if (key > prefix || (key == prefix && q < want)) keep[at_more + below(more) + min(q, want)] = static_cast<int32_t>(i0 + lane);
    at_more += __builtin_popcountll(more), at_same += __builtin_popcountll(same);
  });
  if (out == nullptr) return;
  // The masses in their new places, eight loads in flight a thread.
  __syncthreads();
  for (uint32_t j0 = threadIdx.x; j0 < kept; j0 += 8 * kThreads) {
    uint32_t row[8];
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) row[j] = static_cast<uint32_t>(keep[min(j0 + j * kThreads, kept - 1)]);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = mass[row[j]];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j0 + j * kThreads < kept) out[j0 + j * kThreads] = x[j];
  }
}

// The same by kParts workgroups a sequence and four launches: each but the last counts the rows'
// next digit in its part, and each but the first adds up what the one in front counted. The last
// knows from the counts what the parts in front keep, and writes.
template <int PASS>
__global__ void __launch_bounds__(kThreads) evict_part_kernel(EvictArgs a) {
  __shared__ __align__(16) uint32_t s_bins[kBins][kCopies];
  __shared__ uint32_t s_wave[2][kWaves];
  __shared__ uint32_t s_found[2];
  const uint32_t s = blockIdx.y, part = blockIdx.x, lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n = static_cast<uint32_t>(min(max(a.lens[s], 0), static_cast<int32_t>(a.cols)));
  const float* mass = a.mass + s * a.mass_stride;
  int32_t* keep = a.keep + s * a.keep_stride;
  float* out = a.new_mass == nullptr ? nullptr : a.new_mass + s * a.new_stride;
  Work& work = reinterpret_cast<Work*>(a.work)[s];
  const uint32_t kept = min(n, a.budget);
  if constexpr (PASS == 0) {
    const uint32_t first = part * kThreads + threadIdx.x, step = kParts * kThreads;
    if (first == 0) a.kept[s] = static_cast<int32_t>(kept);
    for (uint32_t i = kept + first; i < a.budget; i += step) keep[i] = -1;
    if (out != nullptr)
      for (uint32_t i = kept + first; i < a.cols; i += step) out[i] = 0.0f;
    if (n <= a.budget)
      for (uint32_t i = first; i < n; i += step) {
        keep[i] = static_cast<int32_t>(i);
        if (out != nullptr) out[i] = mass[i];
      }
  }
  if (n <= a.budget) return;

  // The part's rows, as a sequence's in evict_kernel: the first kHeld steps of a wave in registers.
  constexpr int kHeld = 8;
  const uint32_t rows = (n + kParts * kThreads - 1) / (kParts * kThreads) * kThreads;
  const uint32_t per = rows / kWaves, from = min(n, part * rows + wave * per), to = min(n, from + per);
  float held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = j * 64u < per ? mass[min(from + j * 64 + lane, n - 1)] : 0.0f;
  auto each = [&](auto f) {
    auto one = [&](uint32_t i0, float x) {
      const uint32_t i = i0 + lane, key = i < a.sinks || i >= n - a.recent ? ~0u : key_of(x);
      f(i, i < to ? key : 0u, x);
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j * 64u < per) one(from + j * 64, held[j]);
    for (uint32_t i0 = from + kHeld * 64; i0 < to; i0 += 64) one(i0, mass[min(i0 + lane, n - 1)]);
  };

  // The digit of the launch in front: a thread adds up two bins of all parts, and of those in
  // front of this one.
  constexpr uint32_t kBits[] = {11, 11, 10, 0}, kKnown[] = {0, 11, 22, 32};
  uint32_t prefix = 0, want = a.budget, front = 0, front_same = 0;
  if constexpr (PASS > 0) {
    if constexpr (PASS > 1) prefix = work.prefix[PASS - 2], want = work.want[PASS - 2];
    const uint32_t word = kBins / 2 - 1 - threadIdx.x;
    uint32_t c[kParts], c0 = 0, c1 = 0;
#pragma unroll
    for (uint32_t j = 0; j < kParts; ++j) c[j] = work.counts[PASS - 1][j][word];
#pragma unroll
    for (uint32_t j = 0; j < kParts; ++j) c0 += c[j] >> 16, c1 += c[j] & 0xffffu;
    const uint2 found = pick(c0, c1, want, s_wave[0], s_found);
    if constexpr (PASS == 3) {
#pragma unroll
      for (uint32_t j = 0; j < kParts; ++j) {
        if (j >= part) continue;
        const uint32_t upper = c[j] >> 16, lower = c[j] & 0xffffu;
        front += (2 * word + 1 > found.x ? upper : 0u) + (2 * word > found.x ? lower : 0u);
        front_same += (2 * word + 1 == found.x ? upper : 0u) + (2 * word == found.x ? lower : 0u);
      }
      if (threadIdx.x < part) front += work.above[threadIdx.x];
    }
    prefix = prefix << kBits[PASS - 1] | found.x, want = found.y;
    if constexpr (PASS < 3) {
      if (part == 0 && threadIdx.x == 0) work.prefix[PASS - 1] = prefix, work.want[PASS - 1] = want;
    }
  }
  if constexpr (PASS < 3) {
    constexpr uint32_t bits = kBits[PASS], shift = 32 - kKnown[PASS] - bits;
    for (uint32_t i = threadIdx.x; i < kBins * kCopies / 4; i += kThreads)
      reinterpret_cast<u32x4_t*>(s_bins)[i] = u32x4_t{0, 0, 0, 0};
    __syncthreads();
    uint32_t n_above = 0;
    each([&](uint32_t, uint32_t key, float) {
      const uint32_t top = PASS == 0 ? 0u : key >> ((shift + bits) & 31);
      if (top == prefix) atomicAdd(&s_bins[key >> shift & ((1u << bits) - 1)][lane % kCopies], 1u);
      if (PASS == 2) n_above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(top > prefix));
    });
    if (PASS == 2 && lane == 0) s_wave[1][wave] = n_above;
    __syncthreads();
    uint32_t pair[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < kCopies; ++c) pair[0] += s_bins[2 * threadIdx.x][c], pair[1] += s_bins[2 * threadIdx.x + 1][c];
    work.counts[PASS][part][threadIdx.x] = pair[0] | pair[1] << 16;
    if (PASS == 2 && threadIdx.x == 0) {
      uint32_t all = 0;
      for (int w = 0; w < kWaves; ++w) all += s_wave[1][w];
      work.above[part] = all;
    }
  } else {
    // What the parts in front keep, and what this one's waves do.
    uint32_t n_more = 0, n_same = 0;
    each([&](uint32_t, uint32_t key, float) {
      n_more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > prefix));
      n_same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key == prefix));
    });
    front = sum_upto(front), front_same = sum_upto(front_same);
    __shared__ uint32_t s_front[2][kWaves];
    __syncthreads();  // s_wave has been read
    if (lane == 63) s_front[0][wave] = front, s_front[1][wave] = front_same;
    if (lane == 0) s_wave[0][wave] = n_more, s_wave[1][wave] = n_same;
    __syncthreads();
    auto of_waves = [&](const uint32_t* v, uint32_t waves) {
      return __builtin_amdgcn_readlane(sum_upto(lane < waves ? v[lane & (kWaves - 1)] : 0u), 63);
    };
    uint32_t at_more = of_waves(s_front[0], kWaves) + of_waves(s_wave[0], wave);
    uint32_t at_same = of_waves(s_front[1], kWaves) + of_waves(s_wave[1], wave);
    each([&](uint32_t i, uint32_t key, float x) {
      const uint64_t more = __builtin_amdgcn_ballot_w64(key > prefix), same = __builtin_amdgcn_ballot_w64(key == prefix);
      const uint32_t q = at_same + below(same);
      if (key > prefix || (key == prefix && q < want)) {
        const uint32_t to_row = at_more + below(more) + min(q, want);
        keep[to_row] = static_cast<int32_t>(i);
        if (out != nullptr) out[to_row] = x;
      }
      at_more += __builtin_popcountll(more), at_same += __builtin_popcountll(same);
    });
  }
}

// Three more launches cost 10 us, and every sequence some; a workgroup of its own takes 0.5 us
// a 1000 rows, three times that behind the 65536 that its registers hold. us whole and divided: one
// sequence of 16384 rows 13.4 and 15.4, of 32768 21.4 and 16.1, of 900000 1176 and 75; eight of 20000
// 18.0 and 18.3, of 65536 38.0 and 20.0; 64 of 65536 39.6 and 48.7, of 100000 89 and 61. Parts end
// with their 16-bit counts: one of 983040 81 us divided, of 983041 1370 whole.
bool divided(int64_t cols, int64_t seqs) { return cols > 16384 + 768 * seqs && cols <= int64_t(kParts) * kMostRows; }

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int64_t spiral_cache_evict_workspace_bytes(int64_t mass_cols, int64_t seqs) {
  if (seqs <= 0 || seqs > 65535 || mass_cols <= 0) return 0;
  return divided(mass_cols, seqs) ? seqs * static_cast<int64_t>(sizeof(Work)) : 0;
}

int spiral_cache_evict(const float* mass, int64_t mass_stride, int64_t mass_cols, const int32_t* lens, int64_t seqs,
                       int64_t budget, int64_t sinks, int64_t recent, int32_t* keep, int64_t keep_stride,
                       int32_t* kept, float* new_mass, int64_t new_stride, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  if (seqs < 0 || seqs > 65535 || mass_cols < 0 || mass_cols > INT32_MAX / 2 || mass_stride < mass_cols ||
      mass_stride > (int64_t(1) << 40) || budget < 0 || budget > INT32_MAX / 2 || sinks < 0 || recent < 0 ||
      sinks > budget || recent > budget - sinks || keep_stride < budget || keep_stride > INT32_MAX ||
      (new_mass != nullptr && (new_stride < mass_cols || new_stride > (int64_t(1) << 40))))
    return SPIRAL_ERR_SHAPE;
  if (seqs == 0) return SPIRAL_OK;
  if ((mass == nullptr && mass_cols > 0) || lens == nullptr || kept == nullptr || (keep == nullptr && budget > 0))
    return SPIRAL_ERR_NULL;
  if (!words_aligned({mass, lens, keep, kept, new_mass}) || !aligned16(workspace)) return SPIRAL_ERR_ALIGN;
  if (new_mass != nullptr && new_mass == mass) return SPIRAL_ERR_SHAPE;  // other waves still read it
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const EvictArgs a{mass, mass_stride, static_cast<uint32_t>(mass_cols), lens, static_cast<uint32_t>(budget),
                    static_cast<uint32_t>(sinks), static_cast<uint32_t>(recent), keep, keep_stride, kept, new_mass,
                    new_stride, static_cast<uint8_t*>(workspace)};
  const hipStream_t stream_of = static_cast<hipStream_t>(stream);
  const int64_t need = spiral_cache_evict_workspace_bytes(mass_cols, seqs);
  if (need > 0 && budget > 0 && budget < mass_cols && workspace != nullptr && workspace_bytes >= need) {
    const dim3 grid(kParts, static_cast<unsigned>(seqs)), threads(kThreads);
    hipLaunchKernelGGL(evict_part_kernel<0>, grid, threads, 0, stream_of, a);
    hipLaunchKernelGGL(evict_part_kernel<1>, grid, threads, 0, stream_of, a);
    hipLaunchKernelGGL(evict_part_kernel<2>, grid, threads, 0, stream_of, a);
    hipLaunchKernelGGL(evict_part_kernel<3>, grid, threads, 0, stream_of, a);
  } else {
    hipLaunchKernelGGL(evict_kernel, dim3(static_cast<unsigned>(seqs)), dim3(kThreads), 0, stream_of, a);
  }
  return launch_status();
}

}  // extern "C"

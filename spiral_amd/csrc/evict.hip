// Which cached rows stay (spiral_cache.h): the first, the latest, and of the others those
// of most weight.
//
// A workgroup a sequence. Weights are compared as numbers that order as they do, the first and
// the latest rows as the largest number there is, so that all that is left is the `budget`
// largest. The smallest that stays is found digit by digit from the top (11, 11 and 10 bits): a
// histogram in LDS of the rows that share the digits found so far, and from its upper end
// the digit in which the wanted count falls. Then every wave counts what stays of its
// stretch of rows, and writes it behind what the waves in front of it keep: rows come out in
// order, and of equal weights the first ones stay.
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
      const uint32_t x = sum_upto(c0 + c1);
      if (lane == 63) s_wave[0][wave] = x;
      __syncthreads();
      // The wave sums in front of this wave, a wave a lane.
      const uint32_t upto = sum_upto(lane < kWaves ? s_wave[0][lane] : 0u);
      const uint32_t before = x - c0 - c1 + (wave > 0 ? __builtin_amdgcn_readlane(upto, (wave - 1) & 63) : 0u);
      if (before < want && want <= before + c0) s_found[0] = hi, s_found[1] = want - before;
      if (before + c0 < want && want <= before + c0 + c1) s_found[0] = hi - 1, s_found[1] = want - before - c0;
      __syncthreads();
      prefix = prefix << bits | s_found[0], want = s_found[1], known += bits;
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

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" int spiral_cache_evict(const float* mass, int64_t mass_stride, int64_t mass_cols, const int32_t* lens,
                                  int64_t seqs, int64_t budget, int64_t sinks, int64_t recent, int32_t* keep,
                                  int64_t keep_stride, int32_t* kept, float* new_mass, int64_t new_stride,
                                  void* stream) {
  if (seqs < 0 || seqs > 65535 || mass_cols < 0 || mass_cols > INT32_MAX / 2 || mass_stride < mass_cols ||
      mass_stride > (int64_t(1) << 40) || budget < 0 || budget > INT32_MAX / 2 || sinks < 0 || recent < 0 ||
      sinks > budget || recent > budget - sinks || keep_stride < budget || (new_mass != nullptr && (new_stride < mass_cols || new_stride > (int64_t(1) << 40))) || keep_stride > INT32_MAX)
    return SPIRAL_ERR_SHAPE;
  if (seqs == 0) return SPIRAL_OK;
  if ((mass == nullptr && mass_cols > 0) || lens == nullptr || kept == nullptr || (keep == nullptr && budget > 0))
    return SPIRAL_ERR_NULL;
  if (!words_aligned({mass, lens, keep, kept, new_mass})) return SPIRAL_ERR_ALIGN;
  if (new_mass != nullptr && new_mass == mass) return SPIRAL_ERR_SHAPE;  // other waves still read it
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const EvictArgs a{mass, mass_stride, static_cast<uint32_t>(mass_cols), lens, static_cast<uint32_t>(budget),
                    static_cast<uint32_t>(sinks), static_cast<uint32_t>(recent), keep, keep_stride, kept, new_mass, new_stride};
  hipLaunchKernelGGL(evict_kernel, dim3(static_cast<unsigned>(seqs)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return launch_status();
}

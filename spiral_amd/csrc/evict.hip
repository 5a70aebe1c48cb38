// Which cached rows stay (spiral_cache.h): the first, the latest, and of the others those
// of most weight.
//
// A workgroup a sequence. The smallest weight that stays is found digit by digit from the
// top (11, 11 and 10 bits of the weight as a number that orders as it does): a histogram in
// LDS of the rows that share the digits found so far, and from its upper end the digit in
// which the wanted count falls. Then every wave counts what stays of its stretch of rows,
// and writes it behind what the waves in front of it keep: rows come out in order, and of
// equal weights the first ones stay.
#include "common.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

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

// Weights as numbers that order as they do: NaN on top, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return ~0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 is +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
  __shared__ uint32_t s_bins[kBins];
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
  const uint32_t first = a.sinks, last = n - a.recent;  // the rows that compete
  uint32_t want = a.budget - a.sinks - a.recent;

  uint32_t prefix = 0, known = 0;  // the digits found, and their bits
  if (want > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const uint32_t bits = pass < 2 ? 11u : 10u, shift = 32 - known - bits;
      for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) s_bins[i] = 0;
      __syncthreads();
      for (uint32_t i0 = first + wave * 64; i0 < last; i0 += kThreads) {
        const uint32_t i = i0 + lane;
        const uint32_t key = key_of(mass[min(i, last - 1)]);
        const bool on = i < last && (known == 0 || key >> (32 - known) == prefix);
        const uint32_t digit = key >> shift & ((1u << bits) - 1);
        // Rows of one digit only (weights of nothing, as a rule) would go one after the other.
        const uint64_t some = __builtin_amdgcn_ballot_w64(on);
        if (some == 0) continue;
        const uint32_t lead = __builtin_amdgcn_readlane(digit, __builtin_ctzll(some));
        if (__builtin_amdgcn_ballot_w64(on && digit == lead) == some) {
          if (lane == 0) atomicAdd(&s_bins[lead], static_cast<uint32_t>(__builtin_popcountll(some)));
        } else if (on) {
          atomicAdd(&s_bins[digit], 1u);
        }
      }
      __syncthreads();
      // Thread t has the bins 2 t and 2 t + 1 from the upper end.
      const uint32_t hi = kBins - 1 - 2 * threadIdx.x, c0 = s_bins[hi], c1 = s_bins[hi - 1];
      uint32_t x = c0 + c1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o, 64);
        if (lane >= static_cast<uint32_t>(o)) x += y;
      }
      if (lane == 63) s_wave[0][wave] = x;
      __syncthreads();
      uint32_t before = x - c0 - c1;
      for (uint32_t w = 0; w < wave; ++w) before += s_wave[0][w];
      if (before < want && want <= before + c0) s_found[0] = hi, s_found[1] = want - before;
      if (before + c0 < want && want <= before + c0 + c1) s_found[0] = hi - 1, s_found[1] = want - before - c0;
      __syncthreads();
      prefix = prefix << bits | s_found[0], want = s_found[1], known += bits;
    }
  }
  // Above `prefix` rows stay, and of those equal to it the first `want`.
  const bool none = a.budget == a.sinks + a.recent;
  const uint32_t per = (n + kThreads - 1) / kThreads * 64;  // rows of a wave
  const uint32_t from = min(n, wave * per), to = min(n, from + per);
  auto kinds = [&](uint32_t i, bool& more, bool& same, float& x) {
    const bool on = i < to;
    x = mass[min(i, n - 1)];
    const uint32_t key = key_of(x);
    const bool fixed = i < first || i >= last;
    more = on && (fixed || (!none && key > prefix));
    same = on && !fixed && !none && key == prefix;
  };
  uint32_t n_more = 0, n_same = 0;
  for (uint32_t i0 = from; i0 < to; i0 += 64) {
    bool more, same;
    float x;
    kinds(i0 + lane, more, same, x);
    n_more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(more));
    n_same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(same));
  }
  __syncthreads();  // s_wave has been read
  if (lane == 0) s_wave[0][wave] = n_more, s_wave[1][wave] = n_same;
  __syncthreads();
  uint32_t at_more = 0, at_same = 0;
  for (uint32_t w = 0; w < wave; ++w) at_more += s_wave[0][w], at_same += s_wave[1][w];
  for (uint32_t i0 = from; i0 < to; i0 += 64) {
    bool more, same;
    float x;
    kinds(i0 + lane, more, same, x);
    const uint64_t b_more = __builtin_amdgcn_ballot_w64(more), b_same = __builtin_amdgcn_ballot_w64(same);
    const uint64_t below = (1ull << lane) - 1;
    const uint32_t m = at_more + __builtin_popcountll(b_more & below), q = at_same + __builtin_popcountll(b_same & below);
    if (more || (same && q < want)) {
      const uint32_t at = m + min(q, want);
      keep[at] = static_cast<int32_t>(i0 + lane);
      if (out != nullptr) out[at] = x;
    }
    at_more += __builtin_popcountll(b_more), at_same += __builtin_popcountll(b_same);
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

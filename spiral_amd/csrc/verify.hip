// Verification of drafted tokens by given random numbers (spiral_cache.h).
//
// Three steps, the first over all rows at once, for a walk that read row after row would
// wait for each:
//   stats_kernel   of every kChunk logits of a row: the largest, its first place, and the sum
//                  of exp((l - largest) / T);
//   walk_kernel    a workgroup (with a draft model: one for each chunk of the vocabulary) of a
//                  sequence puts its rows' sums together, looks up the probabilities
//                  of the drafted tokens and walks the tree; a token drawn from p is found
//                  by the chunks' sums, then in its chunk; of max(p - q, 0) each
//                  workgroup sums its chunk;
//   draw_kernel    draws the tokens from max(p - q, 0) by those sums.
// Exponentials and sums are in 64 bits. A token changes when its border in the running sum
// moves past the random number: with fp32 exponentials borders move by about 2^-24 of the
// sum, so that of 100000 equally likely tokens some in a thousand draws come out as
// another; here by about 2^-50. The device's fp64 rate lets it: 11 multiply-adds an
// exponential take about as long as reading an F32 logit.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

constexpr int kChunk = 4096;      // logits of a workgroup
constexpr int kMostTree = 1024;
constexpr int kStats = 256, kWalk = 1024;

struct Stat {
  double sum;  // of exp((l - top) / T)
  float top;   // NaN: the chunk holds a NaN or +infinity; -infinity: nothing
  int32_t best;
};

// What a sequence's walk leaves for draw_kernel.
struct Left {
  double scale_p, scale_q;  // 1 / sums of the rows
  float top_p, top_q;
  int32_t node;             // < 0: nothing to draw
  int32_t at;               // where the token goes, in the row of `out`
};

struct VerifyArgs {
  const uint8_t *logits, *draft;
  int64_t logits_row, draft_row;  // bytes
  uint32_t nodes, vocab, chunks;
  const int32_t *tokens, *parents, *cu;
  uint32_t seqs, max_tree;
  const float *accept, *sample, *temperature;
  int32_t *keep, *kept, *out;
  int64_t keep_stride;
  Stat* stats;     // [nodes (and nodes of the draft)][chunks]
  double* sums;    // [seqs][chunks] of max(p - q, 0)
  Left* left;      // [seqs]
};

template <int TYPE>
__device__ __forceinline__ float logit(const uint8_t* row, uint32_t i) {
  if constexpr (TYPE == SPIRAL_TYPE_F32) return reinterpret_cast<const float*>(row)[i];
  const uint32_t w = reinterpret_cast<const uint16_t*>(row)[i];
  return TYPE == SPIRAL_TYPE_BF16 ? __uint_as_float(w << 16) : fp16_ieee(w);
}

// exp(x) for x <= 0: 2^k times a polynomial for 2^f, |f| <= 1/2, fitted to 2^f at the eleven
// Chebyshev points; within 2^-50 of it.
__device__ __forceinline__ double exp_below(double x) {
  const double t = fmax(x, -800.0) * 1.4426950408889634074;
  const double k = __builtin_rint(t), f = fma(fmax(x, -800.0), 1.4426950408889634074, -k);
  double p = 7.072585949269224e-09;
  p = fma(p, f, 1.0208690299958306e-07);
  p = fma(p, f, 1.321544258792169e-06);
  p = fma(p, f, 1.5252657260200837e-05);
  p = fma(p, f, 0.0001540353044173605);
  p = fma(p, f, 0.0013333558230164974);
  p = fma(p, f, 0.009618129107606888);
  p = fma(p, f, 0.05550410866444772);
  p = fma(p, f, 0.24022650695910097);
  p = fma(p, f, 0.69314718055995);
  p = fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(k));  // 0 for x <= -800
}

// exp((l - top) / T), 0 for l = -infinity.
__device__ __forceinline__ double weight(float l, float top, double inverse) {
  return exp_below((static_cast<double>(l) - static_cast<double>(top)) * inverse);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Whether a temperature draws (0 and what is no number do not).
__device__ __forceinline__ bool draws(float t) { return t > 0.0f; }

__device__ __forceinline__ float temperature_of(const VerifyArgs& a, uint32_t s) {
  return a.temperature == nullptr ? 1.0f : a.temperature[s];
}

struct Tree {
  uint32_t first, count;
  __device__ Tree(const VerifyArgs& a, uint32_t s) {
    const int32_t n0 = min(max(a.cu[s], 0), static_cast<int32_t>(a.nodes));
    const int32_t n1 = min(max(a.cu[s + 1], n0), static_cast<int32_t>(a.nodes));
    first = n0, count = min(static_cast<uint32_t>(n1 - n0), a.max_tree);
  }
};

// One chunk of one row. Threads hold its logits in registers: VEC together, kStats apart.
template <int TYPE>
__global__ void __launch_bounds__(kStats) stats_kernel(VerifyArgs a) {
  constexpr int VEC = TYPE == SPIRAL_TYPE_F32 ? 4 : 8, N = kChunk / kStats, SIZE = TYPE == SPIRAL_TYPE_F32 ? 4 : 2;
  __shared__ float s_top[kStats / 64];
  __shared__ int32_t s_best[kStats / 64];
  __shared__ double s_sum[kStats / 64];
  const uint32_t node = blockIdx.y < a.nodes ? blockIdx.y : blockIdx.y - a.nodes;
  const uint8_t* row = blockIdx.y < a.nodes ? a.logits + node * a.logits_row : a.draft + node * a.draft_row;
  const uint32_t chunk0 = blockIdx.x * kChunk, n = min(a.vocab - chunk0, static_cast<uint32_t>(kChunk));
  float x[N];
#pragma unroll
  for (int v = 0; v < N / VEC; ++v) {
    const uint32_t at = (v * kStats + threadIdx.x) * VEC;
    const uint8_t* src = row + static_cast<int64_t>(chunk0 + at) * SIZE;
    if (at + VEC <= n) {
      uint32_t w[4];
      __builtin_memcpy(w, src, 16);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        x[v * VEC + i] = TYPE == SPIRAL_TYPE_F32    ? __uint_as_float(w[i % 4])
                         : TYPE == SPIRAL_TYPE_BF16 ? (i % 2 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]))
                                                    : fp16_ieee(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[v * VEC + i] = at + i < n ? logit<TYPE>(row, chunk0 + at + i) : -INFINITY;
    }
  }
  // The sequence, for its temperature: the last whose first node is not behind this one.
  uint32_t s = 0;
  for (uint32_t m = a.seqs; m > 1;) {
    const uint32_t half = m / 2;
    if (a.cu[s + half] <= static_cast<int32_t>(node)) s += half;
    m -= half;
  }
  const float t = temperature_of(a, s);
  float top = -INFINITY;
  int32_t best = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    bad = bad || !(x[i] < INFINITY);
    const int32_t at = (i / VEC * kStats + threadIdx.x) * VEC + i % VEC;
    if (x[i] > top) top = x[i], best = at;
  }
  auto later = [&](float o, int32_t o_best) {
    if (o > top || (o == top && o_best < best)) top = o, best = o_best;
  };
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ot = __shfl_xor(top, o, 64);
    later(ot, __shfl_xor(best, o, 64));
  }
  if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top, s_best[threadIdx.x / 64] = best;
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < kStats / 64; ++w) later(s_top[w], s_best[w]);
  double sum = 0.0;
  if (draws(t) && top > -INFINITY && !bad) {
    const double inverse = 1.0 / static_cast<double>(t);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += weight(x[i], top, inverse);
  }
  sum = wave_sum_f64(sum);
  if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kStats / 64; ++w) sum += s_sum[w];
    a.stats[static_cast<int64_t>(blockIdx.y) * a.chunks + blockIdx.x] =
        Stat{sum, bad ? NAN : top, static_cast<int32_t>(chunk0) + best};
  }
}

// A row's statistics from its chunks'.
struct Row {
  double sum;
  float top;
  int32_t best;
  __device__ __forceinline__ bool good() const { return top > -INFINITY; }  // not NaN either
};
// By a wave, a chunk a lane.
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int64_t row, double inverse) {
  const Stat* s = a.stats + row * a.chunks;
  const uint32_t lane = threadIdx.x & 63u;
  Row r{0.0, -INFINITY, 0};
  bool bad = false;
  for (uint32_t b = 0; b < a.chunks; b += 64) {
    const Stat own = b + lane < a.chunks ? s[b + lane] : Stat{0.0, -INFINITY, 0};
    bad = bad || __builtin_amdgcn_ballot_w64(own.top != own.top) != 0;
    float top = own.top;
    int32_t best = own.best;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float ot = __shfl_xor(top, o, 64);
      const int32_t ob = __shfl_xor(best, o, 64);
      if (ot > top || (ot == top && ob < best)) top = ot, best = ob;
    }
    const float now = fmaxf(r.top, top);
    if (!(now > -INFINITY)) continue;
    const double here = wave_sum_f64(own.top > -INFINITY ? own.sum * weight(own.top, now, inverse) : 0.0);
    r.sum = (r.top > -INFINITY ? r.sum * weight(r.top, now, inverse) : 0.0) + here;
    if (top > r.top) r.best = best;
    r.top = now;
  }
  if (bad) r.top = NAN;
  return r;
}

// Sums over the workgroup's threads up to and with this one, and of all; buf: a double a wave.
__device__ __forceinline__ double block_sum_upto(double v, double* buf, double& all) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, 64);
    if (lane >= static_cast<uint32_t>(o)) x += y;
  }
  __syncthreads();  // buf has been read
  if (lane == 63) buf[wave] = x;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
  for (uint32_t w = 0; w < kWalk / 64; ++w) {
    if (w < wave) before += buf[w];
    all += buf[w];
  }
  return before + x;
}

// What a token is drawn from: w(x) = exp((l - top) / T) without the tokens turned down, or
// max(p(x) - q(x), 0).
template <int TYPE>
struct Source {
  const uint8_t *p, *q;  // q: null for the former
  float top_p, top_q;
  double inverse, scale_p, scale_q;
  const int32_t* out;  // tokens turned down
  uint32_t n_out;
  __device__ __forceinline__ double operator()(uint32_t i) const {
    const double w = weight(logit<TYPE>(p, i), top_p, inverse);
    if (q == nullptr) {
      for (uint32_t j = 0; j < n_out; ++j)
        if (out[j] == static_cast<int32_t>(i)) return 0.0;
      return w;
    }
    return fmax(w * scale_p - weight(logit<TYPE>(q, i), top_q, inverse) * scale_q, 0.0);
  }
};

// The first token of chunk c whose sum, with `before` in front of it, passes `goal`; the last of
// any weight if rounding leaves none. By the workgroup; buf: a double a wave; hit: shared.
template <int TYPE>
__device__ int32_t find_in_chunk(const Source<TYPE>& w, uint32_t vocab, uint32_t c, double before, double goal,
                                 double* buf, uint32_t* hit) {
  constexpr int N = kChunk / kWalk;
  const uint32_t first = c * kChunk + threadIdx.x * N;
  double x[N], sum = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = first + i < vocab ? w(first + i) : 0.0;
    sum += x[i];
  }
  if (threadIdx.x == 0) hit[0] = ~0u, hit[1] = 0u;
  double all;
  const double upto = block_sum_upto(sum, buf, all);
  double run = before + (upto - sum);
  uint32_t found = ~0u, last = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    run += x[i];
    if (x[i] > 0.0) {
      last = first + i + 1;
      if (run > goal && found == ~0u) found = first + i;
    }
  }
  if (found != ~0u) atomicMin(&hit[0], found);
  if (last != 0u) atomicMax(&hit[1], last);
  __syncthreads();
  const uint32_t at = hit[0] != ~0u ? hit[0] : max(hit[1], 1u) - 1;
  __syncthreads();
  return static_cast<int32_t>(at);
}

// Of `chunks` sums in `part`, the chunk in which their running sum passes r times their total
// (the last of any weight if rounding leaves none), what is in front of it, and the total.
// By one wave; part in LDS or memory.
struct Found {
  uint32_t chunk;
  double before, total;
};
__device__ __forceinline__ Found find_chunk(const double* part, uint32_t chunks, double r) {
  const uint32_t lane = threadIdx.x & 63u;
  double total = 0.0;
  for (uint32_t b = 0; b < chunks; b += 64) total += wave_sum_f64(b + lane < chunks ? part[b + lane] : 0.0);
  const double goal = r * total;
  Found f{0u, 0.0, total};
  double before = 0.0;
  for (uint32_t b = 0; b < chunks; b += 64) {
    const double own = b + lane < chunks ? part[b + lane] : 0.0;
    double x = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o, 64);
      if (lane >= static_cast<uint32_t>(o)) x += y;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(own > 0.0 && before + x > goal);
    const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
    if ((past | some) != 0) {
      const int l = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      f.chunk = b + l;
      f.before = before + __shfl(x - own, l, 64);
      if (past != 0) return f;
    }
    before += __shfl(x, 63, 64);
  }
  return f;
}

// DRAFT: a workgroup a chunk, which all walk; else one a sequence.
template <int TYPE, bool DRAFT>
__global__ void __launch_bounds__(kWalk) walk_kernel(VerifyArgs a) {
  __shared__ double s_p[kMostTree], s_q[kMostTree], s_buf[kWalk / 64];
  __shared__ int32_t s_parent[kMostTree], s_token[kMostTree], s_out[kMostTree];
  __shared__ float s_u[kMostTree];
  __shared__ uint8_t s_twice[kMostTree];
  __shared__ Row s_row[DRAFT ? 2 : 1][kMostTree];
  __shared__ uint32_t s_hit[2];
  __shared__ int32_t s_walk[4];  // the last node, nodes turned down there, nodes kept, stopped
  const uint32_t s = blockIdx.y, lane = threadIdx.x & 63u;
  const Tree tree(a, s);
  const bool writes = blockIdx.x == 0;
  int32_t* keep = a.keep + s * a.keep_stride;
  int32_t* out = a.out + s * a.keep_stride;
  if (tree.count == 0) {
    if (writes) {
      for (uint32_t i = threadIdx.x; i < a.max_tree; i += kWalk) keep[i] = out[i] = -1;
      if (threadIdx.x == 0) {
        a.kept[s] = 0;
        if (DRAFT) a.left[s].node = -1;
      }
    }
    return;
  }
  const float t = temperature_of(a, s);
  const double inverse = draws(t) ? 1.0 / static_cast<double>(t) : 1.0;

  for (uint32_t i = threadIdx.x / 64; i < tree.count; i += kWalk / 64) {
    const Row r = row_of(a, tree.first + i, inverse);
    if (lane == 0) s_row[0][i] = r;
    if constexpr (DRAFT) {
      const Row d = row_of(a, static_cast<int64_t>(a.nodes) + tree.first + i, inverse);
      if (lane == 0) s_row[1][i] = d;
    }
  }
  __syncthreads();
  // Of each node: its parent, token and random number, and the probabilities of its token
  // behind the parent.
  for (uint32_t i = threadIdx.x; i < tree.count; i += kWalk) {
    const uint32_t node = tree.first + i;
    const int32_t token = a.tokens[node];
    int32_t parent = DRAFT || a.parents == nullptr ? static_cast<int32_t>(i) - 1 : a.parents[node];
    if (parent < 0 || parent >= static_cast<int32_t>(i)) parent = -1;
    s_parent[i] = parent, s_token[i] = token, s_u[i] = a.accept[node];
    double p = 0.0, q = 0.0;
    if (parent >= 0 && token >= 0 && static_cast<uint32_t>(token) < a.vocab) {
      const uint32_t from = tree.first + parent;
      const Row r = s_row[0][parent];
      if (r.good())
        p = !draws(t) ? (r.best == token ? 1.0 : 0.0)
                      : weight(logit<TYPE>(a.logits + from * a.logits_row, token), r.top, inverse) / r.sum;
      if constexpr (DRAFT) {
        const Row d = s_row[1][parent];
        q = !d.good()   ? INFINITY  // turns the token down
            : !draws(t) ? (d.best == token ? 1.0 : 0.0)
                        : weight(logit<TYPE>(a.draft + from * a.draft_row, token), d.top, inverse) / d.sum;
      }
    }
    s_p[i] = p, s_q[i] = q;
  }
  __syncthreads();
  // A node whose token an earlier child of its parent has: that one has been turned down
  // when this one is tried, and its probability with it.
  if constexpr (!DRAFT) {
    for (uint32_t i = threadIdx.x; i < tree.count; i += kWalk) {
      bool twice = false;
      for (uint32_t j = 1; j < i && !twice; ++j) twice = s_parent[j] == s_parent[i] && s_token[j] == s_token[i];
      s_twice[i] = twice;
    }
    __syncthreads();
  }
  if (threadIdx.x < 64) {
    // Children lie behind their parents: one pass over the nodes, 64 at a time.
    int32_t at = 0, kept = 1, turned = 0, stopped = 0;
    double left = 1.0;
    if (writes && lane == 0) keep[0] = 0;
    for (uint32_t b = 0; b < tree.count && !stopped; b += 64) {
      const uint32_t i = b + lane;
      const int32_t parent = i < tree.count ? s_parent[i] : -1;
      uint64_t todo = ~0ull;
      for (;;) {
        const uint64_t mine = __builtin_amdgcn_ballot_w64(parent == at && i > 0) & todo;
        if (mine == 0 || stopped) break;
        const int l = __builtin_ctzll(mine);
        const uint32_t c = b + l;
        todo = l == 63 ? 0ull : ~0ull << (l + 1);
        const double u = s_u[c];
        double chance = s_p[c];
        bool taken;
        if constexpr (DRAFT) {
          taken = u * s_q[c] < chance;
        } else {
          if (s_twice[c]) chance = 0.0;
          taken = u * left < chance;
        }
        if (taken) {
          if (writes && lane == 0) keep[kept] = static_cast<int32_t>(c), out[kept - 1] = s_token[c];
          at = static_cast<int32_t>(c), ++kept, turned = 0, left = 1.0;
        } else {
          if (lane == 0) s_out[turned] = s_token[c];
          ++turned, left -= chance;
          if (DRAFT) stopped = 1;
        }
      }
    }
    if (lane == 0) s_walk[0] = at, s_walk[1] = turned, s_walk[2] = kept, s_walk[3] = stopped;
  }
  __syncthreads();
  const uint32_t node = tree.first + s_walk[0], kept = s_walk[2];
  if (writes) {
    for (uint32_t i = kept + threadIdx.x; i < a.max_tree; i += kWalk) keep[i] = out[i] = -1;
    if (threadIdx.x == 0) a.kept[s] = static_cast<int32_t>(kept);
  }
  const Row r = s_row[0][s_walk[0]];
  Row d{0.0, -INFINITY, 0};
  if (DRAFT && s_walk[3]) d = s_row[DRAFT ? 1 : 0][s_walk[0]];
  const bool rest = DRAFT && d.good() && r.good() && draws(t);
  if (DRAFT && writes && threadIdx.x == 0)
    a.left[s] = Left{1.0 / r.sum, 1.0 / d.sum, r.top, d.top, rest ? static_cast<int32_t>(node) : -1,
                     static_cast<int32_t>(kept) - 1};
  if (!r.good() || !draws(t)) {
    if (writes && threadIdx.x == 0) out[kept - 1] = r.good() ? r.best : -1;
    return;
  }
  Source<TYPE> w{a.logits + node * a.logits_row, nullptr, r.top, 0.0f, inverse, 1.0 / r.sum, 0.0, s_out, 0u};
  if (rest) {
    w.q = a.draft + node * a.draft_row, w.top_q = d.top, w.scale_q = 1.0 / d.sum;
    constexpr int N = kChunk / kWalk;
    double sum = 0.0, all;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t at = blockIdx.x * kChunk + threadIdx.x * N + i;
      sum += at < a.vocab ? w(at) : 0.0;
    }
    block_sum_upto(sum, s_buf, all);
    if (threadIdx.x == 0) a.sums[static_cast<int64_t>(s) * a.chunks + blockIdx.x] = all;
    return;
  }
  if (!writes) return;

  // From p without what was turned down: the chunks' sums, those with such tokens anew.
  extern __shared__ __align__(16) double part[];
  const Stat* st = a.stats + static_cast<int64_t>(node) * a.chunks;
  auto fill = [&]() {
    for (uint32_t c = threadIdx.x; c < a.chunks; c += kWalk)
      part[c] = st[c].top > -INFINITY ? st[c].sum * weight(st[c].top, r.top, inverse) : 0.0;
    __syncthreads();
  };
  fill();
  if constexpr (!DRAFT) {
    w.n_out = s_walk[1];
    for (uint32_t j = 0; j < w.n_out; ++j) {
      const int32_t token = s_out[j];
      if (token < 0 || static_cast<uint32_t>(token) >= a.vocab) continue;
      const uint32_t c = static_cast<uint32_t>(token) / kChunk;
      bool done = false;  // by an earlier token
      for (uint32_t i = 0; i < j; ++i) done = done || (s_out[i] >= 0 && static_cast<uint32_t>(s_out[i]) / kChunk == c);
      if (done) continue;
      constexpr int N = kChunk / kWalk;
      double sum = 0.0, all;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t at = c * kChunk + threadIdx.x * N + i;
        sum += at < a.vocab ? w(at) : 0.0;
      }
      block_sum_upto(sum, s_buf, all);
      if (threadIdx.x == 0) part[c] = all;
    }
    __syncthreads();
  }
  const double u = a.sample[s];
  Found f = find_chunk(part, a.chunks, u);
  if (!(f.total > 0.0)) {
    __syncthreads();
    fill();
    w.n_out = 0;
    f = find_chunk(part, a.chunks, u);
  }
  const int32_t token = find_in_chunk(w, a.vocab, f.chunk, f.before, u * f.total, s_buf, s_hit);
  if (threadIdx.x == 0) out[kept - 1] = token;
}

// Tokens drawn from max(p - q, 0), or from p where that is nothing.
template <int TYPE>
__global__ void __launch_bounds__(kWalk) draw_kernel(VerifyArgs a) {
  __shared__ double s_buf[kWalk / 64];
  __shared__ uint32_t s_hit[2];
  extern __shared__ __align__(16) double part[];
  const uint32_t s = blockIdx.x;
  const Left l = a.left[s];
  if (l.node < 0) return;
  const double inverse = 1.0 / static_cast<double>(temperature_of(a, s)), u = a.sample[s];
  Source<TYPE> w{a.logits + l.node * a.logits_row, a.draft + l.node * a.draft_row, l.top_p, l.top_q, inverse, l.scale_p,
                 l.scale_q, nullptr, 0u};
  Found f = find_chunk(a.sums + static_cast<int64_t>(s) * a.chunks, a.chunks, u);
  if (!(f.total > 0.0)) {
    const Stat* st = a.stats + static_cast<int64_t>(l.node) * a.chunks;
    for (uint32_t c = threadIdx.x; c < a.chunks; c += kWalk)
      part[c] = st[c].top > -INFINITY ? st[c].sum * weight(st[c].top, l.top_p, inverse) : 0.0;
    __syncthreads();
    w.q = nullptr;
    f = find_chunk(part, a.chunks, u);
  }
  const int32_t token = find_in_chunk(w, a.vocab, f.chunk, f.before, u * f.total, s_buf, s_hit);
  if (threadIdx.x == 0) a.out[s * a.keep_stride + l.at] = token;
}

constexpr int64_t kMostVocab = int64_t(1) << 24;  // a chunk's sum each in LDS: 32 KiB

int64_t round16(int64_t n) { return ceil_div(n, 16) * 16; }

bool sizes_ok(int64_t nodes, int64_t seqs, int64_t vocab) {
  return nodes >= 0 && nodes <= 32767 && seqs >= 0 && seqs <= 65535 && vocab > 0 && vocab <= kMostVocab;
}

template <int TYPE>
int run(const VerifyArgs& a, hipStream_t s) {
  const dim3 rows(a.chunks, a.draft != nullptr ? 2 * a.nodes : a.nodes);
  const int lds = static_cast<int>(a.chunks * sizeof(double));
  if (a.nodes > 0) hipLaunchKernelGGL(stats_kernel<TYPE>, rows, dim3(kStats), 0, s, a);
  if (a.draft != nullptr) {
    int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&walk_kernel<TYPE, true>), lds);
    if (rc != SPIRAL_OK) return rc;
    hipLaunchKernelGGL((walk_kernel<TYPE, true>), dim3(a.chunks, a.seqs), dim3(kWalk), lds, s, a);
    hipLaunchKernelGGL(draw_kernel<TYPE>, dim3(a.seqs), dim3(kWalk), lds, s, a);
  } else {
    int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&walk_kernel<TYPE, false>), lds);
    if (rc != SPIRAL_OK) return rc;
    hipLaunchKernelGGL((walk_kernel<TYPE, false>), dim3(1, a.seqs), dim3(kWalk), lds, s, a);
  }
  return launch_status();
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int64_t spiral_draft_verify_workspace_bytes(int64_t nodes, int64_t seqs, int64_t vocab, int has_draft) {
  if (!sizes_ok(nodes, seqs, vocab)) return 0;
  const int64_t chunks = ceil_div(vocab, kChunk);
  return round16((has_draft ? 2 : 1) * nodes * chunks * int64_t(sizeof(Stat))) +
         (has_draft ? round16(seqs * chunks * 8) + seqs * int64_t(sizeof(Left)) : 0);
}

int spiral_draft_verify(int type, const void* logits, int64_t logits_stride, const void* draft, int64_t draft_stride,
                        int64_t nodes, int64_t vocab, const int32_t* tokens, const int32_t* parents, const int32_t* cu,
                        int64_t seqs, int64_t max_tree, const float* accept, const float* sample,
                        const float* temperature, int32_t* keep, int32_t* kept, int32_t* out, int64_t keep_stride,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (type != SPIRAL_TYPE_F32 && type != SPIRAL_TYPE_F16 && type != SPIRAL_TYPE_BF16) return SPIRAL_ERR_TYPE;
  if (!sizes_ok(nodes, seqs, vocab) || max_tree < 0 || max_tree > kMostTree || logits_stride < vocab ||
      logits_stride > (int64_t(1) << 40) || (draft != nullptr && (draft_stride < vocab || draft_stride > (int64_t(1) << 40))) ||
      keep_stride < max_tree || keep_stride > INT32_MAX || (draft != nullptr && parents != nullptr))
    return SPIRAL_ERR_SHAPE;
  if (seqs == 0 || max_tree == 0) return SPIRAL_OK;
  if (cu == nullptr || sample == nullptr || keep == nullptr || kept == nullptr || out == nullptr ||
      (nodes > 0 && (logits == nullptr || tokens == nullptr || accept == nullptr || workspace == nullptr)))
    return SPIRAL_ERR_NULL;
  const uintptr_t size = type == SPIRAL_TYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size != 0 || reinterpret_cast<uintptr_t>(draft) % size != 0 ||
      !words_aligned({tokens, parents, cu, accept, sample, temperature, keep, kept, out}) || !aligned16(workspace))
    return SPIRAL_ERR_ALIGN;
  if (workspace_bytes < spiral_draft_verify_workspace_bytes(nodes, seqs, vocab, draft != nullptr))
    return SPIRAL_ERR_CAPACITY;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  if (nodes == 0) draft = nullptr;  // empty trees only
  const int64_t chunks = ceil_div(vocab, kChunk);
  VerifyArgs a{static_cast<const uint8_t*>(logits), static_cast<const uint8_t*>(draft),
               logits_stride * static_cast<int64_t>(size), draft_stride * static_cast<int64_t>(size),
               static_cast<uint32_t>(nodes), static_cast<uint32_t>(vocab), static_cast<uint32_t>(chunks), tokens,
               parents, cu, static_cast<uint32_t>(seqs), static_cast<uint32_t>(max_tree), accept, sample, temperature,
               keep, kept, out, keep_stride, static_cast<Stat*>(workspace), nullptr, nullptr};
  if (draft != nullptr) {
    uint8_t* p = static_cast<uint8_t*>(workspace) + round16(2 * nodes * chunks * int64_t(sizeof(Stat)));
    a.sums = reinterpret_cast<double*>(p);
    a.left = reinterpret_cast<Left*>(p + round16(seqs * chunks * 8));
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return type == SPIRAL_TYPE_F32   ? run<SPIRAL_TYPE_F32>(a, s)
         : type == SPIRAL_TYPE_F16 ? run<SPIRAL_TYPE_F16>(a, s)
                                   : run<SPIRAL_TYPE_BF16>(a, s);
}

}  // extern "C"

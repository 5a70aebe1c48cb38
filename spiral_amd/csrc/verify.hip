// Verification of drafted tokens by given random numbers (spiral_cache.h).
//
// Three steps, the first over all rows at once, for a walk that read row after row would
// wait for each:
//   stats_kernel   of every kChunk logits of a row: the largest, its first place, and the sum
//                  of exp((l - largest) / T);
//   walk_kernel    a workgroup (with a draft model: one for each chunk of the vocabulary) of a
//                  sequence puts its rows' sums together, looks up the probabilities of the
//                  drafted tokens and walks the tree; a token drawn from p is found by the
//                  chunks' sums, then in its chunk; of max(p - q, 0) each workgroup sums its
//                  chunk, and the last one to have done so draws.
// Exponentials and sums are in 64 bits. A token changes when its border in the running sum
// moves past the random number: with fp32 exponentials borders move by about 2^-24 of the
// sum, so that of 100000 equally likely tokens some in a thousand draws come out as
// another; here by about 2^-50. The device's fp64 rate lets it: 11 multiply-adds an
// exponential take about as long as reading an F32 logit. 133 rows of 100003 F32 logits: 17 us in
// the first step (3.1 TB/s of the 5.1 that a copy reaches); the walk of 16 trees 10 us, a chain of
// 8 with a draft model 11: chains of dependent loads, reductions over 1024 threads and barriers.
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
  uint32_t* done;  // [seqs] workgroups that have written theirs; zeroed by stats_kernel
};

template <int TYPE>
__device__ __forceinline__ float logit(const uint8_t* row, uint32_t i) {
  if constexpr (TYPE == SPIRAL_TYPE_F32) return reinterpret_cast<const float*>(row)[i];
  const uint32_t w = reinterpret_cast<const uint16_t*>(row)[i];
  return TYPE == SPIRAL_TYPE_BF16 ? __uint_as_float(w << 16) : fp16_ieee(w);
}

// exp((l - top) / T) for l <= top, with rate = log2(e) / T: 2^k times a polynomial for 2^f, |f| <=
// 1/2, fitted to 2^f at the eleven Chebyshev points, within 2^-50 of it. 0 for l = -infinity.
__device__ __forceinline__ double weight(float l, float top, double rate) {
  const double t = fmax((static_cast<double>(l) - static_cast<double>(top)) * rate, -2000.0);
  const double k = __builtin_rint(t), f = t - k;
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
  return __builtin_amdgcn_ldexp(p, static_cast<int>(k));
}
__device__ __forceinline__ double rate_of(float temperature) { return 1.4426950408889634074 / static_cast<double>(temperature); }

// v of the lanes that DPP control CTRL names, 0 where there is none or in rows outside ROW_MASK.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROW_MASK, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROW_MASK, 0xF, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum over this lane and those below it.
__device__ __forceinline__ double sum_upto(double v) {
  v += moved<0x111, 0xF>(v);  // row_shr 1
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15: row 0 into row 1, row 2 into row 3
  v += moved<0x143, 0xC>(v);  // row_bcast 31: rows 0-1 into rows 2 and 3
  return v;
}
__device__ __forceinline__ double lane_of(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), l);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ float lane_of(float v, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
}
__device__ __forceinline__ double wave_sum_f64(double v) { return lane_of(sum_upto(v), 63); }

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
  if (blockIdx.x == 0 && blockIdx.y == 0 && a.done != nullptr)
    for (uint32_t i = threadIdx.x; i < a.seqs; i += kStats) a.done[i] = 0;
  const uint32_t node = blockIdx.y < a.nodes ? blockIdx.y : blockIdx.y - a.nodes;
  const uint8_t* row = blockIdx.y < a.nodes ? a.logits + node * a.logits_row : a.draft + node * a.draft_row;
  const uint32_t chunk0 = blockIdx.x * kChunk, n = min(a.vocab - chunk0, static_cast<uint32_t>(kChunk));
  // The sequence, for its temperature: as many as have their first node not behind this one.
  uint32_t s = 0;
  for (uint32_t b = 1; b < a.seqs; b += 64) {
    const uint32_t i = b + threadIdx.x % 64;
    s += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < a.seqs && a.cu[min(i, a.seqs)] <= static_cast<int32_t>(node)));
  }
  const float t = temperature_of(a, s);
  float x[N];
  if (n == kChunk) {  // all loads before the first is looked at
    struct __attribute__((packed, aligned(SIZE))) Words {
      u32x4_t w;
    } raw[N / VEC];
#pragma unroll
    for (int v = 0; v < N / VEC; ++v)
      raw[v] = *reinterpret_cast<const Words*>(row + static_cast<int64_t>(chunk0 + (v * kStats + threadIdx.x) * VEC) * SIZE);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t w = raw[i / VEC].w[i % VEC * SIZE / 4];
      x[i] = TYPE == SPIRAL_TYPE_F32    ? __uint_as_float(w)
             : TYPE == SPIRAL_TYPE_BF16 ? (i % 2 ? bf16_hi(w) : bf16_lo(w))
                                        : fp16_ieee(i % 2 ? w >> 16 : w & 0xffffu);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t at = (i / VEC * kStats + threadIdx.x) * VEC + i % VEC;
      x[i] = logit<TYPE>(row, chunk0 + min(at, n - 1));
      if (at >= n) x[i] = -INFINITY;
    }
  }
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
    const double rate = rate_of(t);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += weight(x[i], top, rate);
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
// By 16 lanes, a chunk a lane; the sum is the last lane's.
template <int CTRL>
__device__ __forceinline__ void better(float& top, int32_t& best) {
  const float ot = dpp_f32<CTRL, 0xF>(top);
  const int32_t ob = __builtin_amdgcn_update_dpp(0, best, CTRL, 0xF, 0xF, false);
  if (ot > top || (ot == top && ob < best)) top = ot, best = ob;
}
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int64_t row, double rate) {
  const Stat* s = a.stats + row * a.chunks;
  const uint32_t lane = threadIdx.x & 15u;
  Row r{0.0, -INFINITY, 0};
  bool bad = false;
  for (uint32_t b = 0; b < a.chunks; b += 16) {
    const Stat own = b + lane < a.chunks ? s[b + lane] : Stat{0.0, -INFINITY, 0};
    bad = bad || own.top != own.top;
    float top = own.top;
    int32_t best = own.best;
    better<0xB1>(top, best);   // quad_perm [1, 0, 3, 2]
    better<0x4E>(top, best);   // quad_perm [2, 3, 0, 1]
    better<0x124>(top, best);  // row_ror 4
    better<0x128>(top, best);  // row_ror 8
    const float now = fmaxf(r.top, top);
    if (!(now > -INFINITY)) continue;
    double here = own.top > -INFINITY ? own.sum * weight(own.top, now, rate) : 0.0;
    here += moved<0xB1, 0xF>(here);
    here += moved<0x4E, 0xF>(here);
    here += moved<0x124, 0xF>(here);
    here += moved<0x128, 0xF>(here);
    r.sum = (r.top > -INFINITY ? r.sum * weight(r.top, now, rate) : 0.0) + here;
    if (top > r.top) r.best = best;
    r.top = now;
  }
  // A NaN in any lane's chunks.
  uint32_t any = bad ? 1u : 0u;
  any |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(any), 0xB1, 0xF, 0xF, false));
  any |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(any), 0x4E, 0xF, 0xF, false));
  any |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(any), 0x124, 0xF, 0xF, false));
  any |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(any), 0x128, 0xF, 0xF, false));
  if (any) r.top = NAN;
  return r;
}

// Sums over the workgroup's threads up to and with this one, and of all; buf: a double a wave.
__device__ __forceinline__ double block_sum_upto(double v, double* buf, double& all) {
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double x = sum_upto(v);
  __syncthreads();  // buf has been read
  if (lane == 63) buf[wave] = x;
  __syncthreads();
  const double waves = sum_upto(lane < kWalk / 64 ? buf[lane] : 0.0);
  all = lane_of(waves, 63);
  return (wave > 0 ? lane_of(waves, static_cast<int>(wave - 1)) : 0.0) + x;
}

// What a token is drawn from: w(x) = exp((l - top) / T) without the tokens turned down, or
// max(p(x) - q(x), 0).
template <int TYPE>
struct Source {
  const uint8_t *p, *q;  // q: null for the former
  float top_p, top_q;
  double rate, scale_p, scale_q;
  const int32_t* out;  // tokens turned down
  uint32_t n_out;
  __device__ __forceinline__ double operator()(uint32_t i) const {
#pragma clang fp contract(off)  // equal products leave nothing, not the rounding of one of them
    const double w = weight(logit<TYPE>(p, i), top_p, rate);
    if (q == nullptr) {
      for (uint32_t j = 0; j < n_out; ++j)
        if (out[j] == static_cast<int32_t>(i)) return 0.0;
      return w;
    }
    return fmax(w * scale_p - weight(logit<TYPE>(q, i), top_q, rate) * scale_q, 0.0);
  }
};

// The first token of chunk c whose sum, with `before` in front of it, passes `goal`; the last of
// any weight if rounding leaves none. By the workgroup; buf: a double a wave; hit: two numbers a
// wave, shared (atomics on one word, from every thread behind the token, took 8 of 15 us).
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
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t past = __builtin_amdgcn_ballot_w64(found != ~0u), some = __builtin_amdgcn_ballot_w64(last != 0u);
  const uint32_t wave_found = past != 0 ? __builtin_amdgcn_readlane(found, __builtin_ctzll(past)) : ~0u;
  const uint32_t wave_last = some != 0 ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(some)) : 0u;
  if (lane == 0) hit[2 * wave] = wave_found, hit[2 * wave + 1] = wave_last;
  __syncthreads();
  uint32_t at = ~0u, end = 1u;
  for (uint32_t w = 0; w < kWalk / 64; ++w) at = min(at, hit[2 * w]), end = max(end, hit[2 * w + 1]);
  if (at == ~0u) at = end - 1;
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
    const double x = sum_upto(own);
    const uint64_t past = __builtin_amdgcn_ballot_w64(own > 0.0 && before + x > goal);
    const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
    if ((past | some) != 0) {
      const int l = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      f.chunk = b + l;
      f.before = before + lane_of(x - own, l);
      if (past != 0) return f;
    }
    before += lane_of(x, 63);
  }
  return f;
}

// DRAFT: a workgroup a chunk, which all walk; else one a sequence.
template <int TYPE, bool DRAFT>
__global__ void __launch_bounds__(kWalk) walk_kernel(VerifyArgs a) {
  __shared__ Row s_row[DRAFT ? 2 : 1][kMostTree];
  __shared__ double s_buf[kWalk / 64], s_weight[DRAFT ? 1 : kMostTree];
  __shared__ int32_t s_out[kMostTree];
  __shared__ uint32_t s_hit[2 * kWalk / 64];
  __shared__ int32_t s_walk[4];  // the last node, tokens turned down there, nodes kept, stopped
  const uint32_t s = blockIdx.y, lane = threadIdx.x & 63u;
  const Tree tree(a, s);
  const bool writes = blockIdx.x == 0;
  int32_t* keep = a.keep + s * a.keep_stride;
  int32_t* out = a.out + s * a.keep_stride;
  if (tree.count == 0) {
    if (writes) {
      for (uint32_t i = threadIdx.x; i < a.max_tree; i += kWalk) keep[i] = out[i] = -1;
      if (threadIdx.x == 0) a.kept[s] = 0;
    }
    return;
  }
  const float t = temperature_of(a, s);
  const double rate = draws(t) ? rate_of(t) : 1.0;

  // A node a lane: its token, parent and random number, and its token's logits behind the parent.
  // The first 64 are asked for ahead of the rows' sums.
  struct Node {
    int32_t token, parent;
    float u, p, q;
    bool known;
  };
  auto load_node = [&](uint32_t b) {
    const uint32_t i = b + lane, node = tree.first + min(i, tree.count - 1);
    Node x;
    x.token = a.tokens[node], x.u = a.accept[node];
    x.parent = DRAFT || a.parents == nullptr ? static_cast<int32_t>(i) - 1 : a.parents[node];
    if (x.parent < 0 || x.parent >= static_cast<int32_t>(i) || i >= tree.count) x.parent = -1;
    x.known = x.token >= 0 && static_cast<uint32_t>(x.token) < a.vocab;
    const uint32_t from = tree.first + max(x.parent, 0), at = x.known ? x.token : 0;
    x.p = logit<TYPE>(a.logits + from * a.logits_row, at);
    x.q = DRAFT ? logit<TYPE>(a.draft + from * a.draft_row, at) : 0.0f;
    return x;
  };
  Node first{};
  if (threadIdx.x < 64) first = load_node(0);
  for (uint32_t i = threadIdx.x / 16; i < (DRAFT ? 2 : 1) * tree.count; i += kWalk / 16) {
    const bool of_draft = DRAFT && i >= tree.count;
    const uint32_t at = of_draft ? i - tree.count : i;
    const Row r = row_of(a, (of_draft ? static_cast<int64_t>(a.nodes) : 0) + tree.first + at, rate);
    if (threadIdx.x % 16 == 15) s_row[DRAFT && of_draft ? 1 : 0][at] = r;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    // Children lie behind their parents: one pass over the nodes, 64 at a time.
    int32_t at = 0, kept = 1, turned = 0, stopped = 0;
    double left = 1.0;
    if (writes && lane == 0) keep[0] = 0;
    for (uint32_t b = 0; b < tree.count && !stopped; b += 64) {
      const Node x = b == 0 ? first : load_node(b);
      double p = 0.0, q = 0.0;
      if (x.parent >= 0 && x.known) {
        const Row r = s_row[0][x.parent];
        if (r.good()) p = !draws(t) ? (r.best == x.token ? 1.0 : 0.0) : weight(x.p, r.top, rate) / r.sum;
        if constexpr (DRAFT) {
          const Row d = s_row[1][x.parent];
          q = !d.good()   ? INFINITY  // turns the token down
              : !draws(t) ? (d.best == x.token ? 1.0 : 0.0)
                          : weight(x.q, d.top, rate) / d.sum;
        }
      }
      uint64_t todo = ~0ull;
      for (;;) {
        const uint64_t mine = __builtin_amdgcn_ballot_w64(x.parent == at) & todo;
        if (mine == 0 || stopped) break;
        const int l = __builtin_ctzll(mine);
        todo = l == 63 ? 0ull : ~0ull << (l + 1);
        const int32_t token = __builtin_amdgcn_readlane(x.token, l);
        double chance = lane_of(p, l);
        const double number = lane_of(x.u, l);
        bool twice = false;  // among those turned down
        if constexpr (!DRAFT) {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          for (int32_t j = 0; j < turned; j += 64)
            twice = twice || __builtin_amdgcn_ballot_w64(j + static_cast<int32_t>(lane) < turned && s_out[j + lane] == token) != 0;
          if (twice) chance = 0.0;
        }
        if (DRAFT ? number * lane_of(q, l) < chance : number * left < chance) {
          const int32_t c = static_cast<int32_t>(b) + l;
          if (writes && lane == 0) keep[kept] = c, out[kept - 1] = token;
          at = c, ++kept, turned = 0, left = 1.0;
        } else {
          left -= chance;
          if (DRAFT) stopped = 1;
          if (!twice && __builtin_amdgcn_readlane(x.known ? 1 : 0, l)) {
            if (lane == 0) s_out[turned] = token;
            ++turned;
          }
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
  if (!r.good() || !draws(t)) {
    if (writes && threadIdx.x == 0) out[kept - 1] = r.good() ? r.best : -1;
    return;
  }
  extern __shared__ __align__(16) double part[];
  const double u = a.sample[s];
  Source<TYPE> w{a.logits + node * a.logits_row, nullptr, r.top, 0.0f, rate, 1.0 / r.sum, 0.0, s_out, 0u};
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
    // The last workgroup of the sequence to get here has all sums, and draws.
    double* sums = a.sums + static_cast<int64_t>(s) * a.chunks;
    if (threadIdx.x == 0) {
      __hip_atomic_store(sums + blockIdx.x, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_hit[0] = __hip_atomic_fetch_add(a.done + s, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_hit[0] != a.chunks - 1) return;
    for (uint32_t c = threadIdx.x; c < a.chunks; c += kWalk)
      part[c] = __hip_atomic_load(sums + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const Found f = find_chunk(part, a.chunks, u);
    if (f.total > 0.0) {
      const int32_t token = find_in_chunk(w, a.vocab, f.chunk, f.before, u * f.total, s_buf, s_hit);
      if (threadIdx.x == 0) out[kept - 1] = token;
      return;
    }
    w.q = nullptr;    // nothing is left: from p
    __syncthreads();  // every wave has found that so
  } else if (!writes) {
    return;
  }

  // From p without what was turned down: the chunks' sums less its weights. A sum of which less
  // than 2^-10 is left is taken anew, without the difference's rounding.
  const Stat* st = a.stats + static_cast<int64_t>(node) * a.chunks;
  auto fill = [&]() {
    bool anew = false;
    for (uint32_t c = threadIdx.x; c < a.chunks; c += kWalk) {
      const double whole = st[c].top > -INFINITY ? st[c].sum * weight(st[c].top, r.top, rate) : 0.0;
      double x = whole;
      if constexpr (!DRAFT)
        for (uint32_t j = 0; j < w.n_out; ++j)
          if (static_cast<uint32_t>(s_out[j]) / kChunk == c) x -= s_weight[j];
      const bool little = x < whole * 0x1p-10;
      anew = anew || little;
      part[c] = little ? -1.0 : x;
    }
    return __syncthreads_or(anew);
  };
  if constexpr (!DRAFT) {
    w.n_out = s_walk[1];
    for (uint32_t j = threadIdx.x; j < w.n_out; j += kWalk)
      s_weight[j] = weight(logit<TYPE>(w.p, static_cast<uint32_t>(s_out[j])), r.top, rate);
    __syncthreads();
  }
  if (fill()) {
    for (uint32_t c = 0; c < a.chunks; ++c) {
      if (part[c] >= 0.0) continue;
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
  Found f = find_chunk(part, a.chunks, u);
  if (!(f.total > 0.0)) {
    __syncthreads();
    w.n_out = 0;
    fill();
    f = find_chunk(part, a.chunks, u);
  }
  const int32_t token = find_in_chunk(w, a.vocab, f.chunk, f.before, u * f.total, s_buf, s_hit);
  if (threadIdx.x == 0) out[kept - 1] = token;
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
         (has_draft ? round16(seqs * chunks * 8) + seqs * 4 : 0);
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
    a.done = reinterpret_cast<uint32_t*>(p + round16(seqs * chunks * 8));
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return type == SPIRAL_TYPE_F32   ? run<SPIRAL_TYPE_F32>(a, s)
         : type == SPIRAL_TYPE_F16 ? run<SPIRAL_TYPE_F16>(a, s)
                                   : run<SPIRAL_TYPE_BF16>(a, s);
}

}  // extern "C"

// What the forms of attention over a paged cache share (tree.hip, tree4.hip): sizes of
// trees, how rows are dealt to workgroups, the running softmax of a wave, the join of
// divided rows, and the limits of a call.
#pragma once

#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

constexpr int kChunk = 32;  // rows a wave takes at a time
constexpr float kSlack = 8.0f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// kLift: p is held as 2^kLift times its value. F16 ends at 2^-24, so that a weight below 2^-14
// of the maximum loses bits and one below 2^-25 is lost, while the sum counts it: 65536 of
// them are four half steps of the result. Lifted by 2^7 they reach 2^-32, and p, below
// 2^kSlack of the maximum, 2^15.
struct Bf16 {
  static constexpr bool kF16 = false;
  static constexpr float kLift = 0.0f;
  static constexpr uint32_t kExp = 0x7F80u;  // exponent bits, all set in infinities and NaN
  static __device__ __forceinline__ float value(uint32_t x) { return __uint_as_float(x << 16); }
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
struct F16 {
  static constexpr bool kF16 = true;
  static constexpr float kLift = 7.0f;
  static constexpr uint32_t kExp = 0x7C00u;
  static __device__ __forceinline__ float value(uint32_t x) { return fp16_ieee(x); }
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
  }
};

struct TreeArgs {
  const uint8_t* q;
  int64_t q_node, q_head;  // bytes
  uint32_t nodes, heads, group;
  const uint8_t *k, *v;
  uint32_t pages, kv_heads, dim;
  uint32_t page_step, row_step;  // in units of 16 bytes
  int64_t head_bytes;
  Divisor page;
  const int32_t* table;
  int64_t table_stride;
  uint32_t table_cols;
  const int32_t *lens, *cu;
  uint32_t seqs;
  const uint64_t* mask;
  uint32_t mask_words;
  float scale;  // of log2 scores
  uint8_t* out;
  float* lse;
  float* part;      // [lines][heads][dim], a line for each node of each part
  float2* part_ml;  // [lines][heads]: maximum (log2), sum
  uint32_t lines;
  uint32_t max_tree, query_groups;
  uint32_t shares;       // workgroups per cached head and query group
  uint32_t want;         // shares to deal (0: every sequence is one),
  uint32_t step, least;  // of whole steps, `least` at least
  uint32_t by_work;      // as long as a place's part of all work, not of all rows
  Divisor block;         // queries of a workgroup
  // Queries of a wave where a tree's say how the waves of its workgroups divide (else 0), and
  // the most of these that have queries of their own.
  uint32_t wave_queries = 0, most_log_waves = 0;
};

struct Tree {
  uint32_t first, count, cached, rows;  // nodes first .. + count - 1; cached rows, all rows
  __device__ Tree(const TreeArgs& a, uint32_t s) {
    const int32_t n0 = min(max(a.cu[s], 0), static_cast<int32_t>(a.nodes));
    const int32_t n1 = min(max(a.cu[s + 1], n0), static_cast<int32_t>(a.nodes));
    first = n0, count = min(static_cast<uint32_t>(n1 - n0), a.max_tree);
    cached = min(max(a.lens[s], 0), 0x3fffffff);
    const uint64_t room = static_cast<uint64_t>(a.table_cols) * a.page.d;  // rows past the table are not there
    rows = min(cached + count, static_cast<uint32_t>(min(room, static_cast<uint64_t>(0x3fffffff))));
  }
};

// How many of a workgroup's waves have queries of their own (the others divide rows): 2 to this.
__device__ __forceinline__ uint32_t log_query_waves(const TreeArgs& a, uint32_t queries) {
  return min(queries > 2 * a.wave_queries ? 2u : queries > a.wave_queries ? 1u : 0u, a.most_log_waves);
}

// The rows of all sequences in shares of `span` rows, a whole number of steps: sequence
// s has ceil(rows / span) and at least one. The span is looked for at which there are
// no more than `want` shares, one for every place on the GPU (576 shares on 512 places
// take two rounds); if a few tries do not find it there are want + seqs at most.
// Where whole sequences are some rounds of workgroups already (by_work) the span is a
// place's part of all work, rows times workgroups of queries: only a sequence that would
// run longer than all the others together is divided, in no more than 2 `want` parts.
// A part has a line of the workspace for each of its sequence's nodes; in order of the
// sequences, those for which there are none left stay whole.
// Every wave works this out for itself, a sequence a lane.
struct Share {
  uint32_t seq, split, parts;  // part `split` of the sequence's `parts`
  uint32_t line;               // their first line
  uint32_t span;
  uint2 mine;  // rows and nodes of sequence `lane`

  __device__ Share(const TreeArgs& a, uint32_t lane) : mine(sizes(a, lane)) {}

  // Where the waves of a workgroup divide rows unless the tree has queries for all of them,
  // rows count as often as they take the workgroup's time.
  static __device__ __forceinline__ uint32_t log_weight(const TreeArgs& a, uint32_t nodes) {
    return a.wave_queries == 0 ? 0u : log_query_waves(a, nodes * a.group);
  }
  static __device__ __forceinline__ uint2 sizes(const TreeArgs& a, uint32_t s) {
    if (s >= a.seqs) return make_uint2(0u, 0u);
    const Tree t(a, s);
    return make_uint2(t.rows << log_weight(a, t.count), t.count);
  }
  __device__ __forceinline__ uint2 sizes_of(const TreeArgs& a, uint32_t b, uint32_t lane) const {
    return b == 0 ? mine : sizes(a, b + lane);
  }
  __device__ __forceinline__ uint32_t parts_of(const TreeArgs& a, uint32_t b, uint32_t lane, uint32_t rows) const {
    return b + lane < a.seqs ? max(1u, (rows + span - 1) / span) : 0u;
  }
  // Parts n of sequence b + lane, the lines they need, and the sums of both up to it;
  // `lines` are taken by the sequences in front of b.
  struct Dealt {
    uint32_t n, upto, need, lines_upto, nodes;
  };
  __device__ __forceinline__ Dealt deal(const TreeArgs& a, uint32_t b, uint32_t lane, uint32_t lines) const {
    const uint2 m = sizes_of(a, b, lane);
    Dealt d{parts_of(a, b, lane, m.x), 0u, 0u, 0u, m.y};
    const uint64_t need = static_cast<uint64_t>(d.n) * m.y;
    const bool fits = need <= a.lines;
    if (d.n > 1 && fits) d.need = static_cast<uint32_t>(need);
    d.lines_upto = lines + sum_upto(d.need);
    if (!fits || d.lines_upto > a.lines) d.n = min(d.n, 1u);
    d.upto = sum_upto(d.n);
    return d;
  }
  static __device__ __forceinline__ uint32_t last(uint32_t v) { return __builtin_amdgcn_readlane(v, 63); }
  static __device__ __forceinline__ float sum(float v) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_sum_last(v)), 63));
  }
  template <int CTRL, int ROW_MASK>
  static __device__ __forceinline__ uint32_t moved(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROW_MASK, 0xF, false));
  }
  // Sum over this lane and those below it.
  static __device__ __forceinline__ uint32_t sum_upto(uint32_t v) {
    v += moved<0x111, 0xF>(v);  // row_shr 1
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);  // row_bcast 15: row 0 into row 1, row 2 into row 3
    v += moved<0x143, 0xC>(v);  // row_bcast 31: rows 0-1 into rows 2 and 3
    return v;
  }
  __device__ __forceinline__ void set_span(const TreeArgs& a, uint32_t lane) {
    // In floats, which hold these counts well enough: the sum is within 2^-17 of the
    // rows', and a little more than each share's part of it is taken.
    float all = 0.0f;
    for (uint32_t b = 0; b < a.seqs; b += 64) {
      const uint2 m = sizes_of(a, b, lane);
      if (a.by_work) {
        // A product of whole numbers: a fused multiply and add here and not there would
        // give two kernels two spans.
        const uint32_t blocks = max(1u, a.block.quotient(m.y * a.group + a.block.d - 1));
        all += static_cast<float>(static_cast<uint64_t>(m.x) * blocks);
      } else {
        all += static_cast<float>(m.x);
      }
    }
    const float each = sum(all) / static_cast<float>(a.want) * 1.0001f / static_cast<float>(a.step);
    const uint32_t most = 0x7fffffffu / a.step;
    uint32_t steps = min(max(static_cast<uint32_t>(fminf(each, 6e7f)) + 1u, a.least), most);
    for (int i = 0; i < 4; ++i) {
      span = __builtin_amdgcn_readfirstlane(steps * a.step);
      if (a.by_work) break;
      float n = 0.0f;
      for (uint32_t b = 0; b < a.seqs; b += 64) n += static_cast<float>(parts_of(a, b, lane, sizes_of(a, b, lane).x));
      const float over = sum(n) - static_cast<float>(a.want);
      if (over <= 0.0f || i == 3) break;
      steps = min(steps + max(1u, static_cast<uint32_t>(static_cast<float>(steps) * over / static_cast<float>(a.want))),
                  most);
    }
  }
  // Share `i`; false where there are fewer.
  __device__ __forceinline__ bool find(const TreeArgs& a, uint32_t i, uint32_t lane) {
    if (a.want == 0) {
      seq = i, split = 0, parts = 1, line = 0, span = 0x7fffffffu;
      return seq < a.seqs;
    }
    set_span(a, lane);
    uint32_t base = 0, lines = 0;
    for (uint32_t b = 0; b < a.seqs; b += 64) {
      const Dealt d = deal(a, b, lane, lines);
      const uint64_t past = __builtin_amdgcn_ballot_w64(base + d.upto > i);
      if (past != 0) {
        const int l = __builtin_ctzll(past);
        take(d, l);
        seq = b + l, split = i - (base + __builtin_amdgcn_readlane(d.upto, l) - parts);
        if (parts > 1) span >>= log_weight(a, __builtin_amdgcn_readlane(d.nodes, l));
        return true;
      }
      base += last(d.upto);
      lines = min(last(d.lines_upto), a.lines + 1);  // as good as any more
    }
    return false;
  }
  // The parts of sequence s.
  __device__ __forceinline__ void of(const TreeArgs& a, uint32_t s, uint32_t lane) {
    set_span(a, lane);
    uint32_t lines = 0;
    for (uint32_t b = 0;; b += 64) {
      const Dealt d = deal(a, b, lane, lines);
      if (s < b + 64) return take(d, s - b);
      lines = min(last(d.lines_upto), a.lines + 1);
    }
  }
  __device__ __forceinline__ void take(const Dealt& d, int l) {
    parts = __builtin_amdgcn_readlane(d.n, l);
    line = __builtin_amdgcn_readlane(d.lines_upto - d.need, l);
    if (parts == 1) span = 0x7fffffffu;  // all rows, also where they were to be divided
  }
};

// Bits of the 32 positions from `pos` on that a node sees, of its mask's words.
__device__ __forceinline__ uint32_t seen_bits(const uint64_t* words, uint32_t n_words, uint32_t cached, uint32_t pos) {
  const int32_t j = static_cast<int32_t>(pos - cached);  // the first position's drafted row
  if (j <= -32) return ~0u;
  if (j < 0) {
    const uint64_t w = n_words > 0 ? words[0] : 0;
    return static_cast<uint32_t>(w << -j) | ((1u << -j) - 1u);
  }
  const uint32_t i = static_cast<uint32_t>(j) >> 6, sh = j & 63;
  uint32_t r = i < n_words ? static_cast<uint32_t>(words[i] >> sh) : 0u;
  if (sh > 32 && i + 1 < n_words) r |= static_cast<uint32_t>(words[i + 1] << (64 - sh));
  return r;
}

__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Row of element e of a lane's second operand of O^T, in its chunk.
__device__ __forceinline__ constexpr uint32_t row_of(uint32_t g, uint32_t e) { return 16 * (e / 4) + 4 * g + e % 4; }

// Sums of QT tiles of queries over the rows taken so far: lane (r, g) has query r's.
template <typename E, int DV, int QT>
struct Sums {
  f32x4_t o[QT][DV];  // four dims of product d
  float top[QT], sum[QT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = -INFINITY, sum[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DV; ++d) o[t][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // Scores of a chunk to P^T, the sums brought to the new maximum.
  __device__ __forceinline__ void soften(const f32x4_t (&sc)[QT][2], float scale, u32x4_t (&pf)[QT]) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float most = fmaxf(fmaxf(fmaxf(sc[t][0][0], sc[t][0][1]), fmaxf(sc[t][0][2], sc[t][0][3])),
                         fmaxf(fmaxf(sc[t][1][0], sc[t][1][1]), fmaxf(sc[t][1][2], sc[t][1][3])));
      most *= scale;
      if (__builtin_amdgcn_ballot_w64(most > top[t] + kSlack) != 0) {
        const float now = fmaxf(top[t], across_groups_max(most));
        float shrink = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[t] - now);
        asm volatile("" : "+v"(shrink));  // in this branch, not computed ahead of it for every chunk
        top[t] = now;
        sum[t] *= shrink;
#pragma unroll
        for (int d = 0; d < DV; ++d) o[t][d] *= shrink;
      }
      const float base = top[t] == -INFINITY ? 0.0f : top[t] - E::kLift;
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(sc[t][e / 4][e % 4], scale, -base));
        sum[t] += p[e];
      }
      pf[t] = u32x4_t{E::pack(p[0], p[1]), E::pack(p[2], p[3]), E::pack(p[4], p[5]), E::pack(p[6], p[7])};
    }
  }

  // O^T += V^T P^T, product d.
  __device__ __forceinline__ void add(u32x4_t v, const u32x4_t (&pf)[QT], int d) {
#pragma unroll
    for (int t = 0; t < QT; ++t) o[t][d] = E::mfma(v, pf[t], o[t][d]);
  }
};

// Dims d .. + 3 of a query row from its sums, and with the first of them its lse. Without a
// row that it sees the sum is zero, and only then: scores that are all NaN leave the maximum
// at -infinity too, and their sum is NaN, as the result is to be.
template <typename E>
__device__ __forceinline__ void write(const TreeArgs& a, int64_t row, uint32_t d, f32x4_t v, float m, float total) {
  const bool none = total == 0.0f;
  const float f = 1.0f / total;
  *reinterpret_cast<uint2*>(a.out + (row * a.dim + d) * 2) =
      none ? make_uint2(0u, 0u) : make_uint2(E::pack(v[0] * f, v[1] * f), E::pack(v[2] * f, v[3] * f));
  if (d == 0 && a.lse != nullptr) a.lse[row] = none ? -INFINITY : kLn2 * (m - E::kLift + __builtin_amdgcn_logf(total));
}

// Joins the splits of a sequence's rows. A team of T threads takes a query row:
// dim / 4 of them have four dims each of every `groups`-th part, four parts in flight a
// thread, for the parts are other XCDs' work and come from memory. Many parts want
// the workgroup for a team (one row of 32 parts: 4.5 us, a wave 7.5), few a wave (6400
// rows of 4 parts: 8 us against 20).
template <typename E, int T>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a) {
  __shared__ f32x4_t s_v[256];
  __shared__ float s_f[256];
  __shared__ float s_w[8];
  constexpr uint32_t kTeams = 256 / T;
  const uint32_t s = blockIdx.y, team = threadIdx.x / T, tid = threadIdx.x % T, lane = tid & 63u;
  f32x4_t* tv = s_v + team * T;
  float* tf = s_f + team * T;
  auto meet = []() {
    if constexpr (T == 64)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else
      __syncthreads();
  };
  const Tree tree(a, s);
  Share share(a, lane);
  share.of(a, s, lane);
  const uint32_t n = share.parts;
  if (n == 1) return;  // written already
  const uint32_t lines = tree.count * a.heads, per = a.dim / 4, groups = T / per;
  const uint32_t group = tid / per, d = group < groups ? (tid - group * per) * 4 : 0;
  const int64_t step = static_cast<int64_t>(tree.count) * a.heads, part0 = static_cast<int64_t>(share.line) * a.heads;
  for (uint32_t i = blockIdx.x * kTeams + team; i < lines; i += gridDim.x * kTeams) {
    const int64_t row = static_cast<int64_t>(tree.first) * a.heads + i;
    f32x4_t v{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, total = 0.0f;
    for (uint32_t p0 = 0; p0 < n; p0 += T) {  // T parts at a time, joined as they come
      const uint32_t here = min(static_cast<uint32_t>(T), n - p0);
      f32x4_t x[4];  // the first parts are asked for in front of the maxima
      auto load = [&](uint32_t q) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          x[e] = *reinterpret_cast<const f32x4_t*>(a.part + ((p0 + min(q + e * groups, here - 1)) * step + part0 + i) * a.dim + d);
      };
      load(group);
      const float2 ml = tid < here ? a.part_ml[(p0 + tid) * step + part0 + i] : make_float2(-INFINITY, 0.0f);
      float now = ml.x;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor(now, o, 64));
      meet();  // what was shared before has been read
      if constexpr (T == 256) {
        if (lane == 0) s_w[tid / 64] = now;
        meet();
        now = fmaxf(fmaxf(s_w[0], s_w[1]), fmaxf(s_w[2], s_w[3]));
      }
      now = fmaxf(now, m);
      const float shrink = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      const float f = now == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
      float part = ml.y * f;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) part += __shfl_xor(part, o, 64);
      tf[tid] = f;
      if constexpr (T == 256) {
        if (lane == 0) s_w[4 + tid / 64] = part;
        meet();
        part = s_w[4] + s_w[5] + s_w[6] + s_w[7];
      } else {
        meet();
      }
      total = total * shrink + part;
      v *= shrink, m = now;
      for (uint32_t q = group; q < here && group < groups; q += 4 * groups) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (q + e * groups < here) v += tf[q + e * groups] * x[e];
        if (q + 4 * groups < here) load(q + 4 * groups);
      }
    }
    meet();
    tv[tid] = v;
    meet();
    if (group == 0) {
      for (uint32_t e = 1; e < groups; ++e) v += tv[e * per + tid];
      write<E>(a, row, d, v, m, total);
    }
  }
}

// ---- host ---------------------------------------------------------------------------

constexpr int64_t kMostDealt = 512;  // sequences that every wave looks through

// Bytes of a line of the workspace, a node's row of one part, and of all lines at most. A
// place for the largest tree in every share would be 21.8 GB for 256 sequences beside a
// prompt chunk of 2048 nodes, 32 heads of dim 128.
inline int64_t line_bytes(int64_t heads, int64_t dim) { return heads * (dim * 4 + 8); }
constexpr int64_t kMostBytes = int64_t(256) << 20;

// The join behind a kernel that dealt `want` shares.
template <typename E>
int launch_join(const TreeArgs& a, uint32_t want, int64_t max_tree, hipStream_t s) {
  // Two thousand workgroups at most: each works the shares out before its first row (6400 rows of 4
  // parts, 32 heads: 11.8 us with four times as many, 9.6; the whole call over 16 bits, 8 sequences
  // of up to 60 nodes, 80.3 and 78.4, 16 of 25 96.9 and 96.3; long single rows the same with both).
  const int64_t lines = std::max<int64_t>(max_tree, 1) * a.heads;
  const bool many = want > 8 * a.seqs;  // parts a sequence
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(many ? lines : ceil_div(lines, 4), std::max(1u, 2048 / a.seqs))),
                  a.seqs);
  if (many)
    hipLaunchKernelGGL((tree_join_kernel<E, 256>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((tree_join_kernel<E, 64>), grid, dim3(256), 0, s, a);
  return launch_status();
}

inline bool sizes_ok(int64_t nodes, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, int64_t max_len,
              int64_t max_tree) {
  return nodes >= 0 && nodes <= (1 << 24) && heads > 0 && heads <= 65536 && kv_heads > 0 && heads % kv_heads == 0 &&
         dim > 0 && dim <= 256 && dim % 8 == 0 && seqs >= 0 && seqs <= 65535 && max_len >= 0 &&
         max_len <= 0x3fffffff && max_tree >= 0 && max_tree <= (1 << 24) && max_tree * (heads / kv_heads) <= INT32_MAX;
}

}  // namespace
}  // namespace spiral

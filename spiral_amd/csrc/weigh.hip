// The attention weight that cached rows get (spiral_cache.h): mass[r] += sum over a
// sequence's queries of exp(scale q . K_r - lse).
//
// The products of tree attention's first half, S^T = K Q^T in 16 x 16 x 32 tiles, and no
// softmax to run: lse is known. A lane's results are four rows of one query, so a row's sum
// over queries is kept in the lane, over all tiles of queries and all heads, and over
// lanes at the end. Workgroups own rows: nothing is added by two of them, and the order of a sum
// does not depend on them. Of a workgroup's four waves HW take the cached heads in turn and 4 / HW other
// rows; the heads' sums meet in LDS.
// A wave holds RT tiles of 16 rows of K and passes the queries by: two tiles where queries are few,
// for more workgroups (one sequence of 4096 rows, a token: 6.2 us; its bytes are 1.7); else
// five, because every tile of queries is then loaded for more rows. 16 sequences of up to 8192
// rows, 32 nodes x 4 heads, in 4 bits: 91 us with two tiles, 57 with four, 53 with five (51 now), 85
// with eight (registers spill). Past dim 192 registers hold three (8 cached heads of dim 256: 92 us, 93
// with four, 125 with two; 90 now), past 128 four (23 x 30000 rows, 50 nodes x 3 heads of dim 192: 87 us,
// 100 with three, in the form of 256 118; 81 now). There latencies bound it, with two waves a SIMD to hide them: VALU is
// busy a third of the time, 150 instructions for four tiles and 16 queries. Workgroups are rows and
// sequences alone: many queries over few rows fill part of the GPU, a tile of queries after the other
// (a chunk of 2048 nodes over 4096 rows of one sequence, 32 heads: 1.1 ms).
#include "cache4.h"
#include "tree.h"

namespace spiral {
namespace {

constexpr int kWaves = 4;

struct WeighArgs {
  TreeArgs t;  // out, lse, parts and shares unused
  const float *lse, *counted;
  float* mass;
  int64_t mass_stride;
  uint32_t mass_cols, head_waves;
  uint32_t step_node, step_head;  // 16 queries on: so many nodes, and heads of the group
};

// Lanes 16 .. 31 and 48 .. 63 of a for lanes 0 .. 15 and 32 .. 47 of b (ROWS), lanes 32 .. 63 of a
// for 0 .. 31 of b (else).
template <bool ROWS>
__device__ __forceinline__ void swap_lanes(uint32_t& a, uint32_t& b) {
  const auto r = ROWS ? __builtin_amdgcn_permlane16_swap(a, b, false, false)
                      : __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// A tile of 16 rows of K as operands in 16 bits: lane (r, g) has dims 32 j + 8 g .. + 7 of row r
// in step j, zeros past dim; Q is loaded in the same order, 64 bytes of a row a step.
// Codes are loaded 16 bytes a lane, block g of row r, and turned: a lane's word s of block g
// goes to lane group s in step g.
template <typename E, int KS, bool FOUR>
__device__ __forceinline__ void load_tile(const uint8_t* row, uint32_t page, uint32_t in_page, uint32_t g, uint32_t dim,
                                          u32x4_t (&k)[KS]) {
  if constexpr (!FOUR) {
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const bool on = 32 * j + 8 * g < dim;
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + (on ? 2 * (32 * j + 8 * g) : 0u));
      k[j] = on ? w : u32x4_t{0, 0, 0, 0};
    }
  } else {
    constexpr int kBlocks = KS < 4 ? KS : 4;  // of a row at a time
    const uint8_t* codes = row + in_page * (dim / 2);
    const uint8_t* scales = row + page * (dim / 2) + in_page;
#pragma unroll
    for (int j0 = 0; j0 < KS; j0 += kBlocks) {
      uint32_t w[kBlocks], s;
      if constexpr (kBlocks == 4) {
        const bool on = 32 * (j0 + g) < dim;
        const u32x4_t c = *reinterpret_cast<const u32x4_t*>(codes + (on ? 16 * (j0 + g) : 0u));
        uint32_t mine = scales[on ? page * (j0 + g) : 0u];
        w[0] = c.x, w[1] = c.y, w[2] = c.z, w[3] = c.w;
        swap_lanes<false>(w[0], w[2]);
        swap_lanes<false>(w[1], w[3]);
        swap_lanes<true>(w[0], w[1]);
        swap_lanes<true>(w[2], w[3]);
        uint32_t other = mine;
        swap_lanes<false>(mine, other);  // groups 0 and 1, groups 2 and 3, in both halves
        mine |= other << 16;
        other = mine;
        swap_lanes<true>(mine, other);  // groups 0 and 2, groups 1 and 3
        s = mine | other << 8;
      } else {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
          w[j] = *reinterpret_cast<const uint32_t*>(codes + (32u * j < dim ? 16 * j : 0u) + 4 * g);
        s = scales[0] | static_cast<uint32_t>(scales[32 < dim ? page : 0u]) << 8;
      }
      auto decode = [&](auto block) {
        constexpr int B = decltype(block)::value;
        if constexpr (B < kBlocks) {
          if (j0 + B >= KS) return;
          const float f = scale_byte<B>(s);
          u32x4_t& x = k[j0 + B < KS ? j0 + B : 0];
          x = u32x4_t{fp4_pair<E, 0>(w[B], f), fp4_pair<E, 1>(w[B], f), fp4_pair<E, 2>(w[B], f), fp4_pair<E, 3>(w[B], f)};
          if (32u * (j0 + B) >= dim) x = u32x4_t{0, 0, 0, 0};
        }
      };
      decode(std::integral_constant<int, 0>{});
      decode(std::integral_constant<int, 1>{});
      decode(std::integral_constant<int, 2>{});
      decode(std::integral_constant<int, 3>{});
    }
  }
}

template <typename E, int DV, bool FOUR, int RT>
__global__ void __launch_bounds__(64 * kWaves, 2) weigh_kernel(WeighArgs w) {
  constexpr int KS = DV / 2, kRows = 16 * RT;
  __shared__ __align__(16) float s_sum[kWaves][kRows];
  const TreeArgs& a = w.t;
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t hw = wave % w.head_waves, rw = wave / w.head_waves, row_waves = kWaves / w.head_waves;
  const uint32_t s = blockIdx.y;
  const Tree tree(a, s);
  const uint32_t end = min(tree.rows, w.mass_cols), queries = tree.count * a.group;
  const PagedRows place{a.table + s * a.table_stride, a.table_cols, a.pages, a.page};
  if (queries == 0) return;

  for (uint32_t base = blockIdx.x * row_waves * kRows; base < end; base += gridDim.x * row_waves * kRows) {
    const uint32_t pos = base + rw * kRows;
    // Row r of each tile: where it lies, and a bit for each of the 16 rows that there is.
    int64_t at[RT];
    uint32_t in_page[RT], there[RT];
    bool any = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const uint32_t p = min(pos + 16 * t + r, end - 1), entry = place.page.quotient(p);
      const uint32_t id = static_cast<uint32_t>(place.table[entry]);
      const bool ok = pos + 16 * t + r < end && id < a.pages;  // a negative id is past every page
      in_page[t] = p - entry * place.page.d;
      at[t] = static_cast<int64_t>(ok ? id : 0u) * a.page_step * 16 + (FOUR ? 0 : in_page[t] * static_cast<int64_t>(a.row_step) * 16);
      there[t] = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok)) & 0xffffu;
      any = any || there[t] != 0;
    }
    f32x4_t sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4_t kf[RT][KS];  // zeros past dim
    bool whole = pos + kRows <= tree.cached;  // every query sees every row
#pragma unroll
    for (int t = 0; t < RT; ++t) whole = whole && there[t] == 0xffffu;
    // A tile of queries: lane (r, g) has query r's dims of its group. Tile after tile a lane's
    // query moves on by 16: by some nodes and heads.
    struct Queries {
      u32x4_t q[KS];
      float lse, count;
      uint32_t node;
    };
    for (uint32_t h = hw; any && h < a.kv_heads; h += w.head_waves) {
      uint32_t node = r / a.group, head = r - node * a.group, left = queries;  // of the next tile
      auto load_queries = [&](Queries& x) {
        const bool on = r < left;
        x.node = tree.first + (on ? node : 0u);
        const uint32_t at = h * a.group + (on ? head : 0u);
        const uint8_t* src = a.q + x.node * a.q_node + at * a.q_head;
#pragma unroll
        for (int j = 0; j < KS; ++j) {  // a form's dims start above the form in front: DV 4, 8, 12, 16
          const bool in = 2 * j + 2 <= DV - 4 || 32 * j + 8 * g < a.dim;
          const u32x4_t v = *reinterpret_cast<const u32x4_t*>(src + (in ? 64 * j + 16 * g : 0u));
          x.q[j] = in ? v : u32x4_t{0, 0, 0, 0};  // zeros that meet K's
        }
        x.lse = w.lse[static_cast<int64_t>(x.node) * a.heads + at];
        x.count = w.counted == nullptr ? 1.0f : w.counted[x.node];
        if (!on) x.count = 0.0f;
        head += w.step_head;
        node += w.step_node + (head >= a.group ? 1u : 0u);
        head -= head >= a.group ? a.group : 0u;
        left = left > 16 ? left - 16 : 0u;
      };
      auto take = [&](const Queries& x) {
        const bool live = x.lse != -INFINITY && x.count != 0.0f;
        const float minus = -x.lse * kLog2e;
        f32x4_t sc[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          sc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < KS; ++j) sc[t] = E::mfma(kf[t][j], x.q[j], sc[t]);
        }
        auto add = [&](int t, int e, bool on) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sc[t][e], a.scale, minus));
          sum[t][e] = on ? fmaf(p, x.count, sum[t][e]) : sum[t][e];
        };
        if (whole) {
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) add(t, e, live);
        } else {
          uint32_t from = 4 * g;
          asm volatile("" : "+v"(from));  // in this branch, not computed ahead of it for every tile
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            uint32_t seen = (there[t] & seen_bits(a.mask + static_cast<int64_t>(x.node) * a.mask_words, a.mask_words,
                                                  tree.cached, pos + 16 * t)) >> from;
            seen = live ? seen : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) add(t, e, seen >> e & 1u);
          }
        }
      };
      Queries x;
      load_queries(x);
#pragma unroll
      for (int t = 0; t < RT; ++t)
        load_tile<E, KS, FOUR>(a.k + at[t] + h * a.head_bytes, a.page.d, in_page[t], g, a.dim, kf[t]);
      for (;;) {
        take(x);
        if (left == 0) break;
        load_queries(x);
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[t][e] = group_sum_last<16>(sum[t][e]);
      if (r == 15) *reinterpret_cast<f32x4_t*>(&s_sum[wave][16 * t + 4 * g]) = sum[t];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < row_waves * kRows; i += 64 * kWaves) {
      if (base + i >= end) break;
      float total = 0.0f;
      for (uint32_t h = 0; h < w.head_waves; ++h) total += s_sum[i / kRows * w.head_waves + h][i % kRows];
      w.mass[s * w.mass_stride + base + i] += total;
    }
    __syncthreads();
  }
}

template <typename E, int DV, bool FOUR>
int launch(const WeighArgs& w, int64_t max_len, hipStream_t s) {
  constexpr int kMany = DV == 16 ? 3 : DV == 12 ? 4 : 5;
  // Three tiles of queries and more: more rows a wave, where that keeps every CU busy.
  const int64_t tiles = ceil_div(static_cast<int64_t>(w.t.max_tree) * w.t.group, 16);
  const int64_t row_waves = kWaves / w.head_waves;
  const bool many = tiles >= 3 && ceil_div(max_len, row_waves * 16 * kMany) * w.t.seqs >= device_cu_count();
  const int64_t rows = row_waves * 16 * (many ? kMany : 2);
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, ceil_div(max_len, rows))), w.t.seqs);
  if (many)
    hipLaunchKernelGGL((weigh_kernel<E, DV, FOUR, kMany>), grid, dim3(64 * kWaves), 0, s, w);
  else
    hipLaunchKernelGGL((weigh_kernel<E, DV, FOUR, 2>), grid, dim3(64 * kWaves), 0, s, w);
  return launch_status();
}

// What both forms check and launch; row_step, head_bytes and page_step as the kernel takes them.
int weigh(bool four, int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
          int64_t heads, const void* k, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim, int64_t page_step,
          int64_t row_step, int64_t head_bytes, const int32_t* table, int64_t table_stride, int64_t table_cols,
          const int32_t* lens, const int32_t* cu, int64_t seqs, const uint64_t* mask, int64_t mask_words,
          int64_t max_len, int64_t max_tree, float scale, const float* lse, const float* counted, float* mass,
          int64_t mass_stride, int64_t mass_cols, void* stream) {
  if (type != SPIRAL_TYPE_BF16 && type != SPIRAL_TYPE_F16) return SPIRAL_ERR_TYPE;
  if (!sizes_ok(nodes, heads, kv_heads, dim, seqs, max_len, max_tree) || !table_ok(table_cols, table_stride) ||
      pages <= 0 || pages > INT32_MAX || page <= 0 || page > INT32_MAX || mask_words < 0 || mask_words > (1 << 18) ||
      !std::isfinite(scale) || scale <= 0.0f || mass_cols < 0 || mass_cols > INT32_MAX || mass_stride < mass_cols ||
      mass_stride > (int64_t(1) << 40) || page_step > UINT32_MAX || row_step > UINT32_MAX)
    return SPIRAL_ERR_SHAPE;
  for (int64_t v8 : {q_node_stride, q_head_stride}) {
    if (v8 < 0 || v8 > (int64_t(1) << 40)) return SPIRAL_ERR_SHAPE;
    if (v8 % 8 != 0) return SPIRAL_ERR_ALIGN;
  }
  if (nodes == 0 || seqs == 0 || max_tree == 0 || mass_cols == 0) return SPIRAL_OK;
  if (q == nullptr || k == nullptr || (table == nullptr && table_cols > 0) || lens == nullptr || cu == nullptr ||
      (mask == nullptr && mask_words > 0) || lse == nullptr || mass == nullptr)
    return SPIRAL_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || (reinterpret_cast<uintptr_t>(mask) & 7u) != 0 ||
      !words_aligned({table, lens, cu, lse, counted, mass}))
    return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  WeighArgs w{};
  w.t.q = static_cast<const uint8_t*>(q), w.t.q_node = q_node_stride * 2, w.t.q_head = q_head_stride * 2;
  w.t.nodes = static_cast<uint32_t>(nodes), w.t.heads = static_cast<uint32_t>(heads);
  w.t.group = static_cast<uint32_t>(heads / kv_heads), w.t.k = static_cast<const uint8_t*>(k);
  w.t.pages = static_cast<uint32_t>(pages), w.t.kv_heads = static_cast<uint32_t>(kv_heads);
  w.t.dim = static_cast<uint32_t>(dim), w.t.page_step = static_cast<uint32_t>(page_step);
  w.t.row_step = static_cast<uint32_t>(row_step), w.t.head_bytes = head_bytes;
  w.t.page = Divisor(static_cast<uint32_t>(page)), w.t.table = table, w.t.table_stride = table_stride;
  w.t.table_cols = static_cast<uint32_t>(table_cols), w.t.lens = lens, w.t.cu = cu;
  w.t.seqs = static_cast<uint32_t>(seqs), w.t.mask = mask, w.t.mask_words = static_cast<uint32_t>(mask_words);
  w.t.scale = scale * kLog2e, w.t.max_tree = static_cast<uint32_t>(max_tree);
  w.lse = lse, w.counted = counted, w.mass = mass, w.mass_stride = mass_stride;
  w.mass_cols = static_cast<uint32_t>(mass_cols), w.head_waves = 1;
  while (w.head_waves < kWaves && 2 * w.head_waves <= kv_heads) w.head_waves *= 2;
  w.step_node = 16 / w.t.group, w.step_head = 16 % w.t.group;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int dv = dim <= 64 ? 4 : dim <= 128 ? 8 : dim <= 192 ? 12 : 16;
#define SPIRAL_WEIGH(E, FOUR)                           \
  (dv == 4    ? launch<E, 4, FOUR>(w, max_len, s)       \
   : dv == 8  ? launch<E, 8, FOUR>(w, max_len, s)       \
   : dv == 12 ? launch<E, 12, FOUR>(w, max_len, s)      \
              : launch<E, 16, FOUR>(w, max_len, s))
  if (type == SPIRAL_TYPE_BF16) return four ? SPIRAL_WEIGH(Bf16, true) : SPIRAL_WEIGH(Bf16, false);
  return four ? SPIRAL_WEIGH(F16, true) : SPIRAL_WEIGH(F16, false);
#undef SPIRAL_WEIGH
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int spiral_cache_row_weights(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                             int64_t heads, const void* k, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                             int64_t page_stride, int64_t row_stride, int64_t head_stride, const int32_t* table,
                             int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* cu,
                             int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len, int64_t max_tree,
                             float scale, const float* lse, const float* counted, float* mass, int64_t mass_stride,
                             int64_t mass_cols, void* stream) {
  for (int64_t v8 : {page_stride, row_stride, head_stride}) {
    if (v8 < 0 || v8 > (int64_t(1) << 35)) return SPIRAL_ERR_SHAPE;
    if (v8 % 8 != 0) return SPIRAL_ERR_ALIGN;
  }
  return weigh(false, type, q, q_node_stride, q_head_stride, nodes, heads, k, pages, page, kv_heads, dim,
               page_stride / 8, row_stride / 8, head_stride * 2, table, table_stride, table_cols, lens, cu, seqs, mask,
               mask_words, max_len, max_tree, scale, lse, counted, mass, mass_stride, mass_cols, stream);
}

int spiral_cache4_row_weights(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                              int64_t heads, const void* k, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                              int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                              const int32_t* lens, const int32_t* cu, int64_t seqs, const uint64_t* mask,
                              int64_t mask_words, int64_t max_len, int64_t max_tree, float scale, const float* lse,
                              const float* counted, float* mass, int64_t mass_stride, int64_t mass_cols,
                              void* stream) {
  if (!sizes4_ok(pages, page, kv_heads, dim, page_stride)) return SPIRAL_ERR_SHAPE;
  return weigh(true, type, q, q_node_stride, q_head_stride, nodes, heads, k, pages, page, kv_heads, dim,
               page_stride / 16, 0, Block4{static_cast<uint32_t>(page), static_cast<uint32_t>(dim)}.bytes(), table,
               table_stride, table_cols, lens, cu, seqs, mask, mask_words, max_len, max_tree, scale, lse, counted, mass,
               mass_stride, mass_cols, stream);
}

}  // extern "C"

// Attention of drafted trees over a paged cache in 4 bits (spiral_cache.h): tree.hip's
// products and running softmax with K and V as MXFP4 codes.
//
// A wave takes chunks of 32 rows, two tiles of 16, each in one page. Lane (r, g) of a
// product loads the codes that it needs as they lie, and makes 16-bit pairs of them
// (v_cvt_scalef32_pk, two exact values an instruction):
//   K: 16 bytes, one block of row r (8 where dim <= 64, two of 16 past 128): the four
//      words are the operands of four products. Which dims these stand for is up to Q,
//      whose rows are loaded in the same order.
//   V: word r (4 bytes, 8 dims; 2 bytes where dim <= 64) of the eight rows of its group,
//      so the lanes of a group read a whole row; v_perm_b32 pairs up rows.
// So no value of the cache passes through LDS, and no wave waits for another until the rows are
// done. The bound is the codes' bytes for few queries a row: a CU needs some 40 KiB of
// loads in flight for these, a chunk of dim 128 is 4.3 KiB, so a wave asks for the next two
// chunks (one, where registers hold no more) before it works on the one it has: 64
// sequences of 16384 rows, one query of 32 heads each, 8 cached: 121 us, 4.5 TB/s of the 5.1
// that a copy reaches (one chunk ahead 144). With more queries it is latency: a chunk is a
// chain of products, exponentials and products again, two waves a SIMD keep its vector
// unit busy for half of the time, and each query's sums take the registers of more. Where
// registers would hold fewer waves with them, Q's rows lie in LDS.
//
// A workgroup's four waves have other queries where a tree has as many and other rows
// where it has not (the tree decides, not the call: 16 ragged sequences of up to 25
// nodes: 85 us with the longest tree's division for all, 72 with each tree's own, 61 with rows
// dealt by the time that these take). Waves that share queries
// join their sums through LDS, halving their number each time, lane to lane; workgroups'
// parts of a sequence go through the workspace (tree_join_kernel).
#include "cache4.h"
#include "tree.h"

namespace spiral {
namespace {

// A chunk as loaded. W: blocks of K a lane has, words of V a row.
template <int DV>
struct RawK {
  static constexpr int W = DV == 16 ? 2 : 1, kWords = DV == 4 ? 2 : 4;  // words of a lane's block
  uint32_t codes[2][W][kWords];
  uint32_t scale[2][W];
};
template <int DV>
struct RawV {
  static constexpr int W = DV == 16 ? 2 : 1;
  uint32_t codes[8][W];
  uint32_t scale[2][W];  // a byte each for four rows
};

constexpr int kWaves = 4;

// Workgroups a CU that registers allow.
constexpr int occupancy4(int dv, int qt) { return dv * qt <= 4 ? 4 : dv * qt <= 8 ? 3 : 2; }

template <typename E, int DV, int QT>
struct Shape4 {
  static constexpr int W = DV == 16 ? 2 : 1, kQueries = 16 * QT;
  // Q in LDS, read again for every chunk, where registers would hold fewer waves with it.
  static constexpr bool kQLds = DV * QT >= 16;
  static constexpr int kQBytes = kQLds ? QT * (DV / 2) * 1024 : 0;  // a wave's
  static constexpr int kSlab = QT * (DV * 4 + 2) * 64;                      // floats of a wave's sums
  static constexpr int kLds = 2 * kSlab * 4 > kWaves * kQBytes ? 2 * kSlab * 4 : kWaves * kQBytes;
  static constexpr int kOccupancy = occupancy4(DV, QT);
};

// FULL: dim is 16 DV.
template <typename E, int DV, bool FULL, int QT>
__global__ void __launch_bounds__(256, (Shape4<E, DV, QT>::kOccupancy)) tree4_kernel(TreeArgs a) {
  using S = Shape4<E, DV, QT>;
  constexpr int KS = DV / 2, kQueries = S::kQueries, W = S::W;
  extern __shared__ __align__(16) float slabs[];
  const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Workgroups of the same rows and other queries run on one XCD, one after the other.
  const uint32_t unit = (blockIdx.x / 8 / a.query_groups) * 8 + blockIdx.x % 8;
  const uint32_t qg0 = blockIdx.x / 8 % a.query_groups;
  const uint32_t index = unit / a.kv_heads, h = (unit + index) % a.kv_heads;
  if (index >= a.shares) return;
  Share share(a, lane);
  if (!share.find(a, index, lane)) return;
  const uint32_t s = share.seq;
  const Tree tree(a, s);
  const uint32_t row0 = share.split * share.span;
  const uint32_t row1 = min(tree.rows, row0 + share.span);
  const uint32_t queries = tree.count * a.group;
  const int32_t* table = a.table + s * a.table_stride;
  const uint32_t page = a.page.d, half = FULL ? 8 * DV : a.dim / 2;
  const uint32_t scales = page * half;
  // Of the four waves QB have other queries, as many as this tree has use for, and KW other rows.
  const uint32_t QB = 1u << log_query_waves(a, queries), KW = kWaves / QB;
  const uint32_t qb = wave % QB, kp = wave / QB;

  // The two tiles of a chunk: their pages' ids, and rows in these. Past the last row they are some
  // tile of its page. One chunk after the other without divisions.
  struct Tiles {
    uint32_t id[2], row[2];
  };
  struct Cursor {
    uint32_t entry, row;  // of the table, in the page
  };
  const uint32_t last_entry = a.page.quotient(max(row1, 1u) - 1);
  auto at_row = [&](uint32_t pos) {
    const uint32_t q = a.page.quotient(pos);
    return Cursor{q, pos - q * page};
  };
  auto look = [&](Cursor c) {
    const uint32_t more = c.row + 16 >= page ? 1u : 0u;
    Tiles x;
    x.row[0] = c.row, x.row[1] = more ? 0u : c.row + 16;
    x.id[0] = static_cast<uint32_t>(table[min(c.entry, last_entry)]);
    x.id[1] = static_cast<uint32_t>(table[min(c.entry + more, last_entry)]);
    return x;
  };
  // Bits of the rows of the chunk at `pos` that there are. A negative id is past every page.
  auto rows_there = [&](uint32_t pos, const Tiles& x) {
    const uint32_t left = row1 > pos ? row1 - pos : 0u;
    const uint32_t there = left >= 32u ? ~0u : (1u << left) - 1u;
    return there & ((x.id[0] < a.pages ? 0x0000ffffu : 0u) | (x.id[1] < a.pages ? 0xffff0000u : 0u));
  };
  // Where tile t lies, from the head's block in the first page (of which there is one).
  auto offset = [&](const Tiles& x, int t) {
    return static_cast<uint64_t>(x.id[t] < a.pages ? x.id[t] : 0u) * a.page_step * 16;
  };
  const uint8_t* k0 = a.k + h * a.head_bytes;
  const uint8_t* v0 = a.v + h * a.head_bytes;
  // Lanes past dim read what lies at 0 in its place: K's codes are finite under a scale of
  // one and meet zeros in Q, V's dims are not stored.
  uint32_t k_at[W], v_at[W], ks_at[W], vs_at[W];
  bool k_on[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    k_on[w] = FULL || (DV == 4 ? 16 * g : 128 * w + 32 * g) < a.dim;
    const bool v_on = FULL || (DV == 4 ? 4 * r : 128 * w + 8 * r) < a.dim;
    k_at[w] = r * half + (k_on[w] ? (DV == 4 ? 8 : 16) * g + 64 * w : 0u);
    ks_at[w] = scales + r + (k_on[w] ? page * ((DV == 4 ? g / 2 : g) + 4 * w) : 0u);
    v_at[w] = 4 * g * half + (v_on ? (DV == 4 ? 2 : 4) * r + 64 * w : 0u);
    vs_at[w] = scales + 4 * g + (v_on ? page * ((DV == 4 ? r / 8 : r / 4) + 4 * w) : 0u);
  }
  auto load_k = [&](const Tiles& c, RawK<DV>& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* block = k0 + offset(c, t);
      const uint8_t* codes = block + c.row[t] * half;
      const uint8_t* sc = block + c.row[t];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if constexpr (DV == 4) {
          const u32x2_t q = *reinterpret_cast<const u32x2_t*>(codes + k_at[w]);
          x.codes[t][w][0] = q.x, x.codes[t][w][1] = q.y;
        } else {
          const u32x4_t q = *reinterpret_cast<const u32x4_t*>(codes + k_at[w]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x.codes[t][w][i] = q[i];
        }
        x.scale[t][w] = sc[ks_at[w]];
      }
    }
  };
  auto load_v = [&](const Tiles& c, RawV<DV>& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* block = v0 + offset(c, t);
      const uint8_t* codes = block + c.row[t] * half;
      const uint8_t* sc = block + c.row[t];
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t* src = codes + (v_at[w] + e * half);
          x.codes[4 * t + e][w] =
              DV == 4 ? *reinterpret_cast<const uint16_t*>(src) : *reinterpret_cast<const uint32_t*>(src);
        }
        x.scale[t][w] = *reinterpret_cast<const uint32_t*>(sc + vs_at[w]);
      }
    }
  };
  // A query's row of q, and its line of the workspace for this part.
  auto row_of_query = [&](uint32_t at) {
    return static_cast<int64_t>(tree.first + at / a.group) * a.heads + h * a.group + at % a.group;
  };
  auto line_of_query = [&](uint32_t at) {
    return static_cast<int64_t>(share.line + share.split * tree.count + at / a.group) * a.heads + h * a.group +
           at % a.group;
  };
  // Chunks that reach past the cached rows, or miss rows, are masked.
  auto is_masked = [&](uint32_t pos, uint32_t there) { return there != ~0u || pos + kChunk > tree.cached; };
  auto seen_by = [&](uint32_t node, uint32_t pos, uint32_t there) {
    return there & seen_bits(a.mask + static_cast<int64_t>(node) * a.mask_words, a.mask_words, tree.cached, pos);
  };

  for (uint32_t qg = qg0; qg * (QB * kQueries) < queries; qg += a.query_groups) {
    const uint32_t q0 = (qg * QB + qb) * kQueries;
    Sums<E, DV, QT> sums;
    sums.clear();
    uint32_t node[QT];
    bool odd_values = false;  // a masked chunk had infinities or NaN
    if (q0 < queries) {
      // Q^T: lane (r, g) has dims 32 g + 8 j .. + 7 of query r (16 g + 8 j where DV = 4).
      u32x4_t qf[S::kQLds ? 1 : QT][S::kQLds ? 1 : KS];
      u32x4_t* q_lds = reinterpret_cast<u32x4_t*>(reinterpret_cast<uint8_t*>(slabs) + wave * S::kQBytes) + lane;
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const uint32_t i = min(q0 + 16 * t + r, queries - 1);
        node[t] = tree.first + i / a.group;
        const uint8_t* src = a.q + node[t] * a.q_node + (h * a.group + i % a.group) * a.q_head;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const uint32_t d = DV == 4 ? 16 * g + 8 * j : 128 * (j / 4) + 32 * g + 8 * (j % 4);
          const bool on = FULL || d < a.dim;
          u32x4_t w = *reinterpret_cast<const u32x4_t*>(src + (on ? 2 * d : 0u));
          w = on ? w : u32x4_t{0, 0, 0, 0};
          if constexpr (S::kQLds)
            q_lds[(t * KS + j) * 64] = w;
          else
            qf[t][j] = w;
        }
      }
      auto q_of = [&](int t, int j) {
        if constexpr (S::kQLds)
          return q_lds[(t * KS + j) * 64];
        else
          return qf[t][j];
      };

      // Chunk after chunk, kAhead of them asked for ahead: K of the one after these when this
      // one's has been used, and so V.
      constexpr int kAhead = DV * QT <= 8 ? 2 : 1;
      const uint32_t step = KW * kChunk, step_entries = a.page.quotient(step), step_rows = step - step_entries * page;
      uint32_t pos = row0 + kp * kChunk, there[kAhead];
      RawK<DV> rk[kAhead];
      RawV<DV> rv[kAhead];
      Cursor cursor = at_row(pos);
      auto advance = [&]() {
        cursor.row += step_rows, cursor.entry += step_entries;
        if (cursor.row >= page) cursor.row -= page, ++cursor.entry;
      };
      Tiles next;
      if (pos < row1) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const Tiles c = look(cursor);
          advance();
          there[i] = rows_there(pos + i * step, c);
          load_k(c, rk[i]);
          load_v(c, rv[i]);
        }
        next = look(cursor);
      }
      auto take = [&](RawK<DV>& k, RawV<DV>& v, uint32_t& there_of) {
        f32x4_t sc[QT][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][0] = sc[t][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kWords = RawK<DV>::kWords;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          u32x4_t qj[QT];
#pragma unroll
          for (int t = 0; t < QT; ++t) qj[t] = q_of(t, j);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t w = k.codes[u][j / kWords][j % kWords];
            const float f = k_on[j / kWords] ? scale_byte<0>(k.scale[u][j / kWords]) : 1.0f;
            const u32x4_t kf{fp4_pair<E, 0>(w, f), fp4_pair<E, 1>(w, f), fp4_pair<E, 2>(w, f), fp4_pair<E, 3>(w, f)};
#pragma unroll
            for (int t = 0; t < QT; ++t) sc[t][u] = E::mfma(kf, qj[t], sc[t][u]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t there_now = there_of;
        const Tiles c = next;
        there_of = rows_there(pos + kAhead * step, c);
        advance();
        next = look(cursor);
        load_k(c, k);
        __builtin_amdgcn_sched_barrier(0);
        if (is_masked(pos, there_now)) {
          uint32_t group = g;
          asm volatile("" : "+v"(group));  // in this branch, not computed ahead of it for every chunk
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const uint32_t seen = seen_by(node[t], pos, there_now) >> (4 * group);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (!(seen >> row_of(0, e) & 1u)) sc[t][e / 4][e % 4] = -INFINITY;
          }
          // Rows that are not there count as zeros, and so do codes that are infinities or
          // NaN, which not every query sees: they are added behind the loop.
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool on = there_now >> (4 * group) >> row_of(0, e) & 1u;
#pragma unroll
            for (int w = 0; w < W; ++w) {
              uint32_t& sw = v.scale[e / 4][w];
              const uint32_t scale = sw >> (8 * (e % 4)) & 0xffu;
              const uint32_t odd = first_odd_code(scale, E::kF16);
              if (!on || odd == 0u) {
                bad = bad || (on && odd == 0u);
                v.codes[e][w] = 0u;
                sw = (sw & ~(0xffu << (8 * (e % 4)))) | 127u << (8 * (e % 4));
              } else if (odd < 8u) {
#pragma unroll 1
                for (uint32_t i = 0; i < 32; i += 4)
                  if ((v.codes[e][w] >> i & 7u) >= odd) bad = true, v.codes[e][w] &= ~(15u << i);
              }
            }
          }
          odd_values = __builtin_amdgcn_ballot_w64(bad) != 0 || odd_values;
        }
        u32x4_t pf[QT];
        sums.soften(sc, a.scale, pf);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t s0 = v.scale[0][w], s1 = v.scale[1][w];
          const float f[8] = {scale_byte<0>(s0), scale_byte<1>(s0), scale_byte<2>(s0), scale_byte<3>(s0),
                              scale_byte<0>(s1), scale_byte<1>(s1), scale_byte<2>(s1), scale_byte<3>(s1)};
          auto two = [&](auto sel) {
            constexpr int J = decltype(sel)::value;
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fp4_pair<E, J>(v.codes[e][w], f[e]);
            u32x4_t lo, hi;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              lo[i] = __builtin_amdgcn_perm(y[2 * i + 1], y[2 * i], 0x05040100u);
              hi[i] = __builtin_amdgcn_perm(y[2 * i + 1], y[2 * i], 0x07060302u);
            }
            sums.add(lo, pf, 8 * w + 2 * J);
            sums.add(hi, pf, 8 * w + 2 * J + 1);
          };
          two(std::integral_constant<int, 0>{});
          two(std::integral_constant<int, 1>{});
          if constexpr (DV != 4) {
            two(std::integral_constant<int, 2>{});
            two(std::integral_constant<int, 3>{});
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(c, v);
        pos += step;
      };
      while (pos < row1) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          take(rk[i], rv[i], there[i]);
          if (pos >= row1) break;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) sums.sum[t] = across_groups_sum(sums.sum[t]);

    // Join the waves of a query block, the upper half's sums onto the lower's.
    if (KW > 1) {
      if (S::kQLds) __syncthreads();  // Q has been read
      for (uint32_t n = KW / 2; n > 0; n /= 2) {
        float* slab = slabs + (kp % n * QB + qb) * S::kSlab + lane * 4;
        if (kp >= n && kp < 2 * n) {
#pragma unroll
          for (int t = 0; t < QT; ++t) {
#pragma unroll
            for (int d = 0; d < DV; ++d) *reinterpret_cast<f32x4_t*>(slab + (t * DV + d) * 256) = sums.o[t][d];
            *reinterpret_cast<float2*>(slab - lane * 2 + QT * DV * 256 + t * 128) = make_float2(sums.top[t], sums.sum[t]);
          }
        }
        __syncthreads();
        if (kp < n) {
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const float2 o = *reinterpret_cast<const float2*>(slab - lane * 2 + QT * DV * 256 + t * 128);
            const float m = fmaxf(sums.top[t], o.x);
            const float f0 = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sums.top[t] - m);
            const float f1 = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(o.x - m);
            sums.top[t] = m;
            sums.sum[t] = sums.sum[t] * f0 + o.y * f1;
#pragma unroll
            for (int d = 0; d < DV; ++d)
              sums.o[t][d] = sums.o[t][d] * f0 + *reinterpret_cast<const f32x4_t*>(slab + (t * DV + d) * 256) * f1;
          }
        }
        __syncthreads();  // also: the slabs are read to their end before they are written again
      }
    }
    if (kp == 0 && q0 < queries) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const uint32_t at = q0 + 16 * t + r;
        if (at >= queries) continue;
        const int64_t row = row_of_query(at), line = line_of_query(at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < DV / 4; ++c) {
            const uint32_t d = DV == 4 ? 4 * (4 * g + i) : 128 * (c / 2) + 8 * (4 * g + i) + 4 * (c % 2);
            if (!FULL && d >= a.dim) continue;
            const f32x4_t v{sums.o[t][4 * c][i], sums.o[t][4 * c + 1][i], sums.o[t][4 * c + 2][i],
                            sums.o[t][4 * c + 3][i]};
            if (share.parts > 1) {
              *reinterpret_cast<f32x4_t*>(a.part + line * a.dim + d) = v;
              if (d == 0) a.part_ml[line] = make_float2(sums.top[t], sums.sum[t]);
            } else {
              write<E>(a, row, d, v, sums.top[t], sums.sum[t]);
            }
          }
      }
    }
    // Rare: the masked chunks' infinities and NaN, added to what was written for the queries
    // that see their rows, a dim of a query a thread.
    if (__syncthreads_or(odd_values)) {
      for (uint32_t i = threadIdx.x; i < QB * kQueries * a.dim; i += 256) {
        const uint32_t at = qg * (QB * kQueries) + i / a.dim, d = i % a.dim;
        if (at >= queries) break;
        float more = 0.0f;
        for (uint32_t pos = row0; pos < row1; pos += kChunk) {
          const Tiles x = look(at_row(pos));
          const uint32_t there = rows_there(pos, x);
          if (!is_masked(pos, there)) continue;
          uint32_t seen = seen_by(tree.first + at / a.group, pos, there);
          for (; seen != 0; seen &= seen - 1) {
            const uint32_t j = __builtin_ctz(seen), p = pos + j, in_page = p - a.page.quotient(p) * page;
            const uint8_t* block = v0 + offset(x, j < 16 ? 0 : 1);
            const uint32_t c = block[in_page * half + d / 2] >> (4 * (d % 2)) & 15u;
            const uint32_t odd = first_odd_code(block[scales + d / 32 * page + in_page], E::kF16);
            if ((c & 7u) >= odd) more += odd == 0u ? NAN : c & 8u ? -INFINITY : INFINITY;
          }
        }
        if (more == 0.0f) continue;
        if (share.parts > 1) {
          a.part[line_of_query(at) * a.dim + d] += more;
        } else {
          uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + row_of_query(at) * a.dim + d;
          *o = static_cast<uint16_t>(E::pack(E::value(*o) + more, 0.0f));
        }
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------

// How the queries and rows of a call are divided.
struct Plan {
  int dv, qt, qb;
  int64_t query_groups, step, least, want, shares, lines;
  bool by_work;
};

// As in tree.hip, with this kernel's workgroups a CU, and:
// - From 32 tiles of queries on a wave has four of them where registers hold their sums (a
//   chunk of 512 nodes over 16384 rows, 32 heads: 235 us with two, 198 with four; 64 nodes over
//   8 sequences of 4096: 56 and 66).
// - Short sequences stay whole: a join costs as much as a few steps.
// - Where rows are divided, more than four waves of queries are other workgroups: of two
//   waves of queries, or of one of dim 256, whose four waves share a partial sum (two sequences
//   of 65536 rows, 64 nodes, dim 256: 71 us with four waves of queries, 66 with two, 64 with one, the
//   join of partial sums 13.7, 9.1, 6.9; 8 cached heads of dim 128: 99, 91, 97).
// - Parts for two rounds of workgroups where each has one tile and sequences are many, so that
//   the last to end are short (64 x 16384 rows, a query each: 122 us, 132 with one round).
Plan make_plan(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, int64_t max_len, int64_t max_tree,
               int64_t lines) {
  Plan p;
  p.dv = dim <= 64 ? 4 : dim <= 128 ? 8 : 16;
  const int64_t tiles = std::max<int64_t>(1, ceil_div(max_tree * (heads / kv_heads), 16));
  p.qt = tiles == 1 ? 1 : tiles < 32 || p.dv == 16 ? 2 : 4;
  const int64_t blocks = ceil_div(tiles, p.qt);
  p.step = kChunk * kWaves;
  p.least = blocks == 1 ? 1 : 4;
  p.want = 0, p.shares = seqs, p.lines = 0, p.by_work = false;
  p.qb = 4, p.query_groups = ceil_div(blocks, 4);
  const int64_t all = occupancy4(p.dv, p.qt) * device_cu_count();
  if (max_len <= 4 * p.step || seqs > kMostDealt || (seqs == 1 && kv_heads * p.query_groups >= all)) return p;
  if (blocks > 4) p.qb = p.dv == 16 ? 1 : 2, p.query_groups = ceil_div(blocks, p.qb);
  const int64_t group = kv_heads * p.query_groups;
  p.by_work = seqs * group >= 3 * all;
  const int64_t places = std::max<int64_t>(1, all / (p.by_work ? kv_heads : group));
  const int64_t rounds = std::max<int64_t>(ceil_div(3 * seqs, 2 * places), p.qt > 1 || places >= 8 * seqs ? 1 : 2);
  const int64_t want = p.by_work ? places : places * rounds;
  const int64_t most =
      std::min({std::min(want + seqs, 2 * want) * max_tree, lines, kMostBytes / line_bytes(heads, dim)});
  if (want > 1 && most > 1) p.want = want, p.shares = want + seqs, p.lines = most;
  return p;
}

template <typename E, int DV, bool FULL, int QT>
int launch(const TreeArgs& a, const Plan& p, hipStream_t s) {
  constexpr int lds = Shape4<E, DV, QT>::kLds;
  const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&tree4_kernel<E, DV, FULL, QT>), lds);
  if (rc != SPIRAL_OK) return rc;
  const int64_t units = ceil_div(p.shares * a.kv_heads, 8) * 8;
  if (units * p.query_groups > INT32_MAX) return SPIRAL_ERR_SHAPE;
  hipLaunchKernelGGL((tree4_kernel<E, DV, FULL, QT>), dim3(static_cast<unsigned>(units * p.query_groups)), dim3(256), lds,
                     s, a);
  return launch_status();
}

template <typename E, int DV>
int launch_tiles(const TreeArgs& a, const Plan& p, hipStream_t s) {
  if constexpr (DV <= 8) {
    if (p.qt == 4) return a.dim == 16 * DV ? launch<E, DV, true, 4>(a, p, s) : launch<E, DV, false, 4>(a, p, s);
  }
  if (a.dim == 16 * DV) return p.qt == 1 ? launch<E, DV, true, 1>(a, p, s) : launch<E, DV, true, 2>(a, p, s);
  return p.qt == 1 ? launch<E, DV, false, 1>(a, p, s) : launch<E, DV, false, 2>(a, p, s);
}

template <typename E>
int run_tree(const TreeArgs& a, const Plan& p, int64_t max_tree, hipStream_t s) {
  const int rc = p.dv == 4   ? launch_tiles<E, 4>(a, p, s)
                 : p.dv == 8 ? launch_tiles<E, 8>(a, p, s)
                             : launch_tiles<E, 16>(a, p, s);
  if (rc != SPIRAL_OK || p.want == 0) return rc;
  return launch_join<E>(a, static_cast<uint32_t>(p.want), max_tree, s);
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int64_t spiral_cache4_tree_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs,
                                                     int64_t max_len, int64_t max_tree) {
  if (!sizes_ok(0, heads, kv_heads, dim, seqs, max_len, max_tree) || dim % 32 != 0) return 0;
  const Plan p = make_plan(heads, kv_heads, dim, seqs, max_len, max_tree, INT64_MAX);
  return p.lines * line_bytes(heads, dim);
}

int spiral_cache4_tree_attention(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                                 int64_t heads, const void* k, const void* v, int64_t pages, int64_t page,
                                 int64_t kv_heads, int64_t dim, int64_t page_stride, const int32_t* table,
                                 int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* cu,
                                 int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len,
                                 int64_t max_tree, float scale, void* out, float* lse, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (type != SPIRAL_TYPE_BF16 && type != SPIRAL_TYPE_F16) return SPIRAL_ERR_TYPE;
  if (!sizes_ok(nodes, heads, kv_heads, dim, seqs, max_len, max_tree) || pages == 0 ||
      !sizes4_ok(pages, page, kv_heads, dim, page_stride) || !table_ok(table_cols, table_stride) ||
      table_cols * page >= int64_t(1) << 28 || mask_words < 0 ||
      mask_words > (1 << 18) || !std::isfinite(scale) || scale <= 0.0f)
    return SPIRAL_ERR_SHAPE;
  for (int64_t v8 : {q_node_stride, q_head_stride}) {
    if (v8 < 0 || v8 > (int64_t(1) << 40)) return SPIRAL_ERR_SHAPE;
    if (v8 % 8 != 0) return SPIRAL_ERR_ALIGN;
  }
  if (page_stride / 16 > UINT32_MAX) return SPIRAL_ERR_SHAPE;
  if (nodes == 0 || seqs == 0 || max_tree == 0) return SPIRAL_OK;
  if (q == nullptr || k == nullptr || v == nullptr || (table == nullptr && table_cols > 0) || lens == nullptr ||
      cu == nullptr || (mask == nullptr && mask_words > 0) || out == nullptr)
    return SPIRAL_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(mask) & 7u) != 0 || !words_aligned({table, lens, cu, lse}))
    return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const int64_t lines = workspace == nullptr || workspace_bytes < 0 ? 0 : workspace_bytes / line_bytes(heads, dim);
  const Plan p = make_plan(heads, kv_heads, dim, seqs, max_len, max_tree, lines);
  const Block4 block{static_cast<uint32_t>(page), static_cast<uint32_t>(dim)};
  TreeArgs a{static_cast<const uint8_t*>(q), q_node_stride * 2, q_head_stride * 2, static_cast<uint32_t>(nodes),
             static_cast<uint32_t>(heads), static_cast<uint32_t>(heads / kv_heads), static_cast<const uint8_t*>(k),
             static_cast<const uint8_t*>(v), static_cast<uint32_t>(pages), static_cast<uint32_t>(kv_heads),
             static_cast<uint32_t>(dim), static_cast<uint32_t>(page_stride / 16), 0, block.bytes(),
             Divisor(static_cast<uint32_t>(page)), table, table_stride, static_cast<uint32_t>(table_cols), lens, cu,
             static_cast<uint32_t>(seqs), mask, static_cast<uint32_t>(mask_words), scale * kLog2e,
             static_cast<uint8_t*>(out), lse, nullptr, nullptr, static_cast<uint32_t>(p.lines),
             static_cast<uint32_t>(max_tree), static_cast<uint32_t>(p.query_groups), static_cast<uint32_t>(p.shares),
             static_cast<uint32_t>(p.want), static_cast<uint32_t>(p.step), static_cast<uint32_t>(p.least), p.by_work,
             Divisor(static_cast<uint32_t>(16 * p.qb * p.qt)), static_cast<uint32_t>(16 * p.qt),
             static_cast<uint32_t>(p.qb == 4 ? 2 : p.qb - 1)};
  if (p.want > 0) {
    a.part = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part + p.lines * heads * dim);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return type == SPIRAL_TYPE_BF16 ? run_tree<Bf16>(a, p, max_tree, s) : run_tree<F16>(a, p, max_tree, s);
}

}  // extern "C"

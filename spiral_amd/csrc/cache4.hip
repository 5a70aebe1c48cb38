// Rows of a paged cache in 4 bits (spiral_cache.h): stored, read back, and moved
// together. All three move bytes: HBM bounds the large calls (storing 7.4k rows of 32 heads of dim
// 128, keys and values, 40 us: 3.8 TB/s; reading one of both back 14.6: 5.3 TB/s), the launch
// and the dependent loads of lens, cu and table the small ones (2.4 to 2.8 us). Compaction of accepted
// nodes is as short (12 us with the call); that of an eviction, 16384 of 65536 rows in each of 8
// sequences, takes 244 us for 56 of bytes: moves in order, two waits a batch.
#include <algorithm>

#include "cache4.h"
#include "dequant_impl.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

constexpr int kThreads = 256;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// The nodes of a call and where their rows lie.
struct Rows4 {
  uint32_t nodes, kv_heads, blocks;  // blocks of 32 elements a row of one head
  uint32_t pages;
  int64_t page_stride;
  Divisor page, per_node, per_head;  // pieces of a node, of a head in it
  const int32_t* table;
  int64_t table_stride;
  uint32_t table_cols;
  const int32_t *lens, *cu;
  uint32_t seqs;

  // Offset of node i's row in its page and the page's first byte; false without a page.
  __device__ __forceinline__ bool find(uint32_t i, int64_t& base, uint32_t& row) const {
    uint32_t s = 0;  // the last sequence whose first node is not behind i
    for (uint32_t n = seqs; n > 1;) {
      const uint32_t half = n / 2;
      if (cu[s + half] <= static_cast<int32_t>(i)) s += half;
      n -= half;
    }
    const int32_t first = cu[s];
    if (first > static_cast<int32_t>(i) || cu[s + 1] <= static_cast<int32_t>(i)) return false;
    const PagedRows rows{table + s * table_stride, table_cols, pages, page};
    const int64_t pos = static_cast<int64_t>(max(lens[s], 0)) + (static_cast<int32_t>(i) - first);
    if (!rows.in_table(pos)) return false;
    const uint32_t id = rows.entry(pos);
    if (id >= pages) return false;  // a negative id is past every page
    base = id * page_stride, row = rows.row(pos);
    return true;
  }
};

template <int TYPE>
__device__ __forceinline__ void load8(const uint8_t* p, float (&x)[8]) {
  if constexpr (TYPE == SPIRAL_TYPE_F32) {
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = TYPE == SPIRAL_TYPE_BF16 ? bf16_lo(a[i]) : fp16_ieee(a[i] & 0xffffu);
      x[2 * i + 1] = TYPE == SPIRAL_TYPE_BF16 ? bf16_hi(a[i]) : fp16_ieee(a[i] >> 16);
    }
  }
}

// A workgroup takes kPieces pieces of 8 elements a thread, kThreads apart, of node after node.
// Where the rows of its nodes lie is looked up once a node, while its loads are on their way: a
// search of each piece for itself, and one load in flight a thread, took 56 us where this takes
// 40 (8 ragged sequences of up to 2000 rows, 32 heads of dim 128).
constexpr int kPieces = 4;
constexpr uint32_t kNodes = kThreads * kPieces / 4 + 1;  // of dim 32, one head, at most

// The workgroup's first piece: each XCD (every eighth workgroup) has one stretch of them, so that
// rows of one page, whose scale bytes share lines, meet in one L2.
__device__ __forceinline__ uint32_t first_piece() {
  return (blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8) * (kThreads * kPieces);
}
// Workgroups of a call, a multiple of eight.
int64_t groups_of(int64_t pieces) { return ceil_div(ceil_div(pieces, kThreads * kPieces), 8) * 8; }

struct Places {
  int64_t base[kNodes];  // of the node's page, negative without one
  uint32_t row[kNodes];
  __device__ __forceinline__ uint32_t find(const Rows4& a, uint32_t at0, uint32_t pieces) {
    const uint32_t first = a.per_node.quotient(at0);
    const uint32_t last = a.per_node.quotient(min(at0 + kThreads * kPieces, pieces) - 1);
    for (uint32_t i = threadIdx.x; i <= last - first; i += kThreads) {
      int64_t b = 0;
      uint32_t r = 0;
      if (!a.find(first + i, b, r)) b = -1;
      base[i] = b, row[i] = r;
    }
    __syncthreads();
    return first;
  }
};

// Four lanes a block; blockIdx.y: keys, values.
template <int TYPE>
__global__ void __launch_bounds__(kThreads)
    store_kernel(const uint8_t* new_k, const uint8_t* new_v, int64_t node_bytes, int64_t head_bytes, uint8_t* k,
                 uint8_t* v, Rows4 a, uint32_t pieces) {
  __shared__ Places places;
  constexpr int kSize = TYPE == SPIRAL_TYPE_F32 ? 4 : 2;
  const uint32_t at0 = first_piece();
  if (at0 >= pieces) return;
  float x[kPieces][8];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t at = min(at0 + j * kThreads + threadIdx.x, pieces - 1);
    const uint32_t i = a.per_node.quotient(at), in_node = at - i * a.per_node.d, h = a.per_head.quotient(in_node);
    load8<TYPE>((blockIdx.y == 0 ? new_k : new_v) + i * node_bytes + h * head_bytes +
                    (in_node - h * a.per_head.d) * (8 * kSize), x[j]);
  }
  const uint32_t first = places.find(a, at0, pieces);
  const Block4 block{a.page.d, 32 * a.blocks};
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t at = at0 + j * kThreads + threadIdx.x;
    if (at >= pieces) return;  // whole quads
    // Magnitudes order as their bits do, NaN and infinity above every number.
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[j][e]) & 0x7fffffffu);
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, false)));
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xF, 0xF, false)));
    top >>= 23;
    const uint32_t e = top == 255u ? 255u : top < 2u ? 0u : top - 2u;
    const float s = e8m0_scale(e);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[j][0], x[j][1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[j][2], x[j][3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[j][4], x[j][5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[j][6], x[j][7], s, 3);
    const uint32_t i = a.per_node.quotient(at), in_node = at - i * a.per_node.d, h = a.per_head.quotient(in_node);
    const uint32_t p = in_node - h * a.per_head.d, row = places.row[i - first];
    const int64_t base = places.base[i - first];
    if (base < 0) continue;
    uint8_t* to = (blockIdx.y == 0 ? k : v) + base + h * block.bytes();
    *reinterpret_cast<uint32_t*>(to + row * (16 * a.blocks) + 4 * p) = e == 255u ? 0u : q;
    if (p % 4 == 0) to[block.scales() + p / 4 * a.page.d + row] = static_cast<uint8_t>(e);
  }
}

template <bool HALF>
__global__ void __launch_bounds__(kThreads) load_kernel(const uint8_t* cache, Rows4 a, u32x4_t* out, uint32_t pieces) {
  __shared__ Places places;
  const uint32_t at0 = first_piece();
  if (at0 >= pieces) return;
  const uint32_t first = places.find(a, at0, pieces);
  const Block4 block{a.page.d, 32 * a.blocks};
  uint32_t w[kPieces], scale[kPieces];
  bool there[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t at = min(at0 + j * kThreads + threadIdx.x, pieces - 1);
    const uint32_t i = a.per_node.quotient(at), in_node = at - i * a.per_node.d, h = a.per_head.quotient(in_node);
    const uint32_t p = in_node - h * a.per_head.d, row = places.row[i - first];
    const int64_t base = places.base[i - first];
    there[j] = base >= 0;
    w[j] = scale[j] = 0;
    if (there[j]) {
      const uint8_t* from = cache + base + h * block.bytes();
      w[j] = *reinterpret_cast<const uint32_t*>(from + row * (16 * a.blocks) + 4 * p);
      scale[j] = from[block.scales() + p / 4 * a.page.d + row];
    }
  }
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t at = at0 + j * kThreads + threadIdx.x;
    if (at >= pieces) return;
    const float s = scale_byte<0>(scale[j]);
    u32x4_t x;
    if constexpr (HALF) {
      x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j], s, 0));
      x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j], s, 1));
      x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j], s, 2));
      x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[j], s, 3));
    } else {
      x[0] = fp4_bf16x2<0>(w[j], s), x[1] = fp4_bf16x2<1>(w[j], s);
      x[2] = fp4_bf16x2<2>(w[j], s), x[3] = fp4_bf16x2<3>(w[j], s);
    }
    if (!there[j]) x = u32x4_t{0u, 0u, 0u, 0u};
    __builtin_nontemporal_store(x, out + at);
  }
}

// ---- compaction -----------------------------------------------------------------

// cache.hip's compaction with a row in pieces: a block's 16 bytes of codes and its scale
// byte, kv_heads * dim / 32 of them a row. A workgroup owns `cols` pieces of one
// sequence, layer and array and takes the moves in order, all loads of a batch, a barrier,
// its stores: keep ascends strictly, so move j reads a row that no earlier move wrote.
constexpr int kMoves = 8;

__global__ void __launch_bounds__(kThreads)
    compact4_kernel(uint8_t* k, uint8_t* v, uint32_t layers, int64_t layer_stride, uint32_t pages, int64_t page_stride,
                    Divisor page, uint32_t kv_heads, Divisor blocks, const int32_t* __restrict__ table,
                    int64_t table_stride, uint32_t table_cols, const int32_t* __restrict__ lens,
                    const int32_t* __restrict__ keep, int64_t keep_stride, uint32_t keep_cols,
                    const int32_t* __restrict__ kept, int32_t* __restrict__ new_lens, uint32_t log_cols) {
  const uint32_t s = blockIdx.y;
  const uint32_t l = blockIdx.z < layers ? blockIdx.z : blockIdx.z - layers;
  uint8_t* base = (blockIdx.z < layers ? k : v) + l * layer_stride;
  const uint32_t n = static_cast<uint32_t>(min(max(kept[s], 0), static_cast<int32_t>(keep_cols)));
  const int32_t first = lens[s];
  if (new_lens != nullptr && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) new_lens[s] = first + n;
  const uint32_t col = (blockIdx.x << log_cols) + (threadIdx.x & ((1u << log_cols) - 1));
  const uint32_t slot = threadIdx.x >> log_cols, step = kThreads >> log_cols;
  const PagedRows rows{table + s * table_stride, table_cols, pages, page};
  const int32_t* kp = keep + s * keep_stride;
  const uint32_t h = blocks.quotient(col), b = col - h * blocks.d;
  const Block4 block{page.d, 32 * blocks.d};
  const int64_t codes = h * block.bytes() + b * 16, scales = h * block.bytes() + block.scales() + b * page.d;

  int32_t from[kMoves];
  int64_t src[kMoves], dst[kMoves];
  uint32_t src_page[kMoves], dst_page[kMoves];
  auto ask_keep = [&](uint32_t j0) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const uint32_t j = j0 + i * step + slot;
      from[i] = j < n ? kp[j] : -1;
    }
  };
  auto ask_pages = [&](uint32_t j0) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int32_t j = static_cast<int32_t>(j0 + i * step + slot);
      src[i] = first + static_cast<int64_t>(from[i]), dst[i] = first + static_cast<int64_t>(j);
      const bool on = from[i] >= 0 && from[i] != j && h < kv_heads && rows.in_table(src[i]) && rows.in_table(dst[i]);
      if (!on) src[i] = -1;
      src_page[i] = on ? rows.entry(src[i]) : 0u, dst_page[i] = on ? rows.entry(dst[i]) : 0u;
    }
  };
  const uint32_t batch = kMoves * step;
  ask_keep(0);
  ask_pages(0);
  ask_keep(batch);
  for (uint32_t j0 = 0; j0 < n; j0 += batch) {
    u32x4_t data[kMoves];
    uint8_t scale[kMoves];
    uint8_t* to[kMoves];
    uint32_t to_row[kMoves];
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      to[i] = nullptr;
      if (src[i] < 0 || src_page[i] >= pages || dst_page[i] >= pages) continue;  // a negative id is past every page
      to[i] = base + dst_page[i] * page_stride, to_row[i] = rows.row(dst[i]);
      const uint8_t* p = base + src_page[i] * page_stride;
      const uint32_t row = rows.row(src[i]);
      data[i] = *reinterpret_cast<const u32x4_t*>(p + codes + row * (16 * blocks.d));
      scale[i] = p[scales + row];
    }
    ask_pages(j0 + batch);
    ask_keep(j0 + 2 * batch);
    // The loads have returned, and every wave's, before a row is overwritten.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      if (to[i] != nullptr) {
        *reinterpret_cast<u32x4_t*>(to[i] + codes + to_row[i] * (16 * blocks.d)) = data[i];
        to[i][scales + to_row[i]] = scale[i];
      }
  }
}

// ---- host ---------------------------------------------------------------------------

Rows4 rows_of(int64_t nodes, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim, int64_t page_stride,
              const int32_t* table, int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* cu,
              int64_t seqs) {
  return Rows4{static_cast<uint32_t>(nodes),
               static_cast<uint32_t>(kv_heads),
               static_cast<uint32_t>(dim / 32),
               static_cast<uint32_t>(pages),
               page_stride,
               Divisor(static_cast<uint32_t>(page)),
               Divisor(static_cast<uint32_t>(kv_heads * dim / 8)),
               Divisor(static_cast<uint32_t>(dim / 8)),
               table,
               table_stride,
               static_cast<uint32_t>(table_cols),
               lens,
               cu,
               static_cast<uint32_t>(seqs)};
}

// Sizes of a call over `nodes` rows; its threads' pieces of 8 elements count in 32 bits.
bool nodes_ok(int64_t nodes, int64_t kv_heads, int64_t dim, int64_t seqs) {
  return nodes >= 0 && nodes <= (1 << 24) && seqs >= 0 && seqs <= 65535 &&
         nodes * (kv_heads * dim / 8) <= INT32_MAX - 8 * kThreads * 4;
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int64_t spiral_cache4_page_bytes(int64_t page, int64_t kv_heads, int64_t dim) {
  if (!sizes4_ok(0, page, kv_heads, dim, int64_t(1) << 40)) return 0;
  return kv_heads * Block4{static_cast<uint32_t>(page), static_cast<uint32_t>(dim)}.bytes();
}

int spiral_cache4_store(int type, const void* new_k, const void* new_v, int64_t node_stride, int64_t head_stride,
                        int64_t nodes, void* k, void* v, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                        int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                        const int32_t* lens, const int32_t* cu, int64_t seqs, void* stream) {
  if (type != SPIRAL_TYPE_F32 && type != SPIRAL_TYPE_F16 && type != SPIRAL_TYPE_BF16) return SPIRAL_ERR_TYPE;
  if (!sizes4_ok(pages, page, kv_heads, dim, page_stride) || !table_ok(table_cols, table_stride) ||
      !nodes_ok(nodes, kv_heads, dim, seqs))
    return SPIRAL_ERR_SHAPE;
  const int64_t size = type == SPIRAL_TYPE_F32 ? 4 : 2;
  for (int64_t stride : {node_stride, head_stride}) {
    if (stride < 0 || stride > (int64_t(1) << 40)) return SPIRAL_ERR_SHAPE;
    if (stride * size % 16 != 0) return SPIRAL_ERR_ALIGN;
  }
  if (nodes == 0 || seqs == 0 || pages == 0) return SPIRAL_OK;
  if (new_k == nullptr || k == nullptr || (new_v == nullptr) != (v == nullptr) ||
      (table == nullptr && table_cols > 0) || lens == nullptr || cu == nullptr)
    return SPIRAL_ERR_NULL;
  if (!aligned16(new_k) || !aligned16(new_v) || !aligned16(k) || !aligned16(v) || !words_aligned({table, lens, cu}))
    return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const Rows4 a =
      rows_of(nodes, pages, page, kv_heads, dim, page_stride, table, table_stride, table_cols, lens, cu, seqs);
  const int64_t pieces = nodes * (kv_heads * dim / 8);
  const dim3 grid(static_cast<unsigned>(groups_of(pieces)), v != nullptr ? 2 : 1);
#define SPIRAL_STORE(T)                                                                                      \
  hipLaunchKernelGGL(store_kernel<T>, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream),             \
                     static_cast<const uint8_t*>(new_k), static_cast<const uint8_t*>(new_v), node_stride * size, \
                     head_stride * size, static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), a,              \
                     static_cast<uint32_t>(pieces))
  if (type == SPIRAL_TYPE_F32)
    SPIRAL_STORE(SPIRAL_TYPE_F32);
  else if (type == SPIRAL_TYPE_F16)
    SPIRAL_STORE(SPIRAL_TYPE_F16);
  else
    SPIRAL_STORE(SPIRAL_TYPE_BF16);
#undef SPIRAL_STORE
  return launch_status();
}

int spiral_cache4_load(int type, const void* cache, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                       int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                       const int32_t* lens, const int32_t* cu, int64_t seqs, int64_t nodes, void* out, void* stream) {
  if (type != SPIRAL_TYPE_F16 && type != SPIRAL_TYPE_BF16) return SPIRAL_ERR_TYPE;
  if (!sizes4_ok(pages, page, kv_heads, dim, page_stride) || !table_ok(table_cols, table_stride) ||
      !nodes_ok(nodes, kv_heads, dim, seqs))
    return SPIRAL_ERR_SHAPE;
  if (nodes == 0 || seqs == 0) return SPIRAL_OK;
  if ((cache == nullptr && pages > 0) || (table == nullptr && table_cols > 0) || lens == nullptr || cu == nullptr ||
      out == nullptr)
    return SPIRAL_ERR_NULL;
  if (!aligned16(cache) || !aligned16(out) || !words_aligned({table, lens, cu})) return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const Rows4 a =
      rows_of(nodes, pages, page, kv_heads, dim, page_stride, table, table_stride, table_cols, lens, cu, seqs);
  const int64_t pieces = nodes * (kv_heads * dim / 8);
  const dim3 grid(static_cast<unsigned>(groups_of(pieces)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (type == SPIRAL_TYPE_F16)
    hipLaunchKernelGGL(load_kernel<true>, grid, dim3(kThreads), 0, s, static_cast<const uint8_t*>(cache), a,
                       static_cast<u32x4_t*>(out), static_cast<uint32_t>(pieces));
  else
    hipLaunchKernelGGL(load_kernel<false>, grid, dim3(kThreads), 0, s, static_cast<const uint8_t*>(cache), a,
                       static_cast<u32x4_t*>(out), static_cast<uint32_t>(pieces));
  return launch_status();
}

int spiral_cache4_compact(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                          int64_t page, int64_t kv_heads, int64_t dim, const int32_t* table, int64_t table_stride,
                          int64_t table_cols, const int32_t* lens, int64_t seqs, const int32_t* keep,
                          int64_t keep_stride, int64_t keep_cols, const int32_t* kept, int32_t* new_lens,
                          void* stream) {
  int64_t a = 0, b = 0, c = 0;
  if (!sizes4_ok(pages, page, kv_heads, dim, page_stride) || layers < 0 || layers > 32767 || layer_stride < 0 ||
      layer_stride % 16 != 0 || __builtin_mul_overflow(layers, layer_stride, &a) ||
      __builtin_mul_overflow(pages, page_stride, &c) || __builtin_add_overflow(a, c, &b) || b > (INT64_MAX >> 1) ||
      seqs < 0 || seqs > 65535 ||
      !table_ok(table_cols, table_stride) || keep_cols < 0 || keep_cols > INT32_MAX / 2 || keep_stride < keep_cols ||
      keep_stride > INT32_MAX)
    return SPIRAL_ERR_SHAPE;
  if (seqs == 0) return SPIRAL_OK;
  if (lens == nullptr || kept == nullptr || (keep == nullptr && keep_cols > 0) ||
      (table == nullptr && table_cols > 0) || (k == nullptr && layers > 0 && pages > 0))
    return SPIRAL_ERR_NULL;
  if (!aligned16(k) || !aligned16(v) || !words_aligned({table, lens, keep, kept, new_lens})) return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const int64_t arrays = std::max<int64_t>(1, v != nullptr ? 2 * layers : layers), cols = kv_heads * (dim / 32);
  int log_cols = 6;
  while (log_cols > 2 && ((int64_t(1) << (log_cols - 1)) >= cols ||
                          ceil_div(cols, int64_t(1) << log_cols) * arrays * seqs < 4 * device_cu_count()))
    --log_cols;
  const dim3 grid(static_cast<unsigned>(ceil_div(cols, int64_t(1) << log_cols)), static_cast<unsigned>(seqs),
                  static_cast<unsigned>(arrays));
  hipLaunchKernelGGL(compact4_kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<uint8_t*>(k), static_cast<uint8_t*>(v),
                     static_cast<uint32_t>(std::max<int64_t>(layers, 1)), layer_stride,
                     static_cast<uint32_t>(layers > 0 ? pages : 0), page_stride, Divisor(static_cast<uint32_t>(page)),
                     static_cast<uint32_t>(kv_heads), Divisor(static_cast<uint32_t>(dim / 32)), table, table_stride,
                     static_cast<uint32_t>(table_cols), lens, keep, keep_stride, static_cast<uint32_t>(keep_cols), kept,
                     new_lens, static_cast<uint32_t>(log_cols));
  return launch_status();
}

}  // extern "C"

// Pages and rows of a paged key/value cache moved in place (spiral_cache.h): copies
// for forks, compaction of kept rows. Both are copies; HBM bounds the large ones, the
// launch and three dependent loads the small ones.
#include <algorithm>

#include "common.h"
#include "paged.h"
#include "spiral_cache.h"

namespace spiral {
namespace {

constexpr int kThreads = 256;

// ---- page copies ----------------------------------------------------------------

// Thread's pieces of 16 bytes: kPieces of the n * page16 pieces of one layer of k
// or v (blockIdx.y), kThreads apart, all loads before the stores. 16128 rows of 2 KiB
// (1.06 GB read and written): 187 us, 5.7 TB/s; stores through the caches 209.
constexpr int kPieces = 8;

__global__ void __launch_bounds__(kThreads)
    copy_pages_kernel(uint8_t* k, uint8_t* v, uint32_t layers, int64_t layer_stride, uint32_t pages,
                      int64_t page_stride, Divisor page16, const int32_t* __restrict__ src,
                      const int32_t* __restrict__ dst, uint32_t n, uint32_t pieces) {
  const uint32_t l = blockIdx.y < layers ? blockIdx.y : blockIdx.y - layers;
  uint8_t* base = (blockIdx.y < layers ? k : v) + l * layer_stride;
  const uint32_t p0 = blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  u32x4_t data[kPieces];
  uint32_t to[kPieces], off[kPieces];
  bool on[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const uint32_t p = min(p0 + i * kThreads, pieces - 1), pair = page16.quotient(p);
    const uint32_t from = src[pair];
    to[i] = dst[pair];
    on[i] = p0 + i * kThreads < pieces && from < pages && to[i] < pages;  // a negative id is past every page
    off[i] = p - pair * page16.d;
    data[i] = __builtin_nontemporal_load(
        reinterpret_cast<const u32x4_t*>(base + (from < pages ? from : 0u) * page_stride + off[i] * int64_t(16)));
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (on[i])
      __builtin_nontemporal_store(data[i],
                                  reinterpret_cast<u32x4_t*>(base + to[i] * page_stride + off[i] * int64_t(16)));
}

// ---- compaction -----------------------------------------------------------------

// keep ascends strictly, so keep[j] >= j and move j reads a row that no earlier move
// wrote: only the row that move j writes may be waiting to be read by an earlier
// move. A workgroup owns a column slice of `cols` 16-byte pieces of one sequence,
// layer and array (nobody else touches it) and takes the moves in order, kMoves *
// kThreads / cols at a time: all loads of a batch, a barrier, its stores.
// A move is three loads that depend on each other (keep, table, row). They are taken
// in step: with a batch's rows the table entries of the next and the keep of the one
// behind it are asked for. Narrow slices make workgroups enough for one layer of one
// sequence; where layers and sequences are many a slice is up to 1 KiB of a row.
constexpr int kMoves = 8;

__global__ void __launch_bounds__(kThreads)
    compact_kernel(uint8_t* k, uint8_t* v, uint32_t layers, int64_t layer_stride, uint32_t pages, int64_t page_stride,
                   Divisor page, uint32_t row16, const int32_t* __restrict__ table, int64_t table_stride,
                   uint32_t table_cols, const int32_t* __restrict__ lens, const int32_t* __restrict__ keep,
                   int64_t keep_stride, uint32_t keep_cols, const int32_t* __restrict__ kept,
                   int32_t* __restrict__ new_lens, uint32_t log_cols) {
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
  const int64_t row_bytes = row16 * int64_t(16);

  // Move j0 + i step + slot: keep's entry (negative: none), the positions of its rows
  // (negative where there is nothing to move) and their table entries.
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
      const bool on = from[i] >= 0 && from[i] != j && col < row16 && rows.in_table(src[i]) && rows.in_table(dst[i]);
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
    uint8_t* to[kMoves];
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      to[i] = nullptr;
      if (src[i] < 0 || src_page[i] >= pages || dst_page[i] >= pages) continue;  // a negative id is past every page
      to[i] = base + dst_page[i] * page_stride + rows.row(dst[i]) * row_bytes + col * 16;
      data[i] = *reinterpret_cast<const u32x4_t*>(base + src_page[i] * page_stride + rows.row(src[i]) * row_bytes +
                                                  col * 16);
    }
    ask_pages(j0 + batch);
    ask_keep(j0 + 2 * batch);
    // The loads have returned, and every wave's, before a row is overwritten.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      if (to[i] != nullptr) *reinterpret_cast<u32x4_t*>(to[i]) = data[i];
  }
}

bool bad_stride(int64_t v) { return v < 0 || v % 16 != 0; }

// Whether the last byte's offset of an array of layers and pages stays in 62 bits.
bool spans(int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride, int64_t page_bytes) {
  int64_t a = 0, b = 0, c = 0;
  return !__builtin_mul_overflow(layers, layer_stride, &a) && !__builtin_mul_overflow(pages, page_stride, &b) &&
         !__builtin_add_overflow(a, b, &c) && !__builtin_add_overflow(c, page_bytes, &c) && c < (INT64_MAX >> 1);
}

}  // namespace
}  // namespace spiral

using namespace spiral;

extern "C" {

int spiral_cache_copy_pages(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                            int64_t page_bytes, const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  if (layers < 0 || pages < 0 || n < 0 || page_bytes <= 0 || page_bytes % 16 != 0 || bad_stride(layer_stride) ||
      bad_stride(page_stride) || page_stride < page_bytes || layers > 32767 || pages > INT32_MAX ||
      page_bytes > INT32_MAX || !spans(layers, layer_stride, pages, page_stride, page_bytes))
    return SPIRAL_ERR_SHAPE;
  int64_t pieces = 0;
  if (__builtin_mul_overflow(n, page_bytes / 16, &pieces) || pieces > INT32_MAX - kThreads * kPieces)
    return SPIRAL_ERR_SHAPE;
  if (layers == 0 || n == 0 || pages == 0) return SPIRAL_OK;
  if (k == nullptr || src == nullptr || dst == nullptr) return SPIRAL_ERR_NULL;
  if (!aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(src) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(dst) & 3u) != 0)
    return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(pieces, kThreads * kPieces)),
                  static_cast<unsigned>(v != nullptr ? 2 * layers : layers));
  hipLaunchKernelGGL(copy_pages_kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), static_cast<uint32_t>(layers), layer_stride,
                     static_cast<uint32_t>(pages), page_stride, Divisor(static_cast<uint32_t>(page_bytes / 16)), src,
                     dst, static_cast<uint32_t>(n), static_cast<uint32_t>(pieces));
  return launch_status();
}

int spiral_cache_compact(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                         int64_t page, int64_t row_bytes, const int32_t* table, int64_t table_stride,
                         int64_t table_cols, const int32_t* lens, int64_t seqs, const int32_t* keep,
                         int64_t keep_stride, int64_t keep_cols, const int32_t* kept, int32_t* new_lens,
                         void* stream) {
  int64_t page_bytes = 0;
  if (layers < 0 || pages < 0 || seqs < 0 || page <= 0 || row_bytes <= 0 || row_bytes % 16 != 0 ||
      row_bytes > INT32_MAX || page > INT32_MAX || __builtin_mul_overflow(page, row_bytes, &page_bytes) ||
      bad_stride(layer_stride) || bad_stride(page_stride) || page_stride < page_bytes || layers > 32767 ||
      pages > INT32_MAX || seqs > 65535 || table_cols < 0 || table_cols > INT32_MAX || table_stride < table_cols ||
      table_stride > INT32_MAX || keep_cols < 0 || keep_cols > INT32_MAX / 2 || keep_stride < keep_cols ||
      keep_stride > INT32_MAX || !spans(layers, layer_stride, pages, page_stride, page_bytes))
    return SPIRAL_ERR_SHAPE;
  if (seqs == 0) return SPIRAL_OK;
  if (lens == nullptr || kept == nullptr || (keep == nullptr && keep_cols > 0) ||
      (table == nullptr && table_cols > 0) || (k == nullptr && layers > 0 && pages > 0))
    return SPIRAL_ERR_NULL;
  const uintptr_t words = reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lens) |
                          reinterpret_cast<uintptr_t>(keep) | reinterpret_cast<uintptr_t>(kept) |
                          reinterpret_cast<uintptr_t>(new_lens);
  if (!aligned16(k) || !aligned16(v) || (words & 3u) != 0) return SPIRAL_ERR_ALIGN;
  const int rc = require_device();
  if (rc != SPIRAL_OK) return rc;
  // Without layers or rows only the new lengths are written.
  const int64_t arrays = std::max<int64_t>(1, v != nullptr ? 2 * layers : layers), row16 = row_bytes / 16;
  int log_cols = 6;
  while (log_cols > 2 && ((int64_t(1) << (log_cols - 1)) >= row16 ||
                          ceil_div(row16, int64_t(1) << log_cols) * arrays * seqs < 4 * device_cu_count()))
    --log_cols;
  const dim3 grid(static_cast<unsigned>(ceil_div(row16, int64_t(1) << log_cols)), static_cast<unsigned>(seqs),
                  static_cast<unsigned>(arrays));
  hipLaunchKernelGGL(compact_kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), static_cast<uint32_t>(std::max<int64_t>(layers, 1)),
                     layer_stride, static_cast<uint32_t>(layers > 0 ? pages : 0), page_stride,
                     Divisor(static_cast<uint32_t>(page)), static_cast<uint32_t>(row16), table, table_stride,
                     static_cast<uint32_t>(table_cols), lens, keep, keep_stride, static_cast<uint32_t>(keep_cols), kept,
                     new_lens, static_cast<uint32_t>(log_cols));
  return launch_status();
}

}  // extern "C"

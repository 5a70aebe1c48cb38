/*
 * spiral_cache.h -- a paged key/value cache on one HIP device: attention of
 * drafted trees over it, page copies for forks, compaction of kept rows. No
 * counterpart in the reference, which stops at the quantized products
 * (README.md:11-14); llama.cpp keeps its cache in the backend's buffers.
 *
 * A cache is two arrays (keys and values) of `pages` pages of `page` rows; a row
 * holds kv_heads heads of dim elements (BF16 or F16). Row r of page p starts at
 * p * page_stride + r * row_stride, head h in it at h * head_stride, all in
 * elements, multiples of 8, dim elements contiguous; keys and values have the
 * same strides. A table of page ids ([seqs][table_cols] int32, rows of stride
 * table_stride) says where a sequence's rows lie: position i is row i % page of
 * page table[s][i / page]. A page id outside [0, pages), and a position past the
 * table, holds no row: attention does not see it, a move from or to it is left
 * out.
 *
 * All pointers are device memory. Functions return spiral_status codes
 * (spiral_quants.h), launch on `stream` and do not synchronize. What the host
 * cannot see (lengths, page ids, masks) is bounds-checked by the kernels.
 */
#ifndef SPIRAL_CACHE_H
#define SPIRAL_CACHE_H

#include <stdint.h>

#include "spiral_quants.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of one tree of drafted tokens per sequence over its cached rows.
 * Sequence s has lens[s] cached rows and the nodes cu[s] .. cu[s + 1] - 1
 * (cu: seqs + 1 int32, ascending), whose own rows lie behind the cached ones, node
 * i's at position lens[s] + i - cu[s]. Node i sees every cached row, and the row
 * of node cu[s] + j where bit j % 64 of mask[i][j / 64] is set (mask: [nodes]
 * [mask_words] 64-bit words; bits past them count as clear). With one node a
 * sequence and mask 1 this is plain decoding.
 *   out[i][h] = sum_r p_r V_r,  p = softmax over the visible rows r of
 *   scale * q[i][h] . K_r,  lse[i][h] = log sum exp of the same, natural;
 * scale > 0; query head h reads cached head h / (heads / kv_heads). A node that sees
 * no row gets zeros and lse = -infinity, one whose scores hold a NaN gets NaN. Rows
 * that a node does not see have no influence on it whatever they hold (NaN and
 * infinities included).
 *  q: type BF16 or F16, node and head strides in elements (multiples of 8), dim
 *     contiguous; out the same type, contiguous [nodes][heads][dim]; lse F32
 *     [nodes][heads], or NULL.
 *  dim: a multiple of 8 up to 256. max_len: about the longest lens[s] plus its
 *     tree, which only decides whether rows are split over workgroups; max_tree: at
 *     least the largest tree (nodes of a tree past it are left out).
 *  workspace: partial results of split rows, 16-byte aligned, of
 *     spiral_tree_attention_workspace_bytes() bytes (256 MiB at most); with
 *     less (or NULL) rows are split less, which is slower. Not shared by calls in
 *     flight at the same time.
 * Scores, softmax statistics and sums are fp32; p is rounded to the cache's type
 * in front of its product with V. Results do not depend on the order in which
 * workgroups run. nodes or seqs may be 0. */
int64_t spiral_tree_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs,
                                              int64_t max_len, int64_t max_tree);
int spiral_tree_attention(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                          int64_t heads, const void* k, const void* v, int64_t pages, int64_t page, int64_t kv_heads,
                          int64_t dim, int64_t page_stride, int64_t row_stride, int64_t head_stride,
                          const int32_t* table, int64_t table_stride, int64_t table_cols, const int32_t* lens,
                          const int32_t* cu, int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len,
                          int64_t max_tree, float scale, void* out, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* Copies page src[i] over page dst[i] (i < n) in every layer of the keys and the
 * values: layer l's page p is the page_bytes bytes at l * layer_stride + p *
 * page_stride (bytes; all multiples of 16). v may be NULL. The pages in dst must
 * be distinct and not in src; a pair with an id outside [0, pages) is left out. */
int spiral_cache_copy_pages(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                            int64_t page_bytes, const int32_t* src, const int32_t* dst, int64_t n, void* stream);

/* Moves the kept rows of every sequence together, in every layer of the keys and
 * the values: for j < kept[s] (clipped to 0 .. keep_cols), in this order, the row at position
 * lens[s] + keep[s][j] goes to position lens[s] + j (row_bytes bytes, row r of a
 * page at r * row_bytes; strides in bytes, all multiples of 16). keep[s] must
 * ascend strictly. new_lens[s] = lens[s] + kept[s] as clipped above (NULL: not
 * written; never lens itself, which other workgroups still read). v may be NULL. */
int spiral_cache_compact(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                         int64_t page, int64_t row_bytes, const int32_t* table, int64_t table_stride,
                         int64_t table_cols, const int32_t* lens, int64_t seqs, const int32_t* keep,
                         int64_t keep_stride, int64_t keep_cols, const int32_t* kept, int32_t* new_lens, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SPIRAL_CACHE_H */

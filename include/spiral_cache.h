/*
 * spiral_cache.h -- a paged key/value cache on one HIP device, in 16 bits or in 4:
 * attention of drafted trees over it, verification of the drafts, page copies for
 * forks, compaction of kept rows, eviction by accumulated attention weight. No
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

/* ---- a cache in 4 bits -----------------------------------------------------------
 *
 * Keys (and values) are an array of `pages` pages of MXFP4 rows, page p at p *
 * page_stride bytes (a multiple of 16). A page holds `page` rows, a multiple of 16, and
 * is kv_heads blocks one behind the other, each
 *   codes  [page][dim / 2]: byte j of a row has element 2j in its low and 2j + 1 in its
 *          high half, E2M1 as in SPIRAL_TYPE_MXFP4,
 *   scales [dim / 32][page]: the E8M0 byte of 32 elements of a row;
 * dim is a multiple of 32 up to 256. spiral_cache4_page_bytes() is a page's size (0 for
 * sizes that are not taken). A page is copied by spiral_cache_copy_pages as any other. */
int64_t spiral_cache4_page_bytes(int64_t page, int64_t kv_heads, int64_t dim);

/* Rows of nodes to the cache, quantized as spiral_mxfp4_quantize does: node i of
 * cu[s] .. cu[s + 1] - 1 (cu as above) goes to position lens[s] + i - cu[s] of sequence s,
 * where spiral_tree_attention looks for it. new_k, new_v: type F32, F16 or BF16, node and
 * head strides in elements (16-byte aligned rows: multiples of 8, 4 for F32), dim
 * contiguous, both with the same strides. new_v and v may be NULL together. A block with a
 * NaN or an infinity becomes NaN. Other rows of the pages keep their bytes; a row without
 * a page is left out. No two sequences may write the same row. */
int spiral_cache4_store(int type, const void* new_k, const void* new_v, int64_t node_stride, int64_t head_stride,
                        int64_t nodes, void* k, void* v, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                        int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                        const int32_t* lens, const int32_t* cu, int64_t seqs, void* stream);

/* The rows that spiral_cache4_store would write, as the values they hold: out [nodes]
 * [kv_heads][dim] contiguous, BF16 (exact but for overflow to infinity) or F16 (rounded).
 * Zeros for rows without a page, and for nodes of no sequence; without any sequence (seqs 0)
 * nothing is written. */
int spiral_cache4_load(int type, const void* cache, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                       int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                       const int32_t* lens, const int32_t* cu, int64_t seqs, int64_t nodes, void* out, void* stream);

/* spiral_tree_attention over a cache in 4 bits; table_cols * page is below 2^28. Codes are
 * taken as the values they stand for in q's type: exactly in BF16 (past its largest an
 * infinity); in F16 values past 65504 are infinities and those below 2^-24 lose bits, which of
 * rows stored from F16 only blocks do whose largest value is below 2^-20. */
int64_t spiral_cache4_tree_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs,
                                                     int64_t max_len, int64_t max_tree);
int spiral_cache4_tree_attention(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                                 int64_t heads, const void* k, const void* v, int64_t pages, int64_t page,
                                 int64_t kv_heads, int64_t dim, int64_t page_stride, const int32_t* table,
                                 int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* cu,
                                 int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len,
                                 int64_t max_tree, float scale, void* out, float* lse, void* workspace,
                                 int64_t workspace_bytes, void* stream);

/* spiral_cache_compact of a cache in 4 bits. */
int spiral_cache4_compact(void* k, void* v, int64_t layers, int64_t layer_stride, int64_t pages, int64_t page_stride,
                          int64_t page, int64_t kv_heads, int64_t dim, const int32_t* table, int64_t table_stride,
                          int64_t table_cols, const int32_t* lens, int64_t seqs, const int32_t* keep,
                          int64_t keep_stride, int64_t keep_cols, const int32_t* kept, int32_t* new_lens,
                          void* stream);

/* ---- verification of drafted tokens ------------------------------------------------
 *
 * Which nodes of a sequence's tree the target model accepts, and the token drawn behind
 * them, from given random numbers. logits: [nodes][vocab], row i the target's behind node
 * i; node cu[s] of a tree is the last known token, the others are drafted. With p(x | i)
 * the softmax of row i over temperature[s] (0: all on the first of the largest logits),
 * the walk starts at node cu[s] and, at node i:
 *  - trees of given tokens (draft NULL): the nodes j with parents[j] = i - cu[s] (an index
 *    in the tree, below j's own; parents NULL: the node in front) are tried in order. With
 *    T the tokens turned down at i, j is taken if accept[j] * (1 - sum over T of p) <
 *    p(tokens[j] | i) and its token is not in T; else its token joins T. Behind the last,
 *    a token is drawn from p(. | i) without T.
 *  - chains drawn from a draft model (draft: its logits, as above, row i behind node i; its
 *    q(. | i) with the same temperature): node i + 1 is taken if accept[i + 1] * q(token)
 *    < p(token); else a token is drawn from max(p - q, 0), and behind the last node from p.
 * A node that is taken is the next i. A draw is the first token x with sum over y <= x of w(y)
 * > sample[s] * (sum of w), w what is drawn from; where nothing is left, w is p. Tokens
 * outside [0, vocab) are turned down. A row of the target's that the walk comes to and that
 * holds a NaN, +infinity, or no number ends the walk, and the token is -1; such a row of the
 * draft's turns its token down, and the token is drawn from p.
 *  keep: [seqs][max_tree], row stride keep_stride: the path's nodes as indices in the tree, the
 *   first of them 0, -1 behind: spiral_cache_compact's keep. kept: [seqs], how many (0 for an
 *   empty tree). out: [seqs][max_tree], stride keep_stride: the tokens of keep[1 ..], then
 *   the drawn one: kept[s] tokens, -1 behind.
 *  logits, draft: F32, F16 or BF16, the same type, row strides in elements, at least vocab.
 *  nodes: at most 32767 in all, vocab: at most 2^24, seqs: 65535.
 *  accept: [nodes], sample: [seqs], in [0, 1) F32. temperature: [seqs] F32, NULL: 1.
 *  max_tree: at least the largest tree (nodes past it are left out), at most 1024; 0: nothing
 *   is written.
 *  workspace: 16-byte aligned, of spiral_draft_verify_workspace_bytes() bytes (0 for sizes that
 *   are not taken); required, and used by one call at a time. keep, kept and out do not overlap.
 * Probabilities, sums and comparisons are in 64 bits: a draw turns on the last bits of a sum
 * over the vocabulary. */
int64_t spiral_draft_verify_workspace_bytes(int64_t nodes, int64_t seqs, int64_t vocab, int has_draft);
int spiral_draft_verify(int type, const void* logits, int64_t logits_stride, const void* draft, int64_t draft_stride,
                        int64_t nodes, int64_t vocab, const int32_t* tokens, const int32_t* parents, const int32_t* cu,
                        int64_t seqs, int64_t max_tree, const float* accept, const float* sample,
                        const float* temperature, int32_t* keep, int32_t* kept, int32_t* out, int64_t keep_stride,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* ---- eviction by accumulated attention weight ----------------------------------------
 *
 * Adds to mass[s][r] (F32, row stride mass_stride, mass_cols columns) the attention weight that
 * position r of sequence s gets from its tree's nodes, summed over nodes and heads:
 *   sum over i, h of counted[i] * exp(scale q[i][h] . K_r - lse[i][h]),
 * for the rows that node i sees (spiral_tree_attention, whose lse this takes; a node whose
 * lse is -infinity sees none). counted: [nodes] F32, NULL: all 1; a node at 0 is left
 * out whatever it holds. Positions past mass_cols, and those without a page, are left out.
 * max_len: about the longest sequence with its tree, which only decides the grid. Sums are
 * fp32, in an order that does not depend on how workgroups run. */
int spiral_cache_row_weights(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                             int64_t heads, const void* k, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                             int64_t page_stride, int64_t row_stride, int64_t head_stride, const int32_t* table,
                             int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* cu,
                             int64_t seqs, const uint64_t* mask, int64_t mask_words, int64_t max_len, int64_t max_tree,
                             float scale, const float* lse, const float* counted, float* mass, int64_t mass_stride,
                             int64_t mass_cols, void* stream);
int spiral_cache4_row_weights(int type, const void* q, int64_t q_node_stride, int64_t q_head_stride, int64_t nodes,
                              int64_t heads, const void* k, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                              int64_t page_stride, const int32_t* table, int64_t table_stride, int64_t table_cols,
                              const int32_t* lens, const int32_t* cu, int64_t seqs, const uint64_t* mask,
                              int64_t mask_words, int64_t max_len, int64_t max_tree, float scale, const float* lse,
                              const float* counted, float* mass, int64_t mass_stride, int64_t mass_cols, void* stream);

/* The rows of every sequence that stay, at most `budget`: all of them where lens[s] <=
 * budget; else the first `sinks`, the last `recent`, and of the others those of the
 * largest mass[s][r] (a NaN is above all numbers, -0 is +0), of equal ones the first. lens[s]
 * counts as at most mass_cols. keep: [seqs][budget], row stride keep_stride: their
 * positions, ascending, -1 behind; kept: [seqs], how many: what spiral_cache_compact takes
 * for lens of zeros. new_mass ([seqs][mass_cols], stride new_stride, apart from mass; NULL:
 * not written): the masses of the rows that stay, in their new places, zeros behind.
 * sinks + recent <= budget. workspace: 16-byte aligned, used by one call at a time, of
 * spiral_cache_evict_workspace_bytes() bytes, which is 0 where none is used; without it a few long
 * sequences take longer, with the same results. From 983041 columns on none is used, and a
 * sequence takes 1.4 ms a million rows (81 us at 983040). */
int64_t spiral_cache_evict_workspace_bytes(int64_t mass_cols, int64_t seqs);
int spiral_cache_evict(const float* mass, int64_t mass_stride, int64_t mass_cols, const int32_t* lens, int64_t seqs,
                       int64_t budget, int64_t sinks, int64_t recent, int32_t* keep, int64_t keep_stride,
                       int32_t* kept, float* new_mass, int64_t new_stride, void* workspace, int64_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SPIRAL_CACHE_H */

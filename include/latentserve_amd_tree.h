/*
 * latentserve_amd — C ABI of drafted decoding over a bounded fp16 cache in
 * liblatentserve_hip.so: attention of a tree of drafted tokens, the accepted
 * path, weight sums of the cached tokens, eviction by them.
 *
 * The conventions are latentserve_amd.h's: device pointers, sizes and strides,
 * no framework types; calls only enqueue work on `stream` (NULL: the default
 * stream of the current device), allocate nothing, read nothing back and can be
 * captured in a HIP graph; 0 on success, else LS_ERR_* with a message from
 * ls_last_error().  This part of the ABI has a version of its own.
 *
 * Pools are fp16 [num_blocks, 16, H, 128] with pool_strides[3] = (block, token,
 * head) in elements, the same for K and V; token t of a sequence is row t % 16 of
 * block block_tables[b, t / 16].  Blocks outside the pool are skipped, and tokens past
 * the table's width.  Sums of no rows or of no tokens may be null.  Rows of 128 values
 * start on 16 bytes.  Lengths, counts and tables are read on the device; none of them makes
 * a call read or write out of range.
 */
#ifndef LATENTSERVE_AMD_TREE_H
#define LATENTSERVE_AMD_TREE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header (bumped on any change of a declaration, or of what a
 * caller must provide). */
int ls_tree_abi_version(void);

/* masks [batch, nodes, ceil(nodes / 64)] int64: node i's ancestors and itself (bit
 * j % 64 of word j / 64: node j), and depths [batch, nodes] int32 (0: no parent),
 * from parents [batch, nodes] int32.  A parent comes before its children: any other
 * number, like -1, is none.  nodes in 1..256. */
int ls_tree_masks(const int32_t* parents, int64_t* masks, int32_t* depths, int batch, int nodes,
                  void* stream);

/* Bytes of `workspace` (16-byte aligned, any contents) of a tree attention of these
 * sizes.  max_seq_len: the longest sequence expected (0: the table's width); it
 * only sizes the launch.  Calls that may run at the same time need their own. */
size_t ls_tree_attention_workspace_bytes(int batch, int kv_heads, int nodes, int n_rep,
                                         int max_pages, int max_seq_len);

/* Attention of each sequence's last `nodes` tokens: q [batch, nodes, kv_heads,
 * n_rep, 128] fp16, q_strides[4] = (b, n, h, r); out the same shape, out_strides[4];
 * nodes in 1..256, n_rep in 1..16.  seq_lens counts the nodes.  Node i sees the
 * tokens before the nodes and the nodes of masks[b, i] (null: nodes 0..i).  counts
 * [batch] (null: all): a sequence's nodes from counts[b] on, which nobody
 * sees, give zeros.  A sequence of fewer than `nodes` tokens has no context and so
 * many nodes.  lse [batch, nodes, kv_heads, n_rep] fp32 (or null): log of the sum of
 * the exponentials (natural), -inf where a row sees nothing, whose output is zeros. */
int ls_tree_attention(const void* q, const int64_t* q_strides, const void* k_pool,
                      const void* v_pool, const int64_t* pool_strides, int64_t num_blocks,
                      const int32_t* block_tables, int64_t bt_stride, int max_pages,
                      const int32_t* seq_lens, const int64_t* masks, const int32_t* counts,
                      void* out, const int64_t* out_strides, float* lse, void* workspace,
                      size_t workspace_bytes, int batch, int kv_heads, int nodes, int n_rep,
                      int head_dim, int page, int max_seq_len, float softmax_scale, void* stream);

/* Decode attention (q [batch, kv_heads, n_rep, 128], q_strides[3], out alike) that also
 * adds the attention weight each cached token got, summed over a KV head's rows:
 * sums[row, h, t] += ..., fp32, sum_strides[2] = (row, h), unit stride over
 * tokens, positions below sum_len; sequence b's row is sum_rows[b] (null: b; rows
 * outside [0, num_sum_rows): nothing is added).  Rows are distinct.  The workspace
 * holds the scores: 4 bytes for each of batch x kv_heads x n_rep rows and each token
 * of the tables' width, whatever the lengths are. */
size_t ls_decode_weights_workspace_bytes(int batch, int kv_heads, int n_rep, int max_pages,
                                         int max_seq_len);
int ls_paged_decode_weights(const void* q, const int64_t* q_strides, const void* k_pool,
                            const void* v_pool, const int64_t* pool_strides, int64_t num_blocks,
                            const int32_t* block_tables, int64_t bt_stride, int max_pages,
                            const int32_t* seq_lens, void* out, const int64_t* out_strides,
                            float* sums, const int64_t* sum_strides, int64_t sum_len,
                            const int32_t* sum_rows, int num_sum_rows, void* workspace,
                            size_t workspace_bytes, int batch, int kv_heads, int n_rep,
                            int head_dim, int page, int max_seq_len, float softmax_scale,
                            void* stream);

/* The same sums for the tokens of accepted paths, after the attention: q and lse
 * as ls_tree_attention's (lse contiguous); path [batch, path_len] int32 the
 * nodes in order (null: nodes 0, 1, ...; then path_len is nodes), lengths [batch] how
 * many of them count (null: path_len), whose K are the sequence's last lengths[b]
 * tokens; the i-th sees the tokens up to its own.  Nodes outside [0, nodes) add
 * nothing. */
int ls_add_weights(const void* q, const int64_t* q_strides, const float* lse, const void* k_pool,
                   const int64_t* pool_strides, int64_t num_blocks, const int32_t* block_tables,
                   int64_t bt_stride, int max_pages, const int32_t* seq_lens, float* sums,
                   const int64_t* sum_strides, int64_t sum_len, const int32_t* sum_rows,
                   int num_sum_rows, const int32_t* path, const int32_t* lengths, int batch,
                   int kv_heads, int nodes, int path_len, int n_rep, int head_dim, int page,
                   int max_seq_len, float softmax_scale, void* stream);

/* The path from node 0 by the first child whose token is its parent's choice: tokens and
 * choices [batch, nodes] int64, parents as ls_tree_masks, counts as ls_tree_attention.
 * path [batch, nodes] int32 (-1 behind its end), lengths [batch] int32 (0: no
 * nodes), next_tokens [batch] int64 (the last one's choice; -1: no nodes).  Then the
 * rows of the path's nodes, the sequences' last `nodes` tokens, become the first of them in
 * every pool: HOST arrays k_pools, v_pools[num_pools] of device pointers with one
 * pool_strides[3]. */
int ls_accept_tokens(const int64_t* tokens, const int32_t* parents, const int64_t* choices,
                     const int32_t* counts, int32_t* path, int32_t* lengths,
                     int64_t* next_tokens, void* const* k_pools, void* const* v_pools,
                     int num_pools, const int64_t* pool_strides, int64_t num_blocks,
                     const int32_t* block_tables, int64_t bt_stride, int max_pages,
                     const int32_t* seq_lens, int batch, int kv_heads, int nodes, int head_dim,
                     int page, void* stream);

/* Of the first seq_lens[b] positions of each row sums [layers, batch, kv_heads, .]
 * (fp32, sum_strides[3] = (layer, b, h)) the min(length, budget) to keep, ascending: the
 * first `sinks`, the last `recent`, and the largest sums (a NaN before all numbers;
 * equal ones: the lower position).  keep [layers, batch, kv_heads, budget] int32 (-1 behind
 * the last), kept (fp32, the same shape; 0 behind the last): their sums.  sinks +
 * recent <= budget.  Positions past sum_len (at most 2^30) count as none. */
int ls_select_tokens(const float* sums, const int64_t* sum_strides, int64_t sum_len,
                     const int32_t* seq_lens, int32_t* keep, float* kept, int layers, int batch,
                     int kv_heads, int budget, int sinks, int recent, void* stream);

/* Rows keep[l, b, h, j] of each sequence become its rows j, j < min(seq_lens[b],
 * budget), in every layer's K and V: keep as ls_select_tokens writes it (ascending;
 * a negative entry moves nothing). */
int ls_move_tokens(void* const* k_pools, void* const* v_pools, int layers,
                   const int64_t* pool_strides, int64_t num_blocks, const int32_t* block_tables,
                   int64_t bt_stride, int max_pages, const int32_t* seq_lens,
                   const int32_t* keep, int batch, int kv_heads, int budget, int head_dim,
                   int page, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LATENTSERVE_AMD_TREE_H */

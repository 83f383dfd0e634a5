/*
 * latentserve_amd — C ABI of the operators of branching generation in
 * liblatentserve_hip.so: the 4-bit paged cache (write, read, decode
 * attention), page copies, token log probabilities.
 *
 * The conventions are latentserve_amd.h's: device pointers, sizes and strides,
 * no framework types; calls only enqueue work on `stream` (NULL: the default
 * stream of the current device), allocate nothing, read nothing back and can be
 * captured in a HIP graph; 0 on success, else LS_ERR_* with a message from
 * ls_last_error().  This part of the ABI has a version of its own, so the
 * entry points of latentserve_amd.h stay at theirs.
 *
 * 4-bit pools: nb pages of 16 tokens, H KV heads, 128 channels.  Per (token,
 * head), each group of 32 adjacent channels has a minimum m and a step
 * s = fp16((max - m) / 15) (difference and quotient in fp32; the next smaller
 * fp16 where m + 15 s would round to infinity), fp16 both; a channel's code is the whole number nearest to (x - m) / s, ties to even, in
 * 0..15 (0 where s is 0), and stands for fp16(m + s * code), rounded once.
 * Values are finite (a group with an infinity or a NaN has no finite entries).
 *   k_codes   uint8 [nb, H, 16, 64]     a token's row: 16 words of 8 codes,
 *                                       word 4 g + j: channels 32 j + 8 g + (0..7)
 *   k_affine  fp16  [nb, H, 16, 4, 2]   (s, m) by token and group
 *   v_codes   uint8 [nb, H, 16, 16, 4]  word (o, t): channels 8 o + (0..7), token t
 *   v_affine  fp16  [nb, H, 4, 4, 2, 4] by group and token quad: s of the quad's
 *                                       four tokens, then their m
 * Code i of a word is its bits 4 i .. 4 i + 3.  A page's heads are adjacent (as
 * the shapes say); from page to page a pool may have any stride that is a
 * multiple of 16 bytes: page_strides[4], in bytes, of k_codes, k_affine,
 * v_codes, v_affine.  Pools, like k, v, q and out rows, start on 16 bytes.
 */
#ifndef LATENTSERVE_AMD_SERVING_H
#define LATENTSERVE_AMD_SERVING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header (bumped on any change of a declaration, or of what a
 * caller must provide). */
int ls_serving_abi_version(void);

/* New tokens' K and V, [batch, kv_heads, tokens, 128] fp16 with k_strides[3] /
 * v_strides[3] = (b, h, t) in elements, quantized into flat slots [batch *
 * tokens] int64 (block * 16 + offset; outside the pool: not written).  Slots
 * are distinct; of two tokens with one slot, either's codes may end up there.
 * Other tokens of a page are left as they are.  A group that holds a NaN or an
 * infinity reads back as NaN. */
int ls_int4_write(const void* k, const int64_t* k_strides, const void* v,
                  const int64_t* v_strides, const int64_t* slots, void* k_codes, void* k_affine,
                  void* v_codes, void* v_affine, const int64_t* page_strides, int64_t num_blocks,
                  int batch, int kv_heads, int tokens, int head_dim, int page, void* stream);

/* The first `length` positions of each sequence as values: k_out, v_out
 * [batch, length, kv_heads, 128] fp16, contiguous; zeros at positions past the
 * sequence, past the table and in blocks outside the pool. */
int ls_int4_read(const void* k_codes, const void* k_affine, const void* v_codes,
                 const void* v_affine, const int64_t* page_strides, int64_t num_blocks,
                 const int32_t* block_tables, int64_t bt_stride, int max_pages,
                 const int32_t* seq_lens, void* k_out, void* v_out, int batch, int kv_heads,
                 int head_dim, int page, int length, void* stream);

/* Workgroups a KV head that a decode of these sizes is launched with
 * (max_seq_len: the longest sequence expected, 0 for the table's width; longer
 * ones are still attended whole). */
int ls_int4_decode_groups(int batch, int kv_heads, int max_pages, int max_seq_len);

/* Bytes of `workspace` (16-byte aligned, any contents) and int32 elements of
 * `counters` (zero before the first call, left zero by every call) that a decode
 * with `groups` takes.  Calls that may run at the same time need their own. */
size_t ls_int4_decode_workspace_bytes(int groups, int kv_heads, int n_rep);
size_t ls_int4_decode_counter_ints(int groups, int kv_heads);

/* Decode attention over 4-bit pools: q [batch, kv_heads, n_rep, 128] fp16,
 * q_strides[3] = (b, h, r); out the same shape, out_strides[3]; n_rep in
 * 1..16.  Sequences of no tokens give zeros; blocks outside the pool are
 * skipped.  batch * (max_pages + 16) + groups < 2^31. */
int ls_paged_decode_int4(const void* q, const int64_t* q_strides, const void* k_codes,
                         const void* k_affine, const void* v_codes, const void* v_affine,
                         const int64_t* page_strides, int64_t num_blocks,
                         const int32_t* block_tables, int64_t bt_stride, int max_pages,
                         const int32_t* seq_lens, void* out, const int64_t* out_strides,
                         float* workspace, size_t workspace_bytes, int32_t* counters, int batch,
                         int kv_heads, int n_rep, int head_dim, int page, int groups,
                         float softmax_scale, void* stream);

/* Page dst[i] of every tensor becomes its page src[i], i < pairs.  HOST arrays:
 * tensors[num_tensors] device base pointers, page_strides and page_bytes
 * (bytes from page to page, and of one page), src and dst page numbers, all
 * in [0, num_pages).  dst holds no page twice and none of src's (refused). */
int ls_page_copy(void* const* tensors, const int64_t* page_strides, const int64_t* page_bytes,
                 int num_tensors, int64_t num_pages, const int32_t* src, const int32_t* dst,
                 int pairs, void* stream);

/* Bytes of `workspace` (16-byte aligned, any contents) and int32 elements of
 * `counters` (zero before the first call, left zero) of a log-probability call;
 * 0 where none is needed. */
size_t ls_token_logprobs_workspace_bytes(int rows, int n, int top);
size_t ls_token_logprobs_counter_ints(int rows, int n, int top);

/* Rows of n logits (fp16: elem_bytes 2, fp32: 4; row stride x_stride in
 * elements, unit stride inside): logprob[r] = log softmax(x_r)[tokens[r]]
 * (0 for a token outside [0, n): padding), entropy[r] = -sum p log p, both
 * fp32, and the `top` (0..32, at most n) largest: their log probabilities
 * top_val [rows, top] fp32 and numbers top_id [rows, top] int64, largest
 * first, equal logits by the lower number.  Logits of -inf have probability
 * 0; a row of nothing else gives -inf, entropy 0.  A NaN or +inf makes its
 * row's results NaN (NaN ranks first). */
int ls_token_logprobs(const void* x, int64_t x_stride, int elem_bytes, const int64_t* tokens,
                      int64_t token_stride, float* logprob, float* entropy, float* top_val,
                      int64_t* top_id, void* workspace, size_t workspace_bytes, int32_t* counters,
                      int rows, int n, int top, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LATENTSERVE_AMD_SERVING_H */

// C ABI of drafted decoding over a bounded cache: argument checks, then launches on the
// caller's stream.  Declared in include/latentserve_amd_tree.h.

#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <cmath>

#include "../../include/latentserve_amd.h"
#include "../../include/latentserve_amd_tree.h"
#include "ls_common.h"
#include "ls_tree.h"

namespace ls {
int abi_fail(int code, const char* message);      // ls_abi.hip: sets ls_last_error()
}

namespace {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return ls::abi_fail(code, buf);
}

int hip_status(hipError_t e, const char* what) {
    if (e != hipSuccess) return fail(LS_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    return LS_OK;
}

bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }

bool rows_aligned(const void* p, const int64_t* st, int count, int64_t elem) {
    if (!aligned(p, 16)) return false;
    for (int i = 0; i < count; ++i)
        if ((st[i] * elem) % 16 != 0) return false;
    return true;
}

int check_batch(int batch, int kv_heads) {
    if (batch < 0 || batch > 65535) return fail(LS_ERR_INVALID, "batch must be in [0, 65535], got %d", batch);
    if (kv_heads < 1 || kv_heads > 65535)
        return fail(LS_ERR_INVALID, "kv_heads must be in [1, 65535], got %d", kv_heads);
    return LS_OK;
}

int check_pool(const int64_t* strides, int64_t num_blocks, int head_dim, int page) {
    if (!strides) return fail(LS_ERR_INVALID, "null pointer argument");
    if (head_dim != ls::HEAD_DIM) return fail(LS_ERR_INVALID, "head_dim must be 128, got %d", head_dim);
    if (page != ls::PAGE) return fail(LS_ERR_INVALID, "page (block_size) must be 16, got %d", page);
    if (num_blocks < 1 || num_blocks > (1LL << 31) - 1)
        return fail(LS_ERR_INVALID, "num_blocks must be in [1, 2^31)");
    for (int i = 0; i < 3; ++i)
        if (strides[i] < 0 || strides[i] % 8 != 0)
            return fail(LS_ERR_INVALID, "pool rows must start on 16 bytes and not run backwards");
    // (a row's place in its page is a 32-bit number of bytes)
    if (strides[1] > 1 << 24) return fail(LS_ERR_INVALID, "a pool's token stride must be at most 2^24");
    return LS_OK;
}

int check_tables(const int32_t* block_tables, int64_t bt_stride, int max_pages,
                 const int32_t* seq_lens) {
    if (!block_tables || !seq_lens) return fail(LS_ERR_INVALID, "null pointer argument");
    if (max_pages < 1 || max_pages > (1 << 24))
        return fail(LS_ERR_INVALID, "max_pages (block-table width) must be in [1, 2^24]");
    if (bt_stride < 0) return fail(LS_ERR_INVALID, "block-table rows must not run backwards");
    return LS_OK;
}

int check_tree(int nodes, int n_rep) {
    if (nodes < 1 || nodes > ls::TREE_MAX_NODES)
        return fail(LS_ERR_INVALID, "nodes must be in [1, %d], got %d", ls::TREE_MAX_NODES, nodes);
    if (n_rep < 1 || n_rep > ls::MAX_NREP)
        return fail(LS_ERR_INVALID, "n_rep must be in [1, 16], got %d", n_rep);
    return LS_OK;
}

int check_sums(const float* sums, const int64_t* strides, int64_t sum_len, int num_sum_rows) {
    // (a tensor of nothing has no address)
    if (!strides || (!sums && sum_len > 0 && num_sum_rows > 0))
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (!aligned(sums, 4)) return fail(LS_ERR_INVALID, "sums must be 4-byte aligned");
    if (sum_len < 0 || num_sum_rows < 0 || strides[0] < 0 || strides[1] < 0)
        return fail(LS_ERR_INVALID, "bad sum_len, num_sum_rows or strides of the sums");
    return LS_OK;
}

int check_scale(float scale) {
    if (!std::isfinite(scale) || scale <= 0.f)
        return fail(LS_ERR_INVALID, "softmax_scale must be finite and above 0");
    return LS_OK;
}

int64_t keys_bound(int max_pages, int max_seq_len) {
    const int64_t keys = (int64_t)max_pages * ls::PAGE;
    return max_seq_len > 0 ? std::min<int64_t>(keys, max_seq_len) : keys;
}

// A launch's places (steps of all units) are 32-bit numbers; a step is 64 keys at least.
bool too_large(int batch, int kv_heads, int max_pages) {
    return (int64_t)batch * kv_heads * ((int64_t)max_pages / 4 + 2 + ls::TREE_EXTRA) >= (1LL << 31) ||
           (int64_t)batch * kv_heads >= (1LL << 22);
}

// Before the records: where the units lie in the groups.
size_t units_bytes(int batch, int kv_heads) {
    return (((size_t)batch * kv_heads + ls::TREE_CUS) * sizeof(int2) + 255) & ~(size_t)255;
}
void set_units(ls::TreeParams& a, void* workspace, int batch, int kv_heads) {
    a.split = (int2*)workspace;
    a.info = a.split + ls::TREE_CUS;
    a.work = (float*)((char*)workspace + units_bytes(batch, kv_heads));
}

int64_t score_len(int max_pages) { return ((int64_t)max_pages * ls::PAGE + 31) / 32 * 32; }

void set_q(ls::TreeParams& a, const void* q, const int64_t* st, void* out, const int64_t* so) {
    a.q = (const _Float16*)q;
    a.sq_b = st[0];
    a.sq_n = st[1];
    a.sq_h = st[2];
    a.sq_r = st[3];
    a.out = (_Float16*)out;
    a.so_b = so[0];
    a.so_n = so[1];
    a.so_h = so[2];
    a.so_r = so[3];
}

template <class P>
void set_pool(P& a, const int64_t* strides, int64_t num_blocks, const int32_t* tables,
              int64_t bt_stride, int max_pages, const int32_t* lens) {
    a.sp_b = 2 * strides[0];
    a.sp_t = 2 * strides[1];
    a.sp_h = 2 * strides[2];
    a.num_blocks = (int)num_blocks;
    a.tables = tables;
    a.st_b = bt_stride;
    a.max_pages = max_pages;
    a.lens = lens;
}

}  // namespace

extern "C" {

int ls_tree_abi_version(void) { return 1; }

int ls_tree_masks(const int32_t* parents, int64_t* masks, int32_t* depths, int batch, int nodes,
                  void* stream) {
    if (int rc = check_batch(batch, 1)) return rc;
    if (int rc = check_tree(nodes, 1)) return rc;
    if (batch == 0) return LS_OK;
    if (!parents || !masks || !depths) return fail(LS_ERR_INVALID, "null pointer argument");
    return hip_status(ls::launch_tree_masks(parents, (uint64_t*)masks, depths, batch, nodes,
                                            (hipStream_t)stream), "ls_tree_masks");
}

size_t ls_tree_attention_workspace_bytes(int batch, int kv_heads, int nodes, int n_rep,
                                         int max_pages, int max_seq_len) {
    if (batch < 1 || kv_heads < 1 || nodes < 1 || nodes > ls::TREE_MAX_NODES || n_rep < 1 ||
        n_rep > ls::MAX_NREP || max_pages < 1)
        return 0;
    return units_bytes(batch, kv_heads) +
           ls::tree_record_bytes(ls::tree_shape(batch, kv_heads, nodes * n_rep,
                                                keys_bound(max_pages, max_seq_len)));
}

int ls_tree_attention(const void* q, const int64_t* q_strides, const void* k_pool,
                      const void* v_pool, const int64_t* pool_strides, int64_t num_blocks,
                      const int32_t* block_tables, int64_t bt_stride, int max_pages,
                      const int32_t* seq_lens, const int64_t* masks, const int32_t* counts,
                      void* out, const int64_t* out_strides, float* lse, void* workspace,
                      size_t workspace_bytes, int batch, int kv_heads, int nodes, int n_rep,
                      int head_dim, int page, int max_seq_len, float softmax_scale, void* stream) {
    if (!q || !q_strides || !k_pool || !v_pool || !out || !out_strides || !workspace)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (int rc = check_pool(pool_strides, num_blocks, head_dim, page)) return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens)) return rc;
    if (int rc = check_tree(nodes, n_rep)) return rc;
    if (int rc = check_scale(softmax_scale)) return rc;
    if (too_large(batch, kv_heads, max_pages))
        return fail(LS_ERR_INVALID, "batch x kv_heads x max_pages too large for one call");
    if (!rows_aligned(q, q_strides, 4, 2) || !rows_aligned(out, out_strides, 4, 2) ||
        !aligned(k_pool, 16) || !aligned(v_pool, 16))
        return fail(LS_ERR_INVALID, "q, out and pool rows must be 16-byte aligned");
    if (batch == 0) return LS_OK;
    const ls::TreeShape s = ls::tree_shape(batch, kv_heads, nodes * n_rep,
                                           keys_bound(max_pages, max_seq_len));
    const size_t need = units_bytes(batch, kv_heads) + ls::tree_record_bytes(s);
    if (!aligned(workspace, 16) || workspace_bytes < need)
        return fail(LS_ERR_INVALID, "needs a 16-byte aligned workspace of %zu bytes", need);
    ls::TreeParams a = {};
    set_q(a, q, q_strides, out, out_strides);
    set_pool(a, pool_strides, num_blocks, block_tables, bt_stride, max_pages, seq_lens);
    a.pool[0] = (const char*)k_pool;
    a.pool[1] = (const char*)v_pool;
    a.masks = (const uint64_t*)masks;
    a.words = (nodes + 63) / 64;
    a.counts = counts;
    a.lse = lse;
    set_units(a, workspace, batch, kv_heads);
    a.B = batch;
    a.H = kv_heads;
    a.N = nodes;
    a.NR = n_rep;
    a.scale2 = softmax_scale * 1.4426950408889634f;
    return hip_status(ls::launch_tree_attention(a, s, (hipStream_t)stream), "ls_tree_attention");
}

size_t ls_decode_weights_workspace_bytes(int batch, int kv_heads, int n_rep, int max_pages,
                                         int max_seq_len) {
    const size_t tree =
        ls_tree_attention_workspace_bytes(batch, kv_heads, 1, n_rep, max_pages, max_seq_len);
    if (tree == 0) return 0;
    const size_t rows = (size_t)batch * kv_heads * n_rep;
    return ((tree + 255) & ~(size_t)255) + ((rows * 4 + 255) & ~(size_t)255) +
           rows * score_len(max_pages) * 4;
}

int ls_paged_decode_weights(const void* q, const int64_t* q_strides, const void* k_pool,
                            const void* v_pool, const int64_t* pool_strides, int64_t num_blocks,
                            const int32_t* block_tables, int64_t bt_stride, int max_pages,
                            const int32_t* seq_lens, void* out, const int64_t* out_strides,
                            float* sums, const int64_t* sum_strides, int64_t sum_len,
                            const int32_t* sum_rows, int num_sum_rows, void* workspace,
                            size_t workspace_bytes, int batch, int kv_heads, int n_rep,
                            int head_dim, int page, int max_seq_len, float softmax_scale,
                            void* stream) {
    if (!q || !q_strides || !k_pool || !v_pool || !out || !out_strides || !workspace)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (int rc = check_pool(pool_strides, num_blocks, head_dim, page)) return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens)) return rc;
    if (int rc = check_tree(1, n_rep)) return rc;
    if (int rc = check_sums(sums, sum_strides, sum_len, num_sum_rows)) return rc;
    if (int rc = check_scale(softmax_scale)) return rc;
    if (too_large(batch, kv_heads, max_pages))
        return fail(LS_ERR_INVALID, "batch x kv_heads x max_pages too large for one call");
    if (!rows_aligned(q, q_strides, 3, 2) || !rows_aligned(out, out_strides, 3, 2) ||
        !aligned(k_pool, 16) || !aligned(v_pool, 16))
        return fail(LS_ERR_INVALID, "q, out and pool rows must be 16-byte aligned");
    if (batch == 0) return LS_OK;
    const int64_t bound = keys_bound(max_pages, max_seq_len);
    const ls::TreeShape s = ls::tree_shape(batch, kv_heads, n_rep, bound);
    const size_t need =
        ls_decode_weights_workspace_bytes(batch, kv_heads, n_rep, max_pages, max_seq_len);
    if (!aligned(workspace, 16) || workspace_bytes < need)
        return fail(LS_ERR_INVALID, "needs a 16-byte aligned workspace of %zu bytes", need);
    ls::TreeParams a = {};
    const int64_t qs[4] = {q_strides[0], 0, q_strides[1], q_strides[2]};
    const int64_t os[4] = {out_strides[0], 0, out_strides[1], out_strides[2]};
    set_q(a, q, qs, out, os);
    set_pool(a, pool_strides, num_blocks, block_tables, bt_stride, max_pages, seq_lens);
    a.pool[0] = (const char*)k_pool;
    a.pool[1] = (const char*)v_pool;
    a.words = 1;
    const size_t rows = (size_t)batch * kv_heads * n_rep;
    char* w = (char*)workspace;
    set_units(a, w, batch, kv_heads);
    w += (units_bytes(batch, kv_heads) + ls::tree_record_bytes(s) + 255) & ~(size_t)255;
    a.lse = (float*)w;
    a.scores = (float*)(w + ((rows * 4 + 255) & ~(size_t)255));
    a.score_len = score_len(max_pages);
    a.B = batch;
    a.H = kv_heads;
    a.N = 1;
    a.NR = n_rep;
    a.scale2 = softmax_scale * 1.4426950408889634f;
    a.sums = sums;
    a.ss_row = sum_strides[0];
    a.ss_h = sum_strides[1];
    a.sum_len = sum_len;
    a.sum_rows = sum_rows;
    a.num_sum_rows = num_sum_rows;
    // four keys a thread of eight waves, in more rounds where sequences are longer
    a.score_parts = (int)std::min<int64_t>((bound + 2047) / 2048, 1024);
    return hip_status(ls::launch_tree_attention(a, s, (hipStream_t)stream), "ls_paged_decode_weights");
}

int ls_add_weights(const void* q, const int64_t* q_strides, const float* lse, const void* k_pool,
                   const int64_t* pool_strides, int64_t num_blocks, const int32_t* block_tables,
                   int64_t bt_stride, int max_pages, const int32_t* seq_lens, float* sums,
                   const int64_t* sum_strides, int64_t sum_len, const int32_t* sum_rows,
                   int num_sum_rows, const int32_t* path, const int32_t* lengths, int batch,
                   int kv_heads, int nodes, int path_len, int n_rep, int head_dim, int page,
                   int max_seq_len, float softmax_scale, void* stream) {
    if (!q || !q_strides || !lse || !k_pool) return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (int rc = check_pool(pool_strides, num_blocks, head_dim, page)) return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens)) return rc;
    if (int rc = check_tree(nodes, n_rep)) return rc;
    if (path_len < 0 || path_len > nodes || (!path && path_len != nodes))
        return fail(LS_ERR_INVALID, "path_len must be in [0, nodes], and nodes without a path; got %d",
                    path_len);
    if (int rc = check_sums(sums, sum_strides, sum_len, num_sum_rows)) return rc;
    if (int rc = check_scale(softmax_scale)) return rc;
    if (!rows_aligned(q, q_strides, 4, 2) || !aligned(k_pool, 16))
        return fail(LS_ERR_INVALID, "q and pool rows must be 16-byte aligned");
    if (batch == 0 || path_len == 0) return LS_OK;
    ls::WeighParams a = {};
    a.q = (const _Float16*)q;
    a.sq_b = q_strides[0];
    a.sq_n = q_strides[1];
    a.sq_h = q_strides[2];
    a.sq_r = q_strides[3];
    a.lse = lse;
    a.pool = (const char*)k_pool;
    set_pool(a, pool_strides, num_blocks, block_tables, bt_stride, max_pages, seq_lens);
    a.sums = sums;
    a.ss_row = sum_strides[0];
    a.ss_h = sum_strides[1];
    a.sum_len = sum_len;
    a.sum_rows = sum_rows;
    a.num_sum_rows = num_sum_rows;
    a.path = path;
    a.lengths = lengths;
    a.B = batch;
    a.H = kv_heads;
    a.N = nodes;
    a.P = path_len;
    a.NR = n_rep;
    a.scale2 = softmax_scale * 1.4426950408889634f;
    return hip_status(ls::launch_add_weights(a, keys_bound(max_pages, max_seq_len),
                                             (hipStream_t)stream), "ls_add_weights");
}

static int check_pools(void* const* k_pools, void* const* v_pools, int n) {
    if (n < 0) return fail(LS_ERR_INVALID, "the number of pools must be >= 0");
    if (n > 0 && (!k_pools || !v_pools)) return fail(LS_ERR_INVALID, "null pointer argument");
    for (int i = 0; i < n; ++i) {
        if (!k_pools[i] || !v_pools[i]) return fail(LS_ERR_INVALID, "null pointer argument");
        if (!aligned(k_pools[i], 16) || !aligned(v_pools[i], 16))
            return fail(LS_ERR_INVALID, "pool rows must be 16-byte aligned");
    }
    return LS_OK;
}

int ls_accept_tokens(const int64_t* tokens, const int32_t* parents, const int64_t* choices,
                     const int32_t* counts, int32_t* path, int32_t* lengths,
                     int64_t* next_tokens, void* const* k_pools, void* const* v_pools,
                     int num_pools, const int64_t* pool_strides, int64_t num_blocks,
                     const int32_t* block_tables, int64_t bt_stride, int max_pages,
                     const int32_t* seq_lens, int batch, int kv_heads, int nodes, int head_dim,
                     int page, void* stream) {
    if (!tokens || !parents || !choices || !path || !lengths || !next_tokens)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (int rc = check_tree(nodes, 1)) return rc;
    if (int rc = check_pools(k_pools, v_pools, num_pools)) return rc;
    if (int rc = check_pool(pool_strides, num_blocks, head_dim, page)) return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens)) return rc;
    if (batch == 0) return LS_OK;
    ls::MoveParams a = {};
    set_pool(a, pool_strides, num_blocks, block_tables, bt_stride, max_pages, seq_lens);
    a.B = batch;
    a.H = kv_heads;
    a.tokens = tokens;
    a.parents = parents;
    a.choices = choices;
    a.counts = counts;
    a.path = path;
    a.lengths = lengths;
    a.next = next_tokens;
    a.N = nodes;
    int at = 0;
    do {
        const int n = std::min(num_pools - at, ls::MOVE_POOLS / 2);
        for (int i = 0; i < n; ++i) {
            a.pool[2 * i] = (char*)k_pools[at + i];
            a.pool[2 * i + 1] = (char*)v_pools[at + i];
        }
        if (int rc = hip_status(ls::launch_accept_tokens(a, 2 * n, (hipStream_t)stream),
                                "ls_accept_tokens"))
            return rc;
        at += n;
    } while (at < num_pools);
    return LS_OK;
}

int ls_select_tokens(const float* sums, const int64_t* sum_strides, int64_t sum_len,
                     const int32_t* seq_lens, int32_t* keep, float* kept, int layers, int batch,
                     int kv_heads, int budget, int sinks, int recent, void* stream) {
    if ((!sums && sum_len > 0) || !sum_strides || !seq_lens || !keep || !kept)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (layers < 0 || (int64_t)layers * batch * kv_heads >= 1LL << 22)
        return fail(LS_ERR_INVALID, "layers x batch x kv_heads must be below 2^22");
    if (sum_len < 0 || sum_len > (int64_t)1 << 30)
        return fail(LS_ERR_INVALID, "sum_len must be in [0, 2^30], got %lld", (long long)sum_len);
    for (int i = 0; i < 3; ++i)
        if (sum_strides[i] < 0) return fail(LS_ERR_INVALID, "rows of sums must not run backwards");
    if (budget < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
        return fail(LS_ERR_INVALID, "budget must be >= 1 and hold sinks + recent, got %d for %d + %d",
                    budget, sinks, recent);
    if (batch == 0 || layers == 0) return LS_OK;
    ls::SelectParams a = {};
    a.sums = sums;
    a.ss_l = sum_strides[0];
    a.ss_b = sum_strides[1];
    a.ss_h = sum_strides[2];
    a.sum_len = sum_len;
    a.lens = seq_lens;
    a.keep = keep;
    a.kept = kept;
    a.L = layers;
    a.B = batch;
    a.H = kv_heads;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    return hip_status(ls::launch_select_tokens(a, (hipStream_t)stream), "ls_select_tokens");
}

int ls_move_tokens(void* const* k_pools, void* const* v_pools, int layers,
                   const int64_t* pool_strides, int64_t num_blocks, const int32_t* block_tables,
                   int64_t bt_stride, int max_pages, const int32_t* seq_lens,
                   const int32_t* keep, int batch, int kv_heads, int budget, int head_dim,
                   int page, void* stream) {
    if (!keep) return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = check_batch(batch, kv_heads)) return rc;
    if (int rc = check_pools(k_pools, v_pools, layers)) return rc;
    if (int rc = check_pool(pool_strides, num_blocks, head_dim, page)) return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens)) return rc;
    if (budget < 1) return fail(LS_ERR_INVALID, "budget must be >= 1, got %d", budget);
    if (batch == 0 || layers == 0) return LS_OK;
    ls::MoveParams a = {};
    set_pool(a, pool_strides, num_blocks, block_tables, bt_stride, max_pages, seq_lens);
    a.B = batch;
    a.H = kv_heads;
    a.keep = keep;
    a.budget = budget;
    for (int at = 0; at < layers; at += ls::MOVE_POOLS / 2) {
        const int n = std::min(layers - at, ls::MOVE_POOLS / 2);
        for (int i = 0; i < n; ++i) {
            a.pool[2 * i] = (char*)k_pools[at + i];
            a.pool[2 * i + 1] = (char*)v_pools[at + i];
        }
        a.first_layer = at;
        if (int rc = hip_status(ls::launch_move_tokens(a, 2 * n, (hipStream_t)stream), "ls_move_tokens"))
            return rc;
    }
    return LS_OK;
}

}  // extern "C"

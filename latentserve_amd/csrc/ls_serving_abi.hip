// C ABI of the 4-bit cache, page copies and token log probabilities: argument
// checks, then launches on the caller's stream.  Declared in
// include/latentserve_amd_serving.h.

#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/latentserve_amd.h"
#include "../../include/latentserve_amd_serving.h"
#include "ls_common.h"
#include "ls_serving.h"

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

int make_pools(ls::Int4Pools& p, const void* k_codes, const void* k_affine, const void* v_codes,
               const void* v_affine, const int64_t* page_strides, int64_t num_blocks, int kv_heads,
               int head_dim, int page) {
    if (!k_codes || !k_affine || !v_codes || !v_affine || !page_strides)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (head_dim != ls::HEAD_DIM) return fail(LS_ERR_INVALID, "head_dim must be 128, got %d", head_dim);
    if (page != ls::PAGE) return fail(LS_ERR_INVALID, "page (block_size) must be 16, got %d", page);
    if (kv_heads < 1 || kv_heads > 65535)
        return fail(LS_ERR_INVALID, "kv_heads must be in [1, 65535], got %d", kv_heads);
    if (num_blocks < 1 || num_blocks > (1LL << 31) - 1)
        return fail(LS_ERR_INVALID, "num_blocks must be in [1, 2^31)");
    const void* ptrs[4] = {k_codes, k_affine, v_codes, v_affine};
    for (int i = 0; i < 4; ++i)
        if (!aligned(ptrs[i], 16) || page_strides[i] % 16 != 0 || page_strides[i] < 0)
            return fail(LS_ERR_INVALID, "4-bit pools and their pages must start on 16 bytes");
    p.codes[0] = (char*)k_codes;
    p.affine[0] = (char*)k_affine;
    p.codes[1] = (char*)v_codes;
    p.affine[1] = (char*)v_affine;
    p.sc[0] = page_strides[0];
    p.sa[0] = page_strides[1];
    p.sc[1] = page_strides[2];
    p.sa[1] = page_strides[3];
    p.num_blocks = (int)num_blocks;
    return LS_OK;
}

int check_tables(const int32_t* block_tables, int64_t bt_stride, int max_pages,
                 const int32_t* seq_lens, int batch) {
    if (!block_tables || !seq_lens) return fail(LS_ERR_INVALID, "null pointer argument");
    if (batch < 0 || batch > 65535) return fail(LS_ERR_INVALID, "batch must be in [0, 65535], got %d", batch);
    if (max_pages < 1 || max_pages > (1 << 24))
        return fail(LS_ERR_INVALID, "max_pages (block-table width) must be in [1, 2^24]");
    if ((int64_t)batch * max_pages >= (1LL << 31))
        return fail(LS_ERR_INVALID, "batch x max_pages must be below 2^31");
    if (bt_stride < 0) return fail(LS_ERR_INVALID, "block-table rows must not run backwards");
    return LS_OK;
}

}  // namespace

extern "C" {

int ls_serving_abi_version(void) { return 1; }

int ls_int4_write(const void* k, const int64_t* k_strides, const void* v,
                  const int64_t* v_strides, const int64_t* slots, void* k_codes, void* k_affine,
                  void* v_codes, void* v_affine, const int64_t* page_strides, int64_t num_blocks,
                  int batch, int kv_heads, int tokens, int head_dim, int page, void* stream) {
    ls::Int4WriteParams a;
    if (!k || !k_strides || !v || !v_strides || !slots)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = make_pools(a.p, k_codes, k_affine, v_codes, v_affine, page_strides, num_blocks,
                            kv_heads, head_dim, page))
        return rc;
    if (batch < 0 || tokens < 0) return fail(LS_ERR_INVALID, "bad batch or tokens");
    if (batch > 0 && tokens > ((1LL << 31) - 1) / 16 / kv_heads / batch)
        return fail(LS_ERR_INVALID, "batch x heads x tokens too large for one write");
    if (!rows_aligned(k, k_strides, 3, 2) || !rows_aligned(v, v_strides, 3, 2))
        return fail(LS_ERR_INVALID, "k and v rows must be 16-byte aligned");
    if (batch == 0 || tokens == 0) return LS_OK;
    const void* src[2] = {k, v};
    const int64_t* st[2] = {k_strides, v_strides};
    for (int z = 0; z < 2; ++z) {
        a.src[z] = (const char*)src[z];
        a.ss_b[z] = 2 * st[z][0];
        a.ss_h[z] = 2 * st[z][1];
        a.ss_t[z] = 2 * st[z][2];
    }
    a.slots = slots;
    a.B = batch;
    a.H = kv_heads;
    a.N = tokens;
    return hip_status(ls::launch_int4_write(a, (hipStream_t)stream), "ls_int4_write");
}

int ls_int4_read(const void* k_codes, const void* k_affine, const void* v_codes,
                 const void* v_affine, const int64_t* page_strides, int64_t num_blocks,
                 const int32_t* block_tables, int64_t bt_stride, int max_pages,
                 const int32_t* seq_lens, void* k_out, void* v_out, int batch, int kv_heads,
                 int head_dim, int page, int length, void* stream) {
    ls::Int4ReadParams a;
    if (int rc = make_pools(a.p, k_codes, k_affine, v_codes, v_affine, page_strides, num_blocks,
                            kv_heads, head_dim, page))
        return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens, batch)) return rc;
    if (!k_out || !v_out) return fail(LS_ERR_INVALID, "null pointer argument");
    if (!aligned(k_out, 16) || !aligned(v_out, 16))
        return fail(LS_ERR_INVALID, "k_out and v_out must be 16-byte aligned");
    if (length < 0) return fail(LS_ERR_INVALID, "length must be >= 0");
    // (16 threads each, below 2^32)
    if (batch > 0 && length > ((1LL << 28) - 1) / kv_heads / batch)
        return fail(LS_ERR_INVALID, "batch x heads x length too large for one read");
    if (batch == 0 || length == 0) return LS_OK;
    a.tables = block_tables;
    a.st_b = bt_stride;
    a.max_pages = max_pages;
    a.lens = seq_lens;
    a.out[0] = (_Float16*)k_out;
    a.out[1] = (_Float16*)v_out;
    a.B = batch;
    a.H = kv_heads;
    a.L = length;
    return hip_status(ls::launch_int4_read(a, (hipStream_t)stream), "ls_int4_read");
}

int ls_int4_decode_groups(int batch, int kv_heads, int max_pages, int max_seq_len) {
    if (batch < 1 || kv_heads < 1 || max_pages < 1) return 0;
    int64_t pages = max_pages;
    if (max_seq_len > 0) pages = std::min<int64_t>(pages, ((int64_t)max_seq_len + 15) / 16);
    return ls::int4_groups(batch, kv_heads, pages);
}

size_t ls_int4_decode_workspace_bytes(int groups, int kv_heads, int n_rep) {
    if (groups < 1 || kv_heads < 1 || n_rep < 1) return 0;
    return (size_t)groups * 2 * kv_heads * ls::int4_record_floats(n_rep) * sizeof(float);
}

size_t ls_int4_decode_counter_ints(int groups, int kv_heads) {
    if (groups < 1 || kv_heads < 1) return 0;
    return (size_t)groups * kv_heads * ls::I4_COUNTER_STRIDE;
}

int ls_paged_decode_int4(const void* q, const int64_t* q_strides, const void* k_codes,
                         const void* k_affine, const void* v_codes, const void* v_affine,
                         const int64_t* page_strides, int64_t num_blocks,
                         const int32_t* block_tables, int64_t bt_stride, int max_pages,
                         const int32_t* seq_lens, void* out, const int64_t* out_strides,
                         float* workspace, size_t workspace_bytes, int32_t* counters, int batch,
                         int kv_heads, int n_rep, int head_dim, int page, int groups,
                         float softmax_scale, void* stream) {
    ls::Int4DecodeParams a;
    if (!q || !q_strides || !out || !out_strides || !workspace || !counters)
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (int rc = make_pools(a.p, k_codes, k_affine, v_codes, v_affine, page_strides, num_blocks,
                            kv_heads, head_dim, page))
        return rc;
    if (int rc = check_tables(block_tables, bt_stride, max_pages, seq_lens, batch)) return rc;
    if (n_rep < 1 || n_rep > ls::MAX_NREP)
        return fail(LS_ERR_INVALID, "n_rep must be in [1, 16], got %d", n_rep);
    if (groups < 1 || (int64_t)groups * kv_heads > ls::I4_MAX_GROUPS ||
        ls_int4_decode_workspace_bytes(groups, kv_heads, n_rep) >= (size_t)1 << 31)
        return fail(LS_ERR_INVALID, "groups must be >= 1, groups x kv_heads at most %d and the "
                    "workspace below 2^31 bytes", ls::I4_MAX_GROUPS);
    // (what a head's pages and the starts on sequences weigh together: 32-bit places)
    if ((int64_t)batch * ((int64_t)max_pages + 16) + groups >= (1LL << 31))
        return fail(LS_ERR_INVALID, "batch x (max_pages + 16) + groups must be below 2^31");
    if (!std::isfinite(softmax_scale)) return fail(LS_ERR_INVALID, "softmax_scale must be finite");
    if (!rows_aligned(q, q_strides, 3, 2) || !rows_aligned(out, out_strides, 3, 2))
        return fail(LS_ERR_INVALID, "q and out rows must be 16-byte aligned");
    if (!aligned(workspace, 16) ||
        workspace_bytes < ls_int4_decode_workspace_bytes(groups, kv_heads, n_rep))
        return fail(LS_ERR_INVALID, "needs a 16-byte aligned workspace of %zu bytes",
                    ls_int4_decode_workspace_bytes(groups, kv_heads, n_rep));
    if (!aligned(counters, 4)) return fail(LS_ERR_INVALID, "counters must be 4-byte aligned");
    if (batch == 0) return LS_OK;
    a.q = (const _Float16*)q;
    a.sq_b = q_strides[0];
    a.sq_h = q_strides[1];
    a.sq_r = q_strides[2];
    a.tables = block_tables;
    a.st_b = bt_stride;
    a.max_pages = max_pages;
    a.lens = seq_lens;
    a.out = (_Float16*)out;
    a.so_b = out_strides[0];
    a.so_h = out_strides[1];
    a.so_r = out_strides[2];
    a.work = workspace;
    a.counters = counters;
    a.B = batch;
    a.H = kv_heads;
    a.NR = n_rep;
    a.groups = groups;
    a.scale = softmax_scale;
    return hip_status(ls::launch_int4_decode(a, (hipStream_t)stream), "ls_paged_decode_int4");
}

int ls_page_copy(void* const* tensors, const int64_t* page_strides, const int64_t* page_bytes,
                 int num_tensors, int64_t num_pages, const int32_t* src, const int32_t* dst,
                 int pairs, void* stream) {
    if (num_tensors < 0 || pairs < 0 || num_pages < 0)
        return fail(LS_ERR_INVALID, "bad num_tensors, num_pages or pairs");
    if (pairs == 0) return LS_OK;
    if (!src || !dst || (num_tensors > 0 && (!tensors || !page_strides || !page_bytes)))
        return fail(LS_ERR_INVALID, "null pointer argument");
    for (int k = 0; k < num_tensors; ++k) {
        if (!tensors[k]) return fail(LS_ERR_INVALID, "null pointer argument");
        if (page_bytes[k] < 0 || page_bytes[k] > (1LL << 30))
            return fail(LS_ERR_INVALID, "a page is at most 2^30 bytes");
        if (num_pages > 1 && page_strides[k] < page_bytes[k])
            return fail(LS_ERR_INVALID, "pages must lie apart (stride %lld, %lld bytes)",
                        (long long)page_strides[k], (long long)page_bytes[k]);
    }
    // every page in range; no page written twice, none both read and written
    // (the order of a launch's reads and stores is not defined)
    for (int i = 0; i < pairs; ++i)
        if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
            return fail(LS_ERR_INVALID, "page pair %d (%d to %d) is outside [0, %lld)", i, src[i],
                        dst[i], (long long)num_pages);
    int32_t small[64];
    int32_t* sorted = small;
    if (pairs > 64) {
        sorted = new (std::nothrow) int32_t[pairs];
        if (!sorted) return fail(LS_ERR_INVALID, "out of host memory");
    }
    std::copy(dst, dst + pairs, sorted);
    std::sort(sorted, sorted + pairs);
    const bool twice = std::adjacent_find(sorted, sorted + pairs) != sorted + pairs;
    bool both = false;
    for (int i = 0; i < pairs && !twice && !both; ++i)
        both = std::binary_search(sorted, sorted + pairs, src[i]);
    if (sorted != small) delete[] sorted;
    if (twice) return fail(LS_ERR_INVALID, "a page is written twice");
    if (both) return fail(LS_ERR_INVALID, "a page is both read and written");

    ls::PageCopyParams a;
    for (int k0 = 0; k0 < num_tensors; k0 += ls::COPY_TENSORS) {
        const int nt = std::min(num_tensors - k0, ls::COPY_TENSORS);
        uint64_t bits = 16;
        for (int k = 0; k < nt; ++k) {
            a.base[k] = (char*)tensors[k0 + k];
            a.stride[k] = page_strides[k0 + k];
            a.bytes[k] = (int)page_bytes[k0 + k];
            bits |= (uint64_t)(uintptr_t)a.base[k] | (uint64_t)a.stride[k] | (uint64_t)a.bytes[k];
        }
        const int vec = (int)(bits & (~bits + 1));          // the lowest bit set: at most 16
        for (int p0 = 0; p0 < pairs; p0 += ls::COPY_PAIRS) {
            const int np = std::min(pairs - p0, ls::COPY_PAIRS);
            std::copy(src + p0, src + p0 + np, a.src);
            std::copy(dst + p0, dst + p0 + np, a.dst);
            if (int rc = hip_status(ls::launch_page_copy(a, nt, np, vec, (hipStream_t)stream),
                                    "ls_page_copy"))
                return rc;
        }
    }
    return LS_OK;
}

size_t ls_token_logprobs_workspace_bytes(int rows, int n, int top) {
    if (rows < 1 || n < 1 || top < 0 || top > ls::LOGPROB_MAX_TOP) return 0;
    const int parts = ls::logprob_parts(rows, n, top);
    if (parts == 1) return 0;
    return (size_t)rows * parts * ls::logprob_record_floats(top) * sizeof(float);
}

size_t ls_token_logprobs_counter_ints(int rows, int n, int top) {
    if (rows < 1 || n < 1) return 0;
    return ls::logprob_parts(rows, n, top) == 1 ? 0 : (size_t)rows;
}

int ls_token_logprobs(const void* x, int64_t x_stride, int elem_bytes, const int64_t* tokens,
                      int64_t token_stride, float* logprob, float* entropy, float* top_val,
                      int64_t* top_id, void* workspace, size_t workspace_bytes, int32_t* counters,
                      int rows, int n, int top, void* stream) {
    if (!x || !tokens || !logprob || !entropy || (top > 0 && (!top_val || !top_id)))
        return fail(LS_ERR_INVALID, "null pointer argument");
    if (elem_bytes != 2 && elem_bytes != 4)
        return fail(LS_ERR_INVALID, "elem_bytes must be 2 (fp16) or 4 (fp32), got %d", elem_bytes);
    if (n < 1 || n > (1 << 28)) return fail(LS_ERR_INVALID, "n must be in [1, 2^28], got %d", n);
    if (rows < 0) return fail(LS_ERR_INVALID, "rows must be >= 0");
    if (top < 0 || top > ls::LOGPROB_MAX_TOP || top > n)
        return fail(LS_ERR_INVALID, "top must be in [0, %d] and at most n, got %d",
                    ls::LOGPROB_MAX_TOP, top);
    if (!aligned(x, elem_bytes)) return fail(LS_ERR_INVALID, "x must be aligned to its elements");
    if (rows == 0) return LS_OK;
    ls::LogprobParams a;
    a.parts = ls::logprob_parts(rows, n, top);
    if ((int64_t)rows * a.parts >= 1LL << 24)                  // (256 threads each, below 2^32)
        return fail(LS_ERR_INVALID, "rows x n too large for one call");
    if (a.parts > 1) {
        const size_t need = ls_token_logprobs_workspace_bytes(rows, n, top);
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
            return fail(LS_ERR_INVALID, "needs a 16-byte aligned workspace of %zu bytes", need);
        if (!counters || !aligned(counters, 4))
            return fail(LS_ERR_INVALID, "counters is required");
    }
    a.x = x;
    a.sx = x_stride;
    a.tokens = tokens;
    a.s_tok = token_stride;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_val = top_val;
    a.top_id = top_id;
    a.part = (float*)workspace;
    a.counters = counters;
    a.rows = rows;
    a.n = n;
    a.top = top;
    return hip_status(ls::launch_token_logprobs(a, elem_bytes == 4, (hipStream_t)stream),
                      "ls_token_logprobs");
}

}  // extern "C"

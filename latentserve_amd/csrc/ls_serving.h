// Launch descriptors of the 4-bit cache, page copy and log-probability kernels
// (include/latentserve_amd_serving.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ls {

// ---- 4-bit pools ---------------------------------------------------------------
// One (page, KV head), 128 channels, 16 tokens (byte offsets inside it):
//   k_codes   1024: token t at 64 t; 16-byte piece g (0..3) of a token holds
//                   words j = 0..3, word j the channels 32 j + 8 g + (0..7)
//   k_affine   256: token t at 16 t; (s, m) fp16 pairs of its 4 channel groups
//   v_codes   1024: octet o (channels 8 o + (0..7)) at 64 o; its word of token t at 4 t
//   v_affine   256: group at 64, token quad at 16: s of its 4 tokens, then m
// A word's code i is its bits 4 i .. 4 i + 3.  An entry stands for
// fp16(m + s * code), one rounding.
//
// Why these: a wave's lane (g = lane / 16, c = lane % 16) is row c, k-slice g of
// an MFMA operand.  K: lane (g, c) takes token c's piece g, which is its 8
// channels of each of the four 32-channel steps.  V: lane (g, c) takes octet c's
// words of tokens 4 g .. 4 g + 3, the tokens whose softmax weights it holds.
// So each of a page's four loads is 16 bytes a lane and (codes) 1 KiB in a row,
// and no code moves between lanes.
constexpr int I4_CODES = 1024;    // bytes of a (page, head)
constexpr int I4_AFFINE = 256;
constexpr int I4_GROUP = 32;      // channels a step and minimum cover

struct Int4Pools {
    char* codes[2];               // K, V
    char* affine[2];
    int64_t sc[2], sa[2];         // page strides, bytes
    int num_blocks;
};

// Division by a number that the host knows: n / d = n * mul >> shift for 0 <= n < 2^31
// (mul = floor(2^shift / d) + 1 and 2^(shift - 31) >= d: mul d exceeds 2^shift by at most
// d, so n mul d / 2^shift exceeds n by less than 1).
struct Divisor {
    uint32_t mul;
    int shift;
};
inline Divisor make_divisor(uint32_t d) {
    int l = 0;
    while (l < 31 && (1u << l) < d) ++l;
    return {(uint32_t)((((uint64_t)1 << (31 + l)) / d) + 1), 31 + l};
}
__device__ __forceinline__ int divide(int n, Divisor d) {
    return (int)((uint64_t)(uint32_t)n * d.mul >> d.shift);
}

struct Int4WriteParams {
    const char* src[2];           // k, v [B, H, N, 128] fp16
    int64_t ss_b[2], ss_h[2], ss_t[2];   // strides, bytes
    const int64_t* slots;         // [B * N]
    Int4Pools p;
    int B, H, N;
    Divisor by_tokens, by_heads;  // set at launch
};

struct Int4ReadParams {
    Int4Pools p;
    const int32_t* tables;
    int64_t st_b;
    int max_pages;
    const int32_t* lens;
    _Float16* out[2];             // [B, L, H, 128], contiguous
    int B, H, L;
    Divisor by_heads, by_length;  // set at launch
};

struct Int4DecodeParams {
    const _Float16* q;
    int64_t sq_b, sq_h, sq_r;
    Int4Pools p;
    const int32_t* tables;
    int64_t st_b;
    int max_pages;
    const int32_t* lens;
    _Float16* out;
    int64_t so_b, so_h, so_r;
    float* work;                  // [groups][2][H] records
    int32_t* counters;            // [groups * H * I4_COUNTER_STRIDE], zero at rest
    int B, H, NR;
    int groups;                   // workgroups a KV head
    int rec;                      // floats of a record (set at launch, as the next)
    int extra;                    // pages that starting on a sequence counts as
    int skew;                     // long runs may differ (int4_decode_kernel)
    Divisor by_groups, by_heads;
    float scale;
};

constexpr int I4_COUNTER_STRIDE = 4;      // int32 a (group, head)
constexpr int I4_MAX_GROUPS = 1 << 20;    // groups x heads of a launch, at most

// Workgroups a head for these sizes, and the floats of the split records.
int int4_groups(int batch, int kv_heads, int64_t pages_bound);
constexpr int int4_record_floats(int n_rep) { return n_rep * 128 + 2 * 16; }

hipError_t launch_int4_write(const Int4WriteParams& a, hipStream_t stream);
hipError_t launch_int4_read(const Int4ReadParams& a, hipStream_t stream);
hipError_t launch_int4_decode(const Int4DecodeParams& a, hipStream_t stream);

// ---- page copy --------------------------------------------------------------------
// One launch's tensors and page pairs, in the kernel's arguments (3 KB of the
// 4 KB that a launch may pass): no list is sent to the device first.
constexpr int COPY_TENSORS = 64;
constexpr int COPY_PAIRS = 192;

struct PageCopyParams {
    char* base[COPY_TENSORS];
    int64_t stride[COPY_TENSORS];         // bytes from page to page
    int bytes[COPY_TENSORS];              // of a page
    int src[COPY_PAIRS], dst[COPY_PAIRS];
};

// vec: bytes a lane moves at once (16, 8, 4, 2 or 1; every base, stride and
// size a multiple of it).
hipError_t launch_page_copy(const PageCopyParams& a, int tensors, int pairs, int vec,
                            hipStream_t stream);

// ---- token log probabilities ----------------------------------------------------
constexpr int LOGPROB_MAX_TOP = 32;

struct LogprobParams {
    const void* x;                // logits, row stride sx (elements)
    int64_t sx;
    const int64_t* tokens;
    int64_t s_tok;
    float* logprob;               // [rows]
    float* entropy;
    float* top_val;               // [rows, top]
    int64_t* top_id;
    float* part;                  // [rows * parts] records
    int32_t* counters;            // [rows], zero at rest
    int rows, n, top, parts;
    int part_len;                 // of a streamed part (set at launch)
};

// Parts a row is split over, and the floats of a part's record.
int logprob_parts(int rows, int n, int top);
constexpr int logprob_record_floats(int top) { return 4 + 2 * top; }
hipError_t launch_token_logprobs(const LogprobParams& a, int fp32, hipStream_t stream);

}  // namespace ls

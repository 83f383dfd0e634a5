// The 4-bit cache's write and read kernels: K and V of new tokens quantized into
// their slots, and pool rows read back as fp16 values.
//
//   m = min, s = fp16((max - m) / 15) over a (token, head)'s 32 adjacent channels
//   (the next smaller s where m + 15 s would round past fp16's largest value),
//   code = nearest whole number to (x - m) / s (ties to even) in 0..15, 0 where
//   s is 0; an entry stands for fp16(m + s * code).
//
// Sixteen lanes take a (token, head)'s 16 octets of channels, so a group of 32 is
// a quad of lanes and its minimum and maximum two lane exchanges; a lane reads 16
// bytes and writes one word of codes.
//
// Small calls are bound by the launch and one round trip (16 tokens of 2 heads: 3.1 and 2.9
// us), large ones by their accesses: an item a thread, V's codes 4 bytes and its steps 2 at
// a place.  4 x 2048 tokens, 2 heads, 11 MB: write 6.9 us, read 5.3, a plain copy of as many
// bytes 3.0.

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int I4_THREADS = 256;
constexpr int I4_LANES = HEAD_DIM / 8;      // lanes a (token, head)

// Minimum / maximum / sum over the lane's quad.
__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, dpp_move<0xB1>(v));
    return fminf(v, dpp_move<0x4E>(v));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, dpp_move<0xB1>(v));
    return fmaxf(v, dpp_move<0x4E>(v));
}

__device__ __forceinline__ float quad_sum(float v) {
    v += dpp_move<0xB1>(v);
    return v + dpp_move<0x4E>(v);
}

// (blockIdx.y: K, V)
__global__ __launch_bounds__(I4_THREADS) void int4_write_kernel(const Int4WriteParams a) {
    const int z = blockIdx.y;
    const int o = threadIdx.x % I4_LANES;
    const int item = blockIdx.x * (I4_THREADS / I4_LANES) + threadIdx.x / I4_LANES;
    if (item >= a.B * a.H * a.N) return;                // (whole groups of 16 lanes)
    const int bh = divide(item, a.by_tokens), t_new = item - bh * a.N;     // (b, h, t)
    const int b = divide(bh, a.by_heads), h = bh - b * a.H;
    const int64_t slot = a.slots[(int64_t)b * a.N + t_new];
    const h8 x = *(const h8*)(a.src[z] + b * a.ss_b[z] + h * a.ss_h[z] + t_new * a.ss_t[z] + 16 * o);
    if (slot < 0 || slot >= (int64_t)a.p.num_blocks * PAGE) return;
    float lo = (float)x[0], hi = lo, sum = lo;
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        lo = fminf(lo, (float)x[e]);
        hi = fmaxf(hi, (float)x[e]);
        sum += (float)x[e];
    }
    lo = quad_min(lo);
    hi = quad_max(hi);
    // (min and max pass over a NaN; a sum of fp16 values is finite only if all are.  One
    // that is not makes m NaN, and so all of the group's entries)
    sum = quad_sum(sum);
    lo = sum - sum != 0.f ? __builtin_nanf("") : lo;
    // ((hi - lo) / 15 rounded once: a product with 1 / 15 corrected by its remainder, exact
    // fused steps; checked over all fp32 significands)
    constexpr float FIFTEENTH = 1.f / 15.f;
    const float span = hi - lo, near15 = span * FIFTEENTH;
    half_t s = (half_t)__builtin_fmaf(__builtin_fmaf(-15.f, near15, span), FIFTEENTH, near15);
    // (65520 is where fp16 rounds to infinity; s is then over 4000, and a step of it
    // less takes 15 s below max.  On this side the difference is exact wherever it comes
    // near lo, 15 s being a multiple of 2^-8 at least there; lo + 15 s is not: -2^-24 +
    // 65520 rounds to 65520.  Checked over all lo and all hi from 60000)
    if (lo >= 65520.f - 15.f * (float)s && hi <= 65504.f)
        s = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, s) - 1));
    // The nearest whole number to (x - m) / s, decided exactly: the fp32 quotient is off by
    // at most 16 * 2^-22 (the difference, the reciprocal and the product round once each,
    // the reciprocal by up to a step), so only where one lies within 2^-16 of a border
    // between two codes are a lane's eight taken again in 64 bits, where the difference is
    // exact (fp16 operands span 40 bits) and the quotient's rounding is far finer than the
    // distance of a border (4 x 2048 tokens, all in 64 bits: 1.3 us more).
    uint32_t word = 0;
    float off = 0.f;
    const float sf = (float)s, inv = sf > 0.f ? __builtin_amdgcn_rcpf(sf) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float r = ((float)x[e] - lo) * inv, c = rintf(r);
        off = fmaxf(off, fabsf(r - c));
        word |= (uint32_t)(c < 15.f ? c : 15.f) << (4 * e);
    }
    if (off > 0.5f - 0x1p-16f) {
        word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double c = rint(((double)(float)x[e] - (double)lo) / (double)sf);
            word |= (uint32_t)(c < 15. ? c : 15.) << (4 * e);
        }
    }
    const int64_t blk = slot / PAGE;
    const int t = (int)(slot % PAGE);
    char* codes = a.p.codes[z] + blk * a.p.sc[z] + (int64_t)h * I4_CODES;
    char* aff = a.p.affine[z] + blk * a.p.sa[z] + (int64_t)h * I4_AFFINE;
    const int grp = o / 4;
    if (z == 0) {
        *(uint32_t*)(codes + 64 * t + 16 * (o % 4) + 4 * grp) = word;
        if (o % 4 == 0) {
            const h2 sm = {s, (half_t)lo};
            *(h2*)(aff + 16 * t + 4 * grp) = sm;
        }
    } else {
        *(uint32_t*)(codes + 64 * o + 4 * t) = word;
        if (o % 4 == 0) {
            half_t* q = (half_t*)(aff + 64 * grp + 16 * (t / 4)) + t % 4;
            q[0] = s;
            q[4] = (half_t)lo;
        }
    }
}

// The eight entries of a word: fp16(m + s * code), each pair one fused multiply-add.
// (Codes become fp16 by a splice under the exponent of 1024: 1024 + code, less 1024.)
__device__ __forceinline__ h8 word_values(uint32_t w, half_t s, half_t m) {
    const h2 ss = {s, s}, mm = {m, m}, bias = {(half_t)1024.f, (half_t)1024.f};
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = w >> (4 * i) & 0x000F000Fu;           // codes i and i + 4
        const h2 c = __builtin_bit_cast(h2, two | 0x64006400u) - bias;
        const h2 y = __builtin_elementwise_fma(c, ss, mm);
        r[i] = y[0];
        r[i + 4] = y[1];
    }
    return r;
}

// (blockIdx.y: K, V)  Items (sequence, token, head), 16 lanes each.
__global__ __launch_bounds__(I4_THREADS) void int4_read_kernel(const Int4ReadParams a) {
    const int z = blockIdx.y;
    const int o = threadIdx.x % I4_LANES;
    const int item = blockIdx.x * (I4_THREADS / I4_LANES) + threadIdx.x / I4_LANES;
    if (item >= a.B * a.L * a.H) return;                // (below 2^28)
    const int bt = divide(item, a.by_heads), h = item - bt * a.H;
    const int b = divide(bt, a.by_length), pos = bt - b * a.L;
    h8 y = {};
    const int page = pos / PAGE, t = pos % PAGE;
    const int len = a.lens[b];
    const int blk = a.tables[(int64_t)b * a.st_b + (page < a.max_pages ? page : a.max_pages - 1)];
    if (pos < len && page < a.max_pages) {
        if ((unsigned)blk < (unsigned)a.p.num_blocks) {
            const char* codes = a.p.codes[z] + blk * a.p.sc[z] + (int64_t)h * I4_CODES;
            const char* aff = a.p.affine[z] + blk * a.p.sa[z] + (int64_t)h * I4_AFFINE;
            const int grp = o / 4;
            if (z == 0) {
                const h2 sm = *(const h2*)(aff + 16 * t + 4 * grp);
                y = word_values(*(const uint32_t*)(codes + 64 * t + 16 * (o % 4) + 4 * grp), sm[0],
                                sm[1]);
            } else {
                const half_t* q = (const half_t*)(aff + 64 * grp + 16 * (t / 4)) + t % 4;
                y = word_values(*(const uint32_t*)(codes + 64 * o + 4 * t), q[0], q[4]);
            }
        }
    }
    *(h8*)(a.out[z] + (int64_t)item * HEAD_DIM + 8 * o) = y;
}

hipError_t launch_int4_write(const Int4WriteParams& p, hipStream_t stream) {
    Int4WriteParams a = p;
    a.by_tokens = make_divisor(a.N);
    a.by_heads = make_divisor(a.H);
    const int64_t lanes = (int64_t)a.B * a.H * a.N * I4_LANES;
    hipLaunchKernelGGL(int4_write_kernel, dim3((unsigned)((lanes + I4_THREADS - 1) / I4_THREADS), 2),
                       dim3(I4_THREADS), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_int4_read(const Int4ReadParams& p, hipStream_t stream) {
    Int4ReadParams a = p;
    a.by_heads = make_divisor(a.H);
    a.by_length = make_divisor(a.L);
    const int64_t lanes = (int64_t)a.B * a.L * a.H * I4_LANES;
    hipLaunchKernelGGL(int4_read_kernel, dim3((unsigned)((lanes + I4_THREADS - 1) / I4_THREADS), 2),
                       dim3(I4_THREADS), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ls

// Paged GQA decode attention over 4-bit pools (layout: ls_serving.h).
//
//   out[b, h, r] = sum_t softmax_t(scale * q[b, h, r] . K[t]) V[t], entries of K
//   and V as they are read back: fp16(m + s * code).
//
//  * Partition: each KV head's pages of all sequences are one list, cut into equal
//    runs, one a workgroup, from the lengths on the device (one fixed grid serves
//    growing sequences under graph replay, and ragged batches balance without a
//    deal).  A run that crosses sequences takes them one after the other; a
//    sequence that crosses runs leaves one record a run (acc, m, l), merged by the
//    last of its groups to arrive (over 16 runs: by the last of each 16, then the
//    last of those): one launch.
//  * The waves of a group claim pairs of pages (so two calls on the same operands can differ
//    by a rounding: a wave sums other pages).  QK: S^T[32 tok x 16 rows] = K . Q^T,
//    eight 16x16x32 MFMAs (one a channel group and page); PV: O^T[128 ch x 16 rows]
//    += V^T . P^T, eight more.  The QK result is already the PV operand's layout, as
//    in the fp16 walk (ls_decode.hip).
//  * Codes to fp16: a nibble in a byte is an fp8 value, converted two at once, then one
//    packed fused multiply-add gives fp16(m + s * code).  V's words of two tokens are
//    first interleaved by bytes, so that a pair is two tokens of one channel, the
//    operand V^T needs.  (Spliced under fp16 exponents, two instructions a pair, B16 x
//    64K took 3 us more.)
//  * Bound: 160 bytes a token and head from HBM, and the codes' way to fp16 beside it
//    (351 vector instructions a wave and two pages, 17 MFMAs).  B16 x 16K, 2 heads, 84 MB:
//    22.9 us in a graph, 3.7 TB/s (a plain read of as many bytes 12.6); its loads alone take
//    18 us and its arithmetic alone 16, of each 8 before the first page and after the last
//    (lengths, table, pages; records, arrival, records).  B16 x 64K 62.6 us, 5.4 TB/s; B1 x
//    2048 is that chain, 7.4 us.
//  * Online softmax in the log2 domain; a step in which no row's maximum moved skips
//    the rescale.  Maxima and sums are fp32; a weight is two fp16 numbers, 21 bits and more
//    (one, as the fp16 walk has it, put a rounding of 2^-12 a weight beside the result's
//    own, and lost those below 2^-25 of the largest), summed as they are by an MFMA with
//    ones.  Up to 8 rows the second one takes matrix columns that were idle (B16 x 64K 62.6 ->
//    63.2 us, B48 ragged to 1531 of 8 heads 19.0 -> 19.2; as products of their own 67.6, 19.5).

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float I4_LOG2E = 1.4426950408889634f;
// The largest weight is 2^I4_TOP (it cancels in the division by their sum): the least that
// fp16 holds is then 2^-39 of it.  Against 1, all below 2^-25 vanished, a long tail under a
// large score with them.
constexpr float I4_TOP = 15.f;
constexpr int I4_PAIRED = MAX_NREP / 2;
constexpr int I4_NW = 4;                 // waves a group
constexpr int I4_ROW = HEAD_DIM + 4;     // LDS row: 16 rows written at once fall in different banks
constexpr int I4_RESIDENT = 512;         // groups resident at once: two a CU
// Fewest pages a run has: a pair a wave.
constexpr int I4_MIN_PAGES = 2 * I4_NW;
// Runs of at least this many pages (all groups have one then) differ, where two groups
// share each CU (512 groups in all, so head counts that divide 512; 3, 5, 6 or 7 heads make
// 510 or 511, and their runs stay even): loads of the older group's waves go first, and of even runs its own
// ended 5 us early at B16 x 16K; of 5 to 3 parts they end together.  (us, even /
// 5 to 3, of one machine and with the walk as it was then: B16 x 16K 24.4 / 23.6, B16 x 64K 66.0 / 62.4, 2 x 100K 22.9 / 21.0, B64 ragged to
// 4096 of 8 heads 41.5 / 38.9, B96 ragged to 16K 54.6 / 51.0.  A rule of speed only: any
// group may run anywhere.)
constexpr int I4_LONG_RUN = 24;
// Pages whose blocks a group holds in LDS at once.
constexpr int I4_TABLE = 2048;
// Records that one group merges.
constexpr int I4_CLUSTER = 16;

struct Int4Smem {
    float m[I4_NW][MAX_NREP];
    float l[I4_NW][MAX_NREP];
    alignas(16) float acc[I4_NW][MAX_NREP][I4_ROW];
    alignas(8) int blk[I4_TABLE];
    int claim;
    int is_last;
};

struct Int4Page {
    u4 kc, ka, vc, va;
};

struct Int4State {
    f4 acc[8];    // O^T tile e: row c, channels 8 (4 g + i) + e
    f4 l;         // the sum of row c's weights, in every element and lane group
    float m;      // running maximum of row c (log2 units)
};

__device__ __forceinline__ h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ uint32_t bits(h2 v) { return __builtin_bit_cast(uint32_t, v); }

// Four pairs of a word's codes as fp16, exactly: (0, 2), (1, 3), (4, 6), (5, 7).  A byte
// 0 .. 15 is that many times 2^-9 as fp8 (e4m3: 0 .. 7 its subnormals, 8 .. 15 the first
// normal ones), which the conversion multiplies by its power of two.
__device__ __forceinline__ void code_pairs(uint32_t x, h2 (&p)[4]) {
    const uint32_t lo = x & 0x0F0F0F0Fu, hi = (x >> 4) & 0x0F0F0F0Fu;
    p[0] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, false));
    p[1] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, false));
    p[2] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, true));
    p[3] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, true));
}

__device__ __forceinline__ h2 splat_lo(uint32_t x) {
    const h2 v = as_h2(x);
    return (h2){v[0], v[0]};
}
__device__ __forceinline__ h2 splat_hi(uint32_t x) {
    const h2 v = as_h2(x);
    return (h2){v[1], v[1]};
}

__device__ __forceinline__ f4 mfma32(u4 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), b, c, 0, 0, 0);
}

// Two weights as fp16, towards zero: one over fp16's largest value is that value, not an
// infinity.
__device__ __forceinline__ h2 truncated(float a, float b) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// blk < 0: zeros, without a memory request.
__device__ __forceinline__ void int4_load(const Int4DecodeParams& a, Int4Page& d, int blk, int h,
                                          int g, int c) {
    const bool fetch = blk >= 0;
    const int64_t bk = fetch ? blk : 0;
    const int64_t hc = (int64_t)h * I4_CODES, ha = (int64_t)h * I4_AFFINE;
    d.kc = page_load16(page_rsrc(a.p.codes[0] + bk * a.p.sc[0] + hc, fetch), 64 * c + 16 * g);
    d.ka = page_load16(page_rsrc(a.p.affine[0] + bk * a.p.sa[0] + ha, fetch), 16 * c);
    d.vc = page_load16(page_rsrc(a.p.codes[1] + bk * a.p.sc[1] + hc, fetch), 64 * c + 16 * g);
    d.va = page_load16(page_rsrc(a.p.affine[1] + bk * a.p.sa[1] + ha, fetch), 64 * (c / 4) + 16 * g);
}

// Two adjacent pages, the first one's first token tok0; token tok0 + i counts if it is
// below len[i / 16].  scale > 0.
//
// A weight p goes into the products as two fp16 numbers, itself truncated and what that
// leaves, 21 bits or more of it.  Up to 8 rows: in columns c and c + 8, which hold one
// row's scores (`take` is 0 in the first, -1 in the second), so they cost no product.  More
// rows (WIDE, take -1): a second product each.
template <bool WIDE>
__device__ __forceinline__ void int4_compute(const Int4Page (&d)[2],
                                             Int4State& st, const h8 (&q)[4], int tok0,
                                             const int (&len)[2], float scale, int g, float take) {
    f4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            h2 p[4];
            code_pairs(d[z].kc[j], p);
            const h2 ks = splat_lo(d[z].ka[j]), km = splat_hi(d[z].ka[j]);
            u4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = bits(__builtin_elementwise_fma(p[i], ks, km));
            s[z] = mfma32(w, q[j], s[z]);
        }
    }

    u4 va[2] = {d[0].va, d[1].va};
    // (the same in every lane)
    if (tok0 + PAGE > len[0] || tok0 + 2 * PAGE > len[1]) {
        const int t0 = tok0 + 4 * g;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int t = t0 + 16 * z, n = len[z];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[z][i] = t + i < n ? s[z][i] : neg_inf();
            // tokens past the end may hold anything, NaN steps included: entry 0
            // (a weight of 0 does not remove a NaN)
            const uint32_t m01 = (t < n ? 0xFFFFu : 0u) | (t + 1 < n ? 0xFFFF0000u : 0u);
            const uint32_t m23 = (t + 2 < n ? 0xFFFFu : 0u) | (t + 3 < n ? 0xFFFF0000u : 0u);
            va[z].x &= m01;
            va[z].y &= m23;
            va[z].z &= m01;
            va[z].w &= m23;
        }
    }
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]);
    top = fmaxf(fmaxf(top, s[0][3]), s[1][0]);
    top = fmaxf(fmaxf(top, s[1][1]), fmaxf(s[1][2], s[1][3]));
    top = group4_max(top);
    // (a row of -inf only has nothing valid yet)
    const float m_new = fmaxf(st.m, __builtin_fmaf(top, scale, -I4_TOP));
    const float m_use = m_new == neg_inf() ? 0.f : m_new;
    const float alpha = fast_exp2(st.m - m_use);
    h8 hi, part;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p0 = fast_exp2(__builtin_fmaf(s[i / 2][2 * (i % 2)], scale, -m_use));
        const float p1 = fast_exp2(__builtin_fmaf(s[i / 2][2 * (i % 2) + 1], scale, -m_use));
        const h2 a = truncated(p0, p1);
        const h2 b = truncated(__builtin_fmaf((float)a[0], take, p0),
                               __builtin_fmaf((float)a[1], take, p1));
        hi[2 * i] = a[0];
        hi[2 * i + 1] = a[1];
        part[2 * i] = b[0];
        part[2 * i + 1] = b[1];
    }
    if (__any(alpha != 1.f)) {
        st.l *= alpha;
#pragma unroll
        for (int t = 0; t < 8; ++t) st.acc[t] *= alpha;
    }
    st.m = m_new;
    constexpr uint32_t ONES = 0x3C003C00u;
    st.l = mfma32((u4){ONES, ONES, ONES, ONES}, part, st.l);
    if constexpr (WIDE) st.l = mfma32((u4){ONES, ONES, ONES, ONES}, hi, st.l);

#pragma unroll
    for (int half = 0; half < 2; ++half) {
        // this half's four codes of tokens 4g, 4g + 1 (and 4g + 2, 4g + 3), their bytes in
        // turn: a pair is one code of both
        const uint32_t sel = half ? 0x07030602u : 0x05010400u;
        u4 w[4];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            h2 p01[4], p23[4];
            code_pairs(__builtin_amdgcn_perm(d[z].vc.y, d[z].vc.x, sel), p01);
            code_pairs(__builtin_amdgcn_perm(d[z].vc.w, d[z].vc.z, sel), p23);
            const h2 s01 = as_h2(va[z].x), s23 = as_h2(va[z].y), m01 = as_h2(va[z].z),
                     m23 = as_h2(va[z].w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i][2 * z] = bits(__builtin_elementwise_fma(p01[i], s01, m01));
                w[i][2 * z + 1] = bits(__builtin_elementwise_fma(p23[i], s23, m23));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) st.acc[4 * half + i] = mfma32(w[i], part, st.acc[4 * half + i]);
        if constexpr (WIDE)
#pragma unroll
            for (int i = 0; i < 4; ++i) st.acc[4 * half + i] = mfma32(w[i], hi, st.acc[4 * half + i]);
    }
}

// Inclusive prefix sum over the wave's lanes, and its total: rows of 16 lanes by DPP
// row shifts (a lane whose source is outside its row adds 0), then the rows' totals.
template <int CTRL>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ int wave_incl_scan(int x, int lane, int& total) {
    x = dpp_add<0x118>(dpp_add<0x114>(dpp_add<0x112>(dpp_add<0x111>(x))));
    const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = __builtin_amdgcn_readlane(x, 31),
              r2 = __builtin_amdgcn_readlane(x, 47), r3 = __builtin_amdgcn_readlane(x, 63);
    total = r0 + r1 + r2 + r3;
    const int row = lane >> 4;
    return x + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}

// Lanes c and c ^ 8 of 16 added: a row rotation of 8 as part of the addition (every lane
// has a source; the sum stays where it is made, not under a later branch, apart from the move).
__device__ __forceinline__ float add_paired(float v) {
    float r = v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                                0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true));
    asm("" : "+v"(r));
    return r;
}

// The records of a sequence of a KV head: its first group's among those of sequences
// that start in their group, the others' among those that go on.
struct Int4Records {
    float* work;              // this head's
    int row_bytes;            // of a group's heads (the workspace is below 2^31 bytes)
    int groups, first;
    __device__ __forceinline__ int at(int k) const {
        return (k == 0 ? first : groups + first + k) * row_bytes;
    }
};

// Rows of the records k0, k0 + step, ... (S of them) merged by half-waves (lane j:
// channels 4 j .. 4 j + 3).  A round takes up to 16: lane j reads m and l of record j
// and its weight goes to the others by readlane, so every load of a round is requested
// at once.  The result goes to out, or (out null) to record k0.
__device__ __forceinline__ void merge_records(const Int4Records& R, int k0, int step, int S, int NR,
                                              half_t* out, int64_t so_r) {
    const int j = threadIdx.x % 32, d0 = 4 * j;
    const bool upper = (threadIdx.x & 32) != 0;
    const __amdgpu_buffer_rsrc_t rs = coherent_rsrc(wave_uniform(R.work));
    for (int r = threadIdx.x / 32; r < NR; r += I4_NW * 2) {
        float mg = neg_inf(), lt = 0.f;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        const int vo_a = (r * HEAD_DIM + d0) * (int)sizeof(float);
        const int vo_m = (NR * HEAD_DIM + 2 * r) * (int)sizeof(float);
        for (int i0 = 0; i0 < S; i0 += I4_CLUSTER) {
            const int n = S - i0 < I4_CLUSTER ? S - i0 : I4_CLUSTER;      // the same in every lane
            const uint64_t ml = load_coherent8(rs, vo_m + R.at(k0 + step * (i0 + (j < n ? j : n - 1))), 0);
            f4 av[I4_CLUSTER];
#pragma unroll
            for (int i = 0; i < I4_CLUSTER; ++i)
                av[i] = load_coherent4(rs, vo_a, R.at(k0 + step * (i0 + (i < n ? i : n - 1))));
            const float mj = j < n ? __builtin_bit_cast(float, (uint32_t)ml) : neg_inf();
            const float cm = fmaxf(half_max(mj), mg);
            const bool none = cm == neg_inf();
            const float sc = none ? 1.f : fast_exp2(mg - cm);
            const float wj = none || j >= n ? 0.f : fast_exp2(mj - cm);
            lt = lt * sc + half_sum(wj * __builtin_bit_cast(float, (uint32_t)(ml >> 32)));
            acc *= sc;
#pragma unroll
            for (int i = 0; i < I4_CLUSTER; ++i) {
                const float w0 = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wj), i));
                const float w1 = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wj), 32 + i));
                acc += av[i] * (upper ? w1 : w0);
            }
            mg = cm;
        }
        if (out) {
            const float inv = 1.f / fmaxf(lt, 1e-20f);
            half_t* o = out + (int64_t)r * so_r + d0;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (half_t)(acc[e] * inv);
        } else {
            float* rk = (float*)((char*)R.work + R.at(k0));
            store_coherent4(rk + r * HEAD_DIM + d0, acc);
            if (j == 0) store_coherent2(rk + NR * HEAD_DIM + 2 * r, mg, lt);
        }
    }
}

// WIDE: more than I4_PAIRED rows (int4_compute).
template <bool WIDE>
__global__ __launch_bounds__(WAVE* I4_NW) __attribute__((amdgpu_waves_per_eu(2)))
void int4_decode_kernel(const Int4DecodeParams a) {
    __shared__ Int4Smem sm;
    const int H = a.H, NR = a.NR;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int g = lane >> 4, c = lane & 15;

    // ---- its run of the head's page list, and the sequence that run starts in ----
    // A sequence weighs its pages and `extra` (what starting on it costs a group, in
    // pages), which lie before them.  (One of no tokens counts a page, which nobody
    // reads: its group stores the zeros.)
    const int extra = a.extra;
    auto pages_of = [&](int len) {
        int p = len > 0 ? (len - 1) / PAGE + 1 : 1;
        return p < a.max_pages ? p : a.max_pages;
    };
    // This group's run and head: neighbouring runs on one XCD, whose L2 has their tables
    // and queries.
    int w, h;
    auto place = [&](int u) {
        w = divide(u, a.by_heads);
        h = u - w * H;
    };
    place(xcd_major(blockIdx.x, gridDim.x));
    // A run's pages `per`; with `skew` runs take more and fewer, `big` and 2 per - big, in
    // turn.
    int per, big;
    bool skew;
    auto run_of = [&](int T, int& u0, int& u1) {
        per = divide(T + a.groups - 1, a.by_groups);
        per = per > I4_MIN_PAGES ? per : I4_MIN_PAGES;
        skew = a.skew != 0 && per >= I4_LONG_RUN;
        big = per;
        if (skew) {
            big += per / 4;
            const int L = blockIdx.x, half = gridDim.x / 2;
            place(L < half ? L : L - half);
            w = 2 * w + (L < half ? 0 : 1);
        } else if (per == I4_MIN_PAGES) {
            // (lengths below the bound's: the groups that have a run, over all XCDs)
            const int L = blockIdx.x, used = (T + I4_MIN_PAGES - 1) / I4_MIN_PAGES * H;
            if (used < (int)gridDim.x) place(L < used ? xcd_major(L, used) : L);
        }
        const int64_t at = (int64_t)(w / 2) * 2 * per + (w & 1 ? big : 0);
        const int mine = w & 1 ? 2 * per - big : big;
        u0 = at < T ? at : T;
        u1 = T - u0 < mine ? T : u0 + mine;
    };
    auto group_of = [&](int page) {
        if (!skew) return page / per;
        const int pair = page / (2 * per);
        return 2 * pair + (page - pair * 2 * per < big ? 0 : 1);
    };
    int b, P, len, u0, u1;           // the first sequence, its start, length; the run
    if (a.B <= WAVE) {
        // one sequence a lane
        const int li = lane < a.B ? a.lens[lane] : 0;
        const int n = lane < a.B ? pages_of(li) + extra : 0;
        int T;
        const int incl = wave_incl_scan(n, lane, T);
        run_of(T, u0, u1);
        if (u0 >= T) return;                         // (every wave alike, before any barrier)
        b = __builtin_ctzll(__ballot(u0 < incl));    // (lanes past the batch hold T)
        P = __builtin_amdgcn_readlane(incl - n, b);
        len = __builtin_amdgcn_readlane(li, b);
    } else {
        // a run of sequences a lane
        const int per_lane = (a.B + WAVE - 1) / WAVE;
        const int b0 = lane * per_lane < a.B ? lane * per_lane : a.B;
        const int b1 = b0 + per_lane < a.B ? b0 + per_lane : a.B;
        int mine = 0;
        for (int i = b0; i < b1; ++i) mine += pages_of(a.lens[i]) + extra;
        int T;
        const int incl = wave_incl_scan(mine, lane, T);
        run_of(T, u0, u1);
        if (u0 >= T) return;
        int pos = incl - mine, fb = 0, fp = 0, fl = 0;
        const bool holds = u0 >= pos && u0 < incl;
        if (holds) {
            for (int i = b0; i < b1; ++i) {
                const int li = a.lens[i], n = pages_of(li) + extra;
                if (u0 < pos + n) {
                    fb = i;
                    fp = pos;
                    fl = li;
                    break;
                }
                pos += n;
            }
        }
        const int src = __builtin_ctzll(__ballot(holds));
        b = __builtin_amdgcn_readlane(fb, src);
        P = __builtin_amdgcn_readlane(fp, src);
        len = __builtin_amdgcn_readlane(fl, src);
    }
    if (u1 <= P + extra) return;                     // (none of its pages)

    // q's sign takes the scale's, so that a larger product is a larger score; a scale of
    // 0 is the smallest there is (of -inf, a masked score, nothing else would stay -inf).
    const float scale = fmaxf(fabsf(a.scale) * I4_LOG2E, 0x1p-126f);
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    int mine = 0;                                    // 0, which the compiler does not know
    asm("" : "+v"(mine));
    // Lane c's query row (past n_rep: row 0, never stored), channels 32 j + 8 g + (0..7).
    const int row_of = WIDE ? c : c % I4_PAIRED;
    float take = WIDE || c >= I4_PAIRED ? -1.f : 0.f;
    if constexpr (WIDE) asm("" : "+s"(take));        // (of a known -1, two instructions)
    auto load_q = [&](int bq, u4 (&t)[4]) {
        const half_t* row = a.q + (int64_t)bq * a.sq_b + (int64_t)h * a.sq_h +
                            (int64_t)(row_of < NR ? row_of : 0) * a.sq_r + 8 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = *(const u4*)(row + 32 * j);
    };
    // A block from the table, -1 where it lies outside the pool.
    auto valid = [&](int t) { return (unsigned)t < (unsigned)a.p.num_blocks ? t : -1; };

    int s0 = u0 - P - extra;
    s0 = s0 > 0 ? s0 : 0;
    u4 q_raw[4];
    load_q(b, q_raw);
    // the table entries of the wave's first pair (lanes 0 and 1), past the table's end
    // the last one's
    auto first_entries = [&](int bt, int from) {
        const int p = from + 2 * wv + (lane & 1);
        return a.tables[(int64_t)bt * a.st_b + (p < a.max_pages ? p : a.max_pages - 1)];
    };
    int entry = first_entries(b, s0);
    // ... and the group's first ones, a thread each, requested ahead of any page so
    // that the table need not wait for one
    auto table_entry = [&](int bt, int from) {
        const int p = from + (int)threadIdx.x;
        return a.tables[(int64_t)bt * a.st_b + (p < a.max_pages ? p : a.max_pages - 1)];
    };
    int filled = table_entry(b, s0);

    Int4Page page[2][2];
    int item[2], blk[2][2];
    auto request = [&](int slot, int it, int b0, int b1) {
        item[slot] = it;
        blk[slot][0] = b0;
        blk[slot][1] = b1;
        int4_load(a, page[slot][0], b0, h, g, c);
        int4_load(a, page[slot][1], b1, h, g, c);
    };
    bool requested = false;          // the segment's first pair is on its way
    while (true) {
        // ---- this run's pages [s0, s1) of sequence b ----
        const int n = pages_of(len), start = P + extra;
        const int s1 = u1 - start < n ? u1 - start : n;
        const int pages = len > 0 ? n : 0;
        const bool more = P + extra + n + extra < u1;     // the next sequence has pages here
        auto request_first = [&](int from, int to, int limit) {
            const int i = from + 2 * wv;
            const int b0 = valid(__builtin_amdgcn_readlane(entry, 0));
            const int b1 = valid(__builtin_amdgcn_readlane(entry, 1));
            request(0, wv, i < to && i < limit ? b0 : -1, i + 1 < to && i + 1 < limit ? b1 : -1);
        };
        if (!requested) request_first(s0, s1, pages);
        h8 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const h8 t = __builtin_bit_cast(h8, (u4)(q_raw[j] ^ flip));
            q[j] = (h8){t[0], t[2], t[1], t[3], t[4], t[6], t[5], t[7]};
        }
        // what the next sequence of the run needs, ahead of its turn
        const int b_next = more ? b + 1 : b;
        const int len_next = a.lens[b_next];
        const int entry_next = first_entries(b_next, 0), filled_next = table_entry(b_next, 0);
        load_q(b_next, q_raw);

        Int4State st;
#pragma unroll
        for (int t = 0; t < 8; ++t) st.acc[t] = (f4){0.f, 0.f, 0.f, 0.f};
        st.l = (f4){0.f, 0.f, 0.f, 0.f};
        st.m = neg_inf();
        const int32_t* trow = a.tables + (int64_t)b * a.st_b;
        // The pages' blocks in LDS, a run of more than I4_TABLE pages in pieces; the
        // waves claim pairs of pages one by one (the oldest win memory arbitration: with
        // static shares the youngest ended 5 us later at B16 x 16K), the first pair of
        // each fixed, so that it is requested while the table fills.
        for (int c0 = s0; c0 < s1; c0 += I4_TABLE) {
            const int n_pg = s1 - c0 < I4_TABLE ? s1 - c0 : I4_TABLE, pairs = (n_pg + 1) / 2;
            if (c0 != s0) {
                __syncthreads();                           // the piece before is claimed out
                entry = first_entries(b, c0);
                filled = table_entry(b, c0);
                request_first(c0, s1, pages);
            }
            {
                const int i = threadIdx.x;
                if (i < 2 * pairs) sm.blk[i] = i < n_pg && c0 + i < pages ? valid(filled) : -1;
            }
            for (int i = threadIdx.x + WAVE * I4_NW; i < 2 * pairs; i += WAVE * I4_NW)
                sm.blk[i] = i < n_pg && c0 + i < pages ? valid(trow[c0 + i]) : -1;
            if (threadIdx.x == 0) sm.claim = 2 * I4_NW;
            __syncthreads();
            // A step takes the pair whose blocks the step before read from the table,
            // requests it, computes the one requested before, and meanwhile the pair
            // after has its blocks read and the one after that is claimed: no step
            // waits for LDS.
            auto claim = [&]() {
                int r = 0;
                // (an address of the lane's own: of one known to be the same in every
                // lane the compiler would add for the wave and wait for it at once)
                if (lane == 0)
                    r = __hip_atomic_fetch_add(&sm.claim + mine, 1, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_WORKGROUP);
                return r;
            };
            auto blocks = [&](int it) { return *(const u2*)&sm.blk[2 * (it < pairs ? it : 0)]; };
            int ahead = wv + I4_NW;
            u2 ahead_blk = blocks(ahead);
            int claimed = claim();
            bool live = item[0] < pairs;
            while (live) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    if (!live) break;
                    // (requested past the end too, from no bytes: loads under a branch would
                    // make the compute wait for them, not for the ones before)
                    const bool there = ahead < pairs;
                    const int b0 = __builtin_amdgcn_readfirstlane(ahead_blk.x);
                    const int b1 = __builtin_amdgcn_readfirstlane(ahead_blk.y);
                    request(z ^ 1, ahead, there ? b0 : -1, there ? b1 : -1);
                    ahead = __builtin_amdgcn_readfirstlane(claimed);
                    ahead_blk = blocks(ahead);
                    claimed = claim();
                    const int lens[2] = {blk[z][0] >= 0 ? len : 0, blk[z][1] >= 0 ? len : 0};
                    int4_compute<WIDE>(page[z], st, q, (c0 + 2 * item[z]) * PAGE, lens, scale, g, take);
                    live = there;
                }
            }
        }
        // both parts of each weight (ahead of the next loads, whose registers this takes)
        if constexpr (!WIDE) {
            st.l[0] = add_paired(st.l[0]);
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) st.acc[t][i] = add_paired(st.acc[t][i]);
        }
        // the next sequence's first pair, on its way while this one is merged
        entry = entry_next;
        filled = filled_next;
        if (more) {
            const int n2 = pages_of(len_next), start2 = start + n + extra;
            request_first(0, u1 - start2 < n2 ? u1 - start2 : n2, len_next > 0 ? n2 : 0);
            requested = true;
        }

        // ---- the waves' states merged in LDS ----
        if (c < NR) {
            if (g == 0) {
                sm.m[wv][c] = st.m;
                sm.l[wv][c] = st.l[0];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = st.acc[4 * k + e][i];
                    *(f4*)&sm.acc[wv][c][32 * g + 8 * i + 4 * k] = v;
                }
            }
        }
        __syncthreads();
        const bool whole = s0 == 0 && s1 == n;
        const int first = group_of(start);                   // the sequence's first group
        const Int4Records R = {a.work + (int64_t)h * a.rec, H * a.rec * (int)sizeof(float), a.groups,
                               first};
        const int d0 = 4 * (threadIdx.x % 32);
        float* record = (float*)((char*)R.work + R.at(w - first));
        half_t* orow = a.out + (int64_t)b * a.so_b + (int64_t)h * a.so_h;
        for (int r = threadIdx.x / 32; r < NR; r += I4_NW * 2) {
            float mg = neg_inf();
#pragma unroll
            for (int v = 0; v < I4_NW; ++v) mg = fmaxf(mg, sm.m[v][r]);
            float lt = 0.f;
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < I4_NW; ++v) {
                const float wt = mg == neg_inf() ? 0.f : fast_exp2(sm.m[v][r] - mg);
                lt += sm.l[v][r] * wt;
                acc += *(const f4*)&sm.acc[v][r][d0] * wt;
            }
            if (whole) {
                const float inv = 1.f / fmaxf(lt, 1e-20f);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    orow[(int64_t)r * a.so_r + d0 + e] = (half_t)(acc[e] * inv);
            } else {
                store_coherent4(record + r * HEAD_DIM + d0, acc);
                if (d0 == 0) store_coherent2(record + NR * HEAD_DIM + 2 * r, mg, lt);
            }
        }
        if (!whole) {
            // ---- the last of the sequence's groups to arrive merges their records ----
            const int S = group_of(start + n - 1) - first + 1;
            const int k = w - first, cl = k / I4_CLUSTER;
            const bool tree = S > I4_CLUSTER;
            // arrival counters: [0] the sequence's, at its first group; [1], [2] of 16
            // groups, at the first of them (two, since that group may start another
            // sequence, whose own first 16 count there)
            auto arrive = [&](int group, int which, int all) {
                handoff_release();
                __syncthreads();
                if (threadIdx.x == 0) {
                    int32_t* counter = a.counters + ((int64_t)group * H + h) * I4_COUNTER_STRIDE + which;
                    const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED,
                                                              __HIP_MEMORY_SCOPE_AGENT);
                    sm.is_last = before == all - 1;
                    if (before == all - 1)                 // back to zero for the next launch
                        __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                return sm.is_last != 0;
            };
            int k0 = tree ? cl * I4_CLUSTER : 0, step = 1, count = tree ? S - k0 : S;
            count = count < I4_CLUSTER ? count : I4_CLUSTER;
            int which = tree ? (cl == 0 ? 1 : 2) : 0;
            while (arrive(first + k0, which, count)) {
                merge_records(R, k0, step, count, NR, which == 0 ? orow : nullptr, a.so_r);
                if (which == 0) break;
                which = 0;
                k0 = 0;
                step = I4_CLUSTER;
                count = (S + I4_CLUSTER - 1) / I4_CLUSTER;
            }
        }
        if (!more) return;
        P = start + n;
        s0 = 0;
        b = b_next;
        len = len_next;
        __syncthreads();                 // the merge's LDS reads end before the next states
    }
}

// What starting on a sequence costs a group beside its pages (its first loads, its merge),
// in pages, where groups start on them often: with pages alone, the groups of short
// sequences end late (us, 0 -> 16 -> 32 pages, ragged lengths: B250 to 500, 4 heads 35.0
// -> 23.6 -> 26.6; B48 to 1531, 8 heads 23.3 -> 20.5 -> 25.1; B96 to 16K 61.3 -> 58.4 ->
// 60.9); where most groups start on none, it would take pages from the ones that do.
constexpr int I4_EXTRA = 16;

int int4_groups(int batch, int kv_heads, int64_t pages_bound) {
    int64_t most = I4_RESIDENT / kv_heads;
    most = most > 1 ? most : 1;
    const int64_t need = (batch * pages_bound + I4_MIN_PAGES - 1) / I4_MIN_PAGES;
    return (int)(need < most ? (need > 1 ? need : 1) : most);
}

hipError_t launch_int4_decode(const Int4DecodeParams& a, hipStream_t stream) {
    Int4DecodeParams d = a;
    d.rec = int4_record_floats(a.NR);
    d.by_groups = make_divisor(a.groups);
    d.by_heads = make_divisor(a.H);
    // (pairs of runs to the blocks L and L + 256, which the dispatcher gives one CU)
    d.skew = a.groups * a.H == I4_RESIDENT && a.groups % 2 == 0;
    d.extra = 4 * a.B > a.groups ? I4_EXTRA : 0;
    const dim3 grid(a.groups * a.H), block(WAVE * I4_NW);
    if (a.NR > I4_PAIRED) hipLaunchKernelGGL(int4_decode_kernel<true>, grid, block, 0, stream, d);
    else hipLaunchKernelGGL(int4_decode_kernel<false>, grid, block, 0, stream, d);
    return hipGetLastError();
}

}  // namespace ls

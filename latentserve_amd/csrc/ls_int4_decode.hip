// Paged GQA decode attention over 4-bit pools (layout: ls_serving.h).
//
//   out[b, h, r] = sum_t softmax_t(scale * q[b, h, r] . K[t]) V[t], entries of K
//   and V as they are read back: fp16(m + s * code).
//
//  * Partition: each KV head's pages of all sequences are one list, cut into equal
//    runs, one a workgroup, from the lengths on the device (one fixed grid serves
//    growing sequences under graph replay, and ragged batches balance without a
//    deal).  A run that crosses sequences takes them one after the other; a
//    sequence that crosses runs leaves one record a run (acc, m, l), and the last
//    of its groups to arrive merges them: one launch.
//  * A wave takes a page at a time.  QK: S^T[16 tok x 16 rows] = K . Q^T, four
//    16x16x32 MFMAs (one a channel group); PV: O^T[128 ch x 16 rows] += V^T . P^T,
//    eight 16x16x16 MFMAs.  The QK result is already the PV operand's layout, as
//    in the fp16 walk (ls_decode.hip).
//  * Codes to fp16: two of a word's codes at once are masked under the exponent
//    of 1024.0h (bits 0..3 of a half) or 64.0h (bits 4..7), the bias subtracted
//    exactly, then one packed fused multiply-add gives fp16(m + s * code).  V's
//    words of two tokens are first spliced by halves, so that a pair is two tokens
//    of one channel, the operand V^T needs.
//  * Online softmax in the log2 domain; rows whose maximum did not move skip the
//    rescale.  Sums and maxima are fp32; the weights are rounded to fp16 for the
//    MFMA as the fp16 walk rounds them.

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float I4_LOG2E = 1.4426950408889634f;
constexpr int I4_NW = 4;                 // waves a group
constexpr int I4_ROW = HEAD_DIM + 4;     // LDS row: 16 rows written at once fall in different banks
// Fewest pages a group takes: one a wave.
constexpr int I4_MIN_PAGES = I4_NW;
// Groups resident at once on the 256 CUs.
constexpr int I4_RESIDENT = 256 * 2;

struct Int4Smem {
    float m[I4_NW][MAX_NREP];
    float l[I4_NW][MAX_NREP];
    alignas(16) float acc[I4_NW][MAX_NREP][I4_ROW];
    int is_last;
};

struct Int4Page {
    u4 kc, ka, vc, va;
};

struct Int4State {
    f4 acc[8];    // O^T tile e: row c, channels 8 (4 g + i) + e
    float m, l;   // running maximum of row c (log2 units), lane-partial sum
};

__device__ __forceinline__ h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }

// Four pairs of codes: pair i is codes i and i + 4 of the word (of each half of
// the dword), as fp16, exactly.
__device__ __forceinline__ void code_pairs(uint32_t x, h2 (&p)[4]) {
    const h2 b1024 = {(half_t)1024.f, (half_t)1024.f}, b64 = {(half_t)64.f, (half_t)64.f};
    const uint32_t y = x >> 8;
    p[0] = as_h2((x & 0x000F000Fu) | 0x64006400u) - b1024;
    p[1] = as_h2((x & 0x00F000F0u) | 0x54005400u) - b64;
    p[2] = as_h2((y & 0x000F000Fu) | 0x64006400u) - b1024;
    p[3] = as_h2((y & 0x00F000F0u) | 0x54005400u) - b64;
}

__device__ __forceinline__ h2 splat_lo(uint32_t x) {
    const h2 v = as_h2(x);
    return (h2){v[0], v[0]};
}
__device__ __forceinline__ h2 splat_hi(uint32_t x) {
    const h2 v = as_h2(x);
    return (h2){v[1], v[1]};
}
__device__ __forceinline__ uint32_t bits(h2 v) { return __builtin_bit_cast(uint32_t, v); }

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

// The page's first token is tok0; tokens at or past len do not count.
__device__ __forceinline__ void int4_compute(const Int4Page& d, Int4State& st, const h8 (&q)[4],
                                             int tok0, int len, float scale_log2, int g) {
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h2 p[4];
        code_pairs(d.kc[j], p);
        const h2 ks = splat_lo(d.ka[j]), km = splat_hi(d.ka[j]);
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bits(__builtin_elementwise_fma(p[i], ks, km));
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, w), q[j], s, 0, 0, 0);
    }

    const int t0 = tok0 + 4 * g;
    float x[4];
    float mloc = neg_inf();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = t0 + i < len ? s[i] * scale_log2 : neg_inf();
        mloc = fmaxf(mloc, x[i]);
    }
    const float m_new = fmaxf(st.m, group4_max(mloc));
    const bool dead = m_new == neg_inf();      // nothing valid yet in this row
    const float alpha = dead ? 0.f : fast_exp2(st.m - m_new);
    float psum = 0.f;
    h4 pb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = dead ? 0.f : fast_exp2(x[i] - m_new);
        psum += p;
        pb[i] = (half_t)p;
    }
    st.l = st.l * alpha + psum;
    st.m = m_new;
    if (__any(alpha != 1.f)) {
#pragma unroll
        for (int t = 0; t < 8; ++t) st.acc[t] *= alpha;
    }

    u4 va = d.va;
    if (tok0 + PAGE > len) {
        // tokens past the end may hold anything, NaN steps included: entry 0
        // (a weight of 0 does not remove a NaN)
        const uint32_t m01 = (t0 < len ? 0xFFFFu : 0u) | (t0 + 1 < len ? 0xFFFF0000u : 0u);
        const uint32_t m23 = (t0 + 2 < len ? 0xFFFFu : 0u) | (t0 + 3 < len ? 0xFFFF0000u : 0u);
        va.x &= m01;
        va.y &= m23;
        va.z &= m01;
        va.w &= m23;
    }
    const h2 s01 = as_h2(va.x), s23 = as_h2(va.y), m01 = as_h2(va.z), m23 = as_h2(va.w);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        // this half's four codes of tokens 4g, 4g + 1 (and 4g + 2, 4g + 3)
        const uint32_t sel = half ? 0x07060302u : 0x05040100u;
        h2 p01[4], p23[4];
        code_pairs(__builtin_amdgcn_perm(d.vc.y, d.vc.x, sel), p01);
        code_pairs(__builtin_amdgcn_perm(d.vc.w, d.vc.z, sel), p23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const h2 v01 = __builtin_elementwise_fma(p01[i], s01, m01);
            const h2 v23 = __builtin_elementwise_fma(p23[i], s23, m23);
            const int e = 4 * half + i;
            st.acc[e] = mfma16(as_h4(bits(v01), bits(v23)), pb, st.acc[e]);
        }
    }
}

__device__ __forceinline__ int wave_incl_scan(int x, int lane) {
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

__device__ __forceinline__ void store_coherent(float* p, f4 v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1" : : "v"(p), "v"(v) : "memory");
}
__device__ __forceinline__ void store_coherent(float* p, float x, float y) {
    u2 v;
    v.x = __builtin_bit_cast(uint32_t, x);
    v.y = __builtin_bit_cast(uint32_t, y);
    asm volatile("global_store_dwordx2 %0, %1, off sc1" : : "v"(p), "v"(v) : "memory");
}

__global__ __launch_bounds__(WAVE* I4_NW) __attribute__((amdgpu_waves_per_eu(2)))
void int4_decode_kernel(const Int4DecodeParams a) {
    __shared__ Int4Smem sm;
    const int H = a.H, NR = a.NR;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int g = lane >> 4, c = lane & 15;
    const int u = xcd_major(blockIdx.x, gridDim.x);
    const int w = u / H, h = u - w * H;          // this group's run and head

    // ---- its run of the head's page list, and the sequence that run starts in ----
    // (a sequence of no tokens counts one page, which nobody reads: its group
    // stores the zeros)
    auto units_of = [&](int len) {
        int p = len > 0 ? (len + PAGE - 1) / PAGE : 1;
        return p < a.max_pages ? p : a.max_pages;
    };
    const int per_lane = (a.B + WAVE - 1) / WAVE;
    const int b0 = lane * per_lane < a.B ? lane * per_lane : a.B;
    const int b1 = b0 + per_lane < a.B ? b0 + per_lane : a.B;
    int mine = 0;
    for (int i = b0; i < b1; ++i) mine += units_of(a.lens[i]);
    const int incl = wave_incl_scan(mine, lane);
    const int T = __builtin_amdgcn_readlane(incl, WAVE - 1);
    int per = (T + a.groups - 1) / a.groups;
    per = per > I4_MIN_PAGES ? per : I4_MIN_PAGES;
    if ((int64_t)w * per >= T) return;           // (every wave alike, before any barrier)
    const int u0 = w * per, u1 = T - u0 < per ? T : u0 + per;
    int b = 0, P = 0, len = 0;
    {
        int pos = incl - mine;
        const bool holds = u0 >= pos && u0 < incl;
        int fb = 0, fp = 0, fl = 0;
        if (holds) {
            for (int i = b0; i < b1; ++i) {
                const int li = a.lens[i], n = units_of(li);
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

    const float scale_log2 = a.scale * I4_LOG2E;
    const int64_t rec = (int64_t)NR * HEAD_DIM + 2 * MAX_NREP;
    int at = u0;
    while (true) {
        const int n = units_of(len);
        const int s0 = at - P, s1 = u1 - P < n ? u1 - P : n;      // this run's pages of it

        // query rows (past n_rep: row 0, never stored), channels 32 j + 8 g + (0..7)
        // in the order of the code pairs
        h8 q[4];
        {
            const half_t* row = a.q + (int64_t)b * a.sq_b + (int64_t)h * a.sq_h +
                                (int64_t)(c < NR ? c : 0) * a.sq_r + 8 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const h8 t = *(const h8*)(row + 32 * j);
                q[j] = (h8){t[0], t[4], t[1], t[5], t[2], t[6], t[3], t[7]};
            }
        }
        const int32_t* trow = a.tables + (int64_t)b * a.st_b;
        const int pages = len > 0 ? n : 0;
        // the wave's pages s0 + wv, + NW, ...; lane i holds the block of its
        // (base + i)-th (-1: none, or outside the pool)
        int base = 0, blk_of = -1;
        auto fill = [&](int from) {
            base = from;
            const int64_t pg = s0 + wv + (int64_t)(from + lane) * I4_NW;
            int t = -1;
            if (pg < s1 && pg < pages) t = trow[pg];
            blk_of = t >= 0 && t < a.p.num_blocks ? t : -1;
        };
        fill(0);

        Int4State st;
#pragma unroll
        for (int t = 0; t < 8; ++t) st.acc[t] = (f4){0.f, 0.f, 0.f, 0.f};
        st.m = neg_inf();
        st.l = 0.f;
        const int count = s0 + wv < s1 ? (s1 - s0 - wv + I4_NW - 1) / I4_NW : 0;
        Int4Page page[2];
        int blk[2];
        blk[0] = __builtin_amdgcn_readlane(blk_of, 0);
        if (count > 0) int4_load(a, page[0], blk[0], h, g, c);
        for (int k = 0; k < count; k += 2) {
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                if (k + z >= count) break;
                const int nx = k + z + 1;
                if (nx < count) {
                    if (nx - base == WAVE) fill(nx);
                    blk[z ^ 1] = __builtin_amdgcn_readlane(blk_of, nx - base);
                    int4_load(a, page[z ^ 1], blk[z ^ 1], h, g, c);
                }
                const int pg = s0 + wv + (k + z) * I4_NW;
                int4_compute(page[z], st, q, pg * PAGE, blk[z] >= 0 ? len : 0, scale_log2, g);
            }
        }

        // ---- the waves' states merged in LDS ----
        const float lrow = group4_sum(st.l);
        if (c < NR) {
            if (g == 0) {
                sm.m[wv][c] = st.m;
                sm.l[wv][c] = lrow;
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
        const int d0 = 4 * (threadIdx.x % 32);
        float* record = a.work + ((int64_t)(2 * w + (s0 == 0 ? 1 : 0)) * H + h) * rec;
        half_t* orow = a.out + (int64_t)b * a.so_b + (int64_t)h * a.so_h + d0;
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
                for (int e = 0; e < 4; ++e) orow[(int64_t)r * a.so_r + e] = (half_t)(acc[e] * inv);
            } else {
                store_coherent(record + r * HEAD_DIM + d0, acc);
                if (d0 == 0) store_coherent(record + NR * HEAD_DIM + 2 * r, mg, lt);
            }
        }
        if (!whole) {
            // ---- the last of the sequence's groups merges their records ----
            const int first = P / per, last = (P + n - 1) / per;
            int32_t* counter = a.counters + ((int64_t)first * H + h) * I4_COUNTER_STRIDE;
            handoff_release();
            __syncthreads();
            if (threadIdx.x == 0)
                sm.is_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT) == last - first;
            __syncthreads();
            if (sm.is_last) {
                for (int r = threadIdx.x / 32; r < NR; r += I4_NW * 2) {
                    float mg = neg_inf(), lt = 0.f;
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
                    for (int k = first; k <= last; ++k) {
                        const float* rk = a.work + ((int64_t)(2 * k + (k == first ? 1 : 0)) * H + h) * rec;
                        const float mk = load_coherent(rk + NR * HEAD_DIM + 2 * r);
                        const float lk = load_coherent(rk + NR * HEAD_DIM + 2 * r + 1);
                        f4 ak;
#pragma unroll
                        for (int e = 0; e < 4; ++e) ak[e] = load_coherent(rk + r * HEAD_DIM + d0 + e);
                        const float mn = fmaxf(mg, mk);
                        const bool none = mn == neg_inf();
                        const float wa = none ? 0.f : fast_exp2(mg - mn);
                        const float wb = none ? 0.f : fast_exp2(mk - mn);
                        lt = lt * wa + lk * wb;
                        acc = acc * wa + ak * wb;
                        mg = mn;
                    }
                    const float inv = 1.f / fmaxf(lt, 1e-20f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) orow[(int64_t)r * a.so_r + e] = (half_t)(acc[e] * inv);
                }
                if (threadIdx.x == 0)
                    __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        at = P + n;
        if (at >= u1) return;
        ++b;
        P = at;
        len = a.lens[b];
        __syncthreads();                 // the merge's LDS reads end before the next states
    }
}

int int4_groups(int batch, int kv_heads, int64_t pages_bound) {
    int64_t most = I4_RESIDENT / kv_heads;
    most = most > 1 ? most : 1;
    const int64_t need = (batch * pages_bound + I4_MIN_PAGES - 1) / I4_MIN_PAGES;
    return (int)(need < most ? (need > 1 ? need : 1) : most);
}

hipError_t launch_int4_decode(const Int4DecodeParams& a, hipStream_t stream) {
    hipLaunchKernelGGL(int4_decode_kernel, dim3(a.groups * a.H), dim3(WAVE * I4_NW), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ls

// Log probabilities of given tokens, each row's entropy and its most likely tokens,
// from fp16 or fp32 logits, in one launch that reads them once.
//
//   M = max x, Z = sum exp(x - M), E = sum exp(x - M) (x - M)
//   logprob(t) = x_t - M - log Z, entropy = log Z - E / Z
//
// with 2^x for the exponentials and fp32 sums.  A row is split over workgroups of 256 threads that hold their part in
// registers; each thread sums against its own maximum, so nothing is exchanged before
// the sums are made.  Bound by the logits' read and by a quarter-rate exponential a
// logit, about alike.
//
// Top k of a part: the k-th largest of a wave's 64 thread maxima bounds the k-th largest
// logit from below, so the logits at or over the largest such bound hold the k best;
// they are few, go to LDS and are ranked by counting.  Ranks compare (value, lower
// index), all different, so ties need no rule of their own; where ties leave more
// logits at the bound than LDS takes, the bound is made of such pairs.  The last of a
// row's groups to arrive merges the parts.

#include <type_traits>

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / WAVE;
// Logits a thread holds: 64, or 16 where that leaves more than half of the CUs idle.
constexpr int LP_LONG = 64, LP_SHORT = 16;
constexpr int LP_POOL = LOGPROB_MAX_TOP * LP_LONG;
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

// Unsigned order of a float's value (-0 as 0, NaN largest), 0 for no value.
__device__ __forceinline__ uint32_t value_key(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == 0xFFFFFFFFu) return __builtin_nanf("");
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct LogprobSmem {
    float red[3][LP_WAVES];
    uint32_t wave_bound[LP_WAVES];
    uint64_t best[LP_THREADS];
    uint64_t pool[LP_POOL];
    uint64_t kept[LOGPROB_MAX_TOP];
    uint64_t bound;
    int count;
    int is_last;
};

__device__ __forceinline__ float wave_max_all(float v) {
    const LanePair p = swap32(half_max(v));
    return fmaxf(p.a, p.b);
}

// Z and E against the maximum m; differences in log2 units (of values,
// not of scaled ones: a type's lowest value times log2 e need not be finite, and a
// large maximum's rounding would be in every difference).
struct Sums {
    float m, z, e;
    // Against `to`, which is finite; a maximum of -inf (nothing summed) weighs nothing.
    __device__ __forceinline__ void move(float to) {
        const float d = (m - to) * LP_LOG2E, w = m == neg_inf() ? 0.f : fast_exp2(d);
        // (z may be NaN, which stays)
        e = w == 0.f ? 0.f * z : w * (e + z * d);
        z *= w;
        m = to;
    }
};

// (m, z, e) of the lanes' sums, in every lane.
__device__ __forceinline__ Sums wave_sums(Sums s) {
    const float top = wave_max_all(s.m);
    s.move(top == neg_inf() ? 0.f : top);
    s.z = wave_sum_dpp(s.z);
    s.e = wave_sum_dpp(s.e);
    s.m = top;
    return s;
}

// Ranks the n entries of sm.pool; the k best go to sm.kept in order (0: none).
__device__ __forceinline__ void rank_pool(LogprobSmem& sm, int n, int k) {
    const int tid = threadIdx.x;
    if (tid < k) sm.kept[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += LP_THREADS) {
        const uint64_t key = sm.pool[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) r += sm.pool[j] > key ? 1 : 0;
        if (r < k) sm.kept[r] = key;
    }
    __syncthreads();
}

// The k-th largest of the wave's keys (0 where fewer than k lanes have one).
__device__ __forceinline__ uint32_t wave_kth(uint32_t key, int k) {
    uint32_t ans = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = ans | (1u << bit);
        if (__builtin_popcountll(__ballot(key >= cand)) >= k) ans = cand;
    }
    return ans;
}

template <bool F32, bool TOP, int HELD>
__global__ __launch_bounds__(LP_THREADS) void logprob_kernel(const LogprobParams a) {
    constexpr int VEC = F32 ? 4 : 8, CHUNKS = HELD / VEC, PART = LP_THREADS * HELD;
    using T = std::conditional_t<F32, float, half_t>;
    typedef T tv __attribute__((ext_vector_type(VEC)));
    __shared__ LogprobSmem sm;
    const int tid = threadIdx.x, lane = tid % WAVE, wv = tid / WAVE;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const T* xr = (const T*)a.x + (int64_t)row * a.sx;
    const int top = TOP ? a.top : 0;

    // Chunks lie on 16-byte boundaries: chunk q holds entries q VEC - off + (0..VEC);
    // entries outside the row are -inf.
    const int off = (int)(((uintptr_t)xr % 16) / sizeof(T));
    const int base = (part * (PART / VEC) + tid) * VEC - off;      // of the thread's first chunk
    constexpr int STEP = LP_THREADS * VEC;
    tv x[CHUNKS];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        const int i0 = base + k * STEP;
        if (i0 >= 0 && i0 + VEC <= a.n) {
            x[k] = stream_load((const tv*)(xr + i0));
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int i = i0 + v;
                x[k][v] = i >= 0 && i < a.n ? xr[i] : (T)neg_inf();
            }
        }
    }
    if (tid == 0) sm.count = 0;
    tv mx = x[0];
#pragma unroll
    for (int k = 1; k < CHUNKS; ++k) mx = __builtin_elementwise_max(mx, x[k]);
    float best = (float)mx[0];
#pragma unroll
    for (int v = 1; v < VEC; ++v) best = fmaxf(best, (float)mx[v]);

    Sums s = {best, 0.f, 0.f};
    const float mb = s.m == neg_inf() ? 0.f : s.m;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float d = ((float)x[k][v] - mb) * LP_LOG2E;
            const float p = fast_exp2(d);
            s.z += p;
            s.e = __builtin_fmaf(p, fmaxf(d, -1024.f), s.e);      // (0 for -inf)
        }
    s = wave_sums(s);
    if (lane == 0) {
        sm.red[0][wv] = s.m;
        sm.red[1][wv] = s.z;
        sm.red[2][wv] = s.e;
    }

    // the part's k best to sm.kept
    uint32_t tkey = 0;
    if (top > 0) {
        // (the maximum ignores NaN, which ranks first: any NaN makes the thread's key
        // the largest)
        bool nan = false, any = false;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int i0 = base + k * STEP;
            any = any || (i0 + VEC > 0 && i0 < a.n);
#pragma unroll
            for (int v = 0; v < VEC; ++v) nan = nan || x[k][v] != x[k][v];
        }
        tkey = nan ? 0xFFFFFFFFu : any ? value_key(best) : 0;
        const uint32_t kth = wave_kth(tkey, top);
        if (lane == 0) sm.wave_bound[wv] = kth;
    }
    __syncthreads();
    s = {sm.red[0][lane % LP_WAVES], sm.red[1][lane % LP_WAVES], sm.red[2][lane % LP_WAVES]};
    if (lane >= LP_WAVES) s = {neg_inf(), 0.f, 0.f};
    s = wave_sums(s);
    if (top > 0) {
        uint32_t bound = 1;
#pragma unroll
        for (int v = 0; v < LP_WAVES; ++v) bound = sm.wave_bound[v] > bound ? sm.wave_bound[v] : bound;
        auto collect = [&](uint64_t least) {
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const int i = base + k * STEP + v;
                    const uint64_t key = ((uint64_t)value_key((float)x[k][v]) << 32) | (uint32_t)~i;
                    if (key >= least && i >= 0 && i < a.n) {
                        const int at = atomicAdd(&sm.count, 1);
                        if (at < LP_POOL) sm.pool[at] = key;
                    }
                }
        };
        if (tkey >= bound) collect((uint64_t)bound << 32);
        __syncthreads();
        if (sm.count > LP_POOL) {
            // Ties: the bound as the k-th largest of the threads' best (value, index)
            // pairs.  Only the k threads whose best reaches it hold entries over it.
            uint64_t pair = 0;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const int i = base + k * STEP + v;
                    const uint64_t key = ((uint64_t)value_key((float)x[k][v]) << 32) | (uint32_t)~i;
                    if (i >= 0 && i < a.n && key > pair) pair = key;
                }
            sm.best[tid] = pair;
            __syncthreads();
            if (tid == 0) {
                sm.count = 0;
                sm.bound = 1;
            }
            int r = 0;
#pragma unroll 8
            for (int j = 0; j < LP_THREADS; ++j) r += sm.best[j] > pair ? 1 : 0;
            __syncthreads();
            if (pair != 0 && r == top - 1) sm.bound = pair;
            __syncthreads();
            if (pair >= sm.bound) collect(sm.bound);
            __syncthreads();
        }
        rank_pool(sm, sm.count, top);
    }

    if (a.parts > 1) {
        const int floats = logprob_record_floats(top);
        float* rec = a.part + ((int64_t)row * a.parts + part) * floats;
        auto put = [](float* p, float v) {
            __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        if (tid == 0) {
            put(rec, s.m);
            put(rec + 1, s.z);
            put(rec + 2, s.e);
        }
        if (tid < top)
            __hip_atomic_store((uint64_t*)(rec + 4) + tid, sm.kept[tid], __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        handoff_release();
        __syncthreads();
        if (tid == 0)
            sm.is_last = __hip_atomic_fetch_add(a.counters + row, 1, __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
        __syncthreads();
        if (!sm.is_last) return;
        if (tid == 0) __hip_atomic_store(a.counters + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const float* recs = a.part + (int64_t)row * a.parts * floats;
        // (every wave the same: a part a lane)
        s = {neg_inf(), 0.f, 0.f};
        for (int p0 = 0; p0 < a.parts; p0 += WAVE) {
            Sums t = {neg_inf(), 0.f, 0.f};
            if (p0 + lane < a.parts) {
                const float* rp = recs + (int64_t)(p0 + lane) * floats;
                t = {load_coherent(rp), load_coherent(rp + 1), load_coherent(rp + 2)};
            }
            t = wave_sums(t);
            const float m = fmaxf(s.m, t.m), to = m == neg_inf() ? 0.f : m;
            s.move(to);
            t.move(to);
            s = {m, s.z + t.z, s.e + t.e};
        }
        if (top > 0) {
            // rounds: the kept ones so far, then as many parts' as fit
            const int round = (LP_POOL - LOGPROB_MAX_TOP) / top;
            for (int p0 = 0; p0 < a.parts; p0 += round) {
                const int np = a.parts - p0 < round ? a.parts - p0 : round;
                const int had = p0 == 0 ? 0 : top;
                if (tid < had) sm.pool[tid] = sm.kept[tid];
                for (int i = tid; i < np * top; i += LP_THREADS)
                    sm.pool[had + i] = load_coherent(
                        (const uint64_t*)(recs + (int64_t)(p0 + i / top) * floats + 4) + i % top);
                __syncthreads();
                // (absent entries are 0 and never rank before a present one)
                rank_pool(sm, had + np * top, top);
            }
        }
    }

    // (a row of -inf only: m -inf, z 0)
    const float mr = s.m == neg_inf() ? 0.f : s.m;
    const float lz = __builtin_amdgcn_logf(s.z);                   // log2
    auto logp = [&](float v) {
        return v == neg_inf() && s.z == s.z ? neg_inf()
                                            : (v - mr) - lz * LP_LN2;
    };
    if (tid == 0) {
        const int64_t tok = a.tokens[(int64_t)row * a.s_tok];
        a.logprob[row] = tok >= 0 && tok < a.n ? logp((float)xr[tok]) : 0.f;
        a.entropy[row] = s.z == 0.f ? 0.f : (lz - s.e / s.z) * LP_LN2;
    }
    if (tid < top) {
        const uint64_t key = sm.kept[tid];
        a.top_val[(int64_t)row * top + tid] = logp(key_value((uint32_t)(key >> 32)));
        a.top_id[(int64_t)row * top + tid] = (uint32_t)~(uint32_t)key;
    }
}

// Logits a thread holds for these sizes.
static int held(int rows, int n) {
    const int64_t part = LP_THREADS * LP_LONG;
    return rows * ((n + 7 + part - 1) / part) <= 128 ? LP_SHORT : LP_LONG;
}

int logprob_parts(int rows, int n) {
    // (a row that does not start on 16 bytes takes up to 7 entries more)
    const int part = LP_THREADS * held(rows, n);
    return (n + 7 + part - 1) / part;
}

template <bool F32, bool TOP>
static void launch_held(const LogprobParams& a, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)a.rows * a.parts)), block(LP_THREADS);
    if (held(a.rows, a.n) == LP_SHORT)
        hipLaunchKernelGGL((logprob_kernel<F32, TOP, LP_SHORT>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((logprob_kernel<F32, TOP, LP_LONG>), grid, block, 0, stream, a);
}

hipError_t launch_token_logprobs(const LogprobParams& a, int fp32, hipStream_t stream) {
    if (fp32 && a.top) launch_held<true, true>(a, stream);
    else if (fp32) launch_held<true, false>(a, stream);
    else if (a.top) launch_held<false, true>(a, stream);
    else launch_held<false, false>(a, stream);
    return hipGetLastError();
}

}  // namespace ls

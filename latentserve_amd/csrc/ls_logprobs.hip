// Log probabilities of given tokens, each row's entropy and its most likely tokens,
// from fp16 or fp32 logits, in one launch that reads them once.
//
//   M = max x, Z = sum exp(x - M), E = sum exp(x - M) (x - M)
//   logprob(t) = x_t - M - log Z, entropy = log Z - E / Z
//
// A row is split over workgroups of 256 threads that hold their part in registers.
// Top k of a part: the k-th largest of the threads' best entries bounds the k-th
// largest entry from below, and only the threads whose best reaches it (k of
// them) can hold one of the k, so the entries at or over it are few and fit LDS;
// they are ranked by counting.  Entries are compared as (value, lower index), all
// different, so ties need no rule of their own.  The last of a row's groups to
// arrive merges the parts.

#include <type_traits>

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

constexpr int LP_THREADS = 256;
constexpr int LP_PER_THREAD = 64;                     // entries a thread holds
constexpr int LP_PART = LP_THREADS * LP_PER_THREAD;
constexpr int LP_POOL = LOGPROB_MAX_TOP * LP_PER_THREAD;    // entries at or over the bound, at most

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
__device__ __forceinline__ uint64_t entry_key(float x, int i) {
    return ((uint64_t)value_key(x) << 32) | (uint32_t)~i;
}

struct LogprobSmem {
    float red[3][LP_THREADS / WAVE];
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

// Ranks the n entries of sm.pool; the k best go to sm.kept in order (0: none).
__device__ __forceinline__ void rank_pool(LogprobSmem& sm, int n, int k) {
    const int tid = threadIdx.x;
    if (tid < k) sm.kept[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += LP_THREADS) {
        const uint64_t key = sm.pool[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += sm.pool[j] > key ? 1 : 0;
        if (r < k) sm.kept[r] = key;
    }
    __syncthreads();
}

template <bool F32>
__global__ __launch_bounds__(LP_THREADS) void logprob_kernel(const LogprobParams a) {
    constexpr int VEC = F32 ? 4 : 8, CHUNKS = LP_PER_THREAD / VEC;
    using T = std::conditional_t<F32, float, half_t>;
    __shared__ LogprobSmem sm;
    const int tid = threadIdx.x, lane = tid % WAVE, wv = tid / WAVE;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const T* xr = (const T*)a.x + (int64_t)row * a.sx;
    const int top = a.top;

    // Chunks lie on 16-byte boundaries: chunk q holds entries q VEC - off + (0..VEC).
    const int off = (int)(((uintptr_t)xr % 16) / sizeof(T));
    float x[CHUNKS][VEC];
    int first[CHUNKS];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        const int i0 = (part * (LP_PART / VEC) + k * LP_THREADS + tid) * VEC - off;
        first[k] = i0;
        if (i0 >= 0 && i0 + VEC <= a.n) {
            const u4 t = stream_load((const u4*)(xr + i0));
            const T* e = (const T*)&t;
#pragma unroll
            for (int v = 0; v < VEC; ++v) x[k][v] = (float)e[v];
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int i = i0 + v;
                x[k][v] = i >= 0 && i < a.n ? (float)xr[i] : neg_inf();
            }
        }
    }
    float m = neg_inf();
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) m = fmaxf(m, x[k][v]);
    m = wave_max_all(m);
    if (lane == 0) sm.red[0][wv] = m;
    if (tid == 0) sm.count = 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < LP_THREADS / WAVE; ++v) m = fmaxf(m, sm.red[0][v]);
    const float mb = m == neg_inf() ? 0.f : m;
    float z = 0.f, e = 0.f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float d = x[k][v] - mb;
            const float p = __expf(d);
            z += p;
            e += p == 0.f ? 0.f : p * d;
        }
    z = wave_sum_dpp(z);
    e = wave_sum_dpp(e);
    if (lane == 0) {
        sm.red[1][wv] = z;
        sm.red[2][wv] = e;
    }

    if (top > 0) {
        uint64_t best = 0;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int i = first[k] + v;
                const uint64_t key = i >= 0 && i < a.n ? entry_key(x[k][v], i) : 0;
                best = key > best ? key : best;
            }
        sm.best[tid] = best;
        if (tid == 0) sm.bound = 1;              // fewer than k threads with entries: all of them
        __syncthreads();
        int r = 0;
        for (int j = 0; j < LP_THREADS; ++j) r += sm.best[j] > best ? 1 : 0;
        if (best != 0 && r == top - 1) sm.bound = best;
        __syncthreads();
        const uint64_t bound = sm.bound;
        if (best >= bound) {
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const int i = first[k] + v;
                    const uint64_t key = i >= 0 && i < a.n ? entry_key(x[k][v], i) : 0;
                    if (key >= bound) sm.pool[atomicAdd(&sm.count, 1)] = key;
                }
        }
        __syncthreads();
        rank_pool(sm, sm.count, top);
    } else {
        __syncthreads();
    }
    z = e = 0.f;
#pragma unroll
    for (int v = 0; v < LP_THREADS / WAVE; ++v) {
        z += sm.red[1][v];
        e += sm.red[2][v];
    }

    if (a.parts > 1) {
        const int floats = logprob_record_floats(top);
        float* rec = a.part + ((int64_t)row * a.parts + part) * floats;
        auto put = [](float* p, float v) {
            __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        if (tid == 0) {
            put(rec, m);
            put(rec + 1, z);
            put(rec + 2, e);
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
        m = neg_inf();
        for (int p = 0; p < a.parts; ++p) m = fmaxf(m, load_coherent(recs + (int64_t)p * floats));
        const float mr = m == neg_inf() ? 0.f : m;
        z = e = 0.f;
        for (int p = 0; p < a.parts; ++p) {
            const float* rp = recs + (int64_t)p * floats;
            const float mp = load_coherent(rp), zp = load_coherent(rp + 1);
            const float d = mp - mr, wt = __expf(d);
            // sum p (x - m): shifted to the row's maximum
            z += zp * wt;
            e += wt == 0.f ? 0.f : wt * (load_coherent(rp + 2) + zp * d);
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

    const float lz = __logf(z);
    if (tid == 0) {
        const int64_t tok = a.tokens[(int64_t)row * a.s_tok];
        float lp = 0.f;
        if (tok >= 0 && tok < a.n) {
            const float xt = (float)xr[tok];
            lp = xt == neg_inf() ? neg_inf() : (xt - m) - lz;
        }
        a.logprob[row] = lp;
        a.entropy[row] = m == neg_inf() && z == 0.f ? 0.f : lz - e / z;
    }
    if (tid < top) {
        const uint64_t key = sm.kept[tid];
        const float xv = key_value((uint32_t)(key >> 32));
        a.top_val[(int64_t)row * top + tid] = xv == neg_inf() ? neg_inf() : (xv - m) - lz;
        a.top_id[(int64_t)row * top + tid] = (uint32_t)~(uint32_t)key;
    }
}

int logprob_parts(int rows, int n, int fp32) {
    (void)rows;
    (void)fp32;
    // (a row that does not start on 16 bytes takes up to 7 entries more)
    return (n + 7 + LP_PART - 1) / LP_PART;
}

hipError_t launch_token_logprobs(const LogprobParams& a, int fp32, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)a.rows * a.parts)), block(LP_THREADS);
    if (fp32) hipLaunchKernelGGL(logprob_kernel<true>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(logprob_kernel<false>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace ls

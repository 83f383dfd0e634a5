// Log probabilities of given tokens, each row's entropy and its most likely tokens,
// from fp16 or fp32 logits, in one launch that reads them once.
//
//   M = max x, Z = sum exp(x - M), E = sum exp(x - M) (x - M)
//   logprob(t) = x_t - M - log Z, entropy = log Z - E / Z
//
// with 2^x for the exponentials and fp32 sums.  A row is split over workgroups of 256
// threads that hold their part in registers (one read serves the maximum, the sums and
// the alternatives); each thread sums against its own maximum, so nothing is exchanged
// before the sums are made.  Without alternatives a large call streams instead.
//
// 1021 fp16 rows of 151936: 58 us, 5.3 TB/s; bound by the read (a plain one of as many bytes
// runs at 7.0).
// 16 rows with 20 alternatives: 12.0 us (0.9 us of bytes), 1 row without 4.4 us: bound by
// what each group does once, in turn (load, two exchanges, the ranking, the hand-over to
// the row's last group and its merge).
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

// (a maximum's product with log2 e is rounded once and used as that value everywhere)
#pragma clang fp contract(off)

namespace ls {

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / WAVE;
// Logits a thread holds: 64, or 16 where that makes at most LP_FEW groups, a quarter of the
// CUs (us with 16 / 64, 20 alternatives: 1 row of 152K 10.0 / 11.6, 4 rows 11.1 / 11.7, 8 rows
// 13.1 / 11.9; 32 rows of 32K 10.1 / 10.6, 64 rows 11.6 / 10.8).
constexpr int LP_LONG = 64, LP_SHORT = 16, LP_FEW = 64;
// Streaming groups a call aims at: two a CU (us at 512 / 1024 / 2048, 152K logits a row: 1021
// rows 57 / 61 / 62, 600 rows 39 / 40 / -, 300 rows 24 / 24 / -).
constexpr int LP_GROUPS = 512;
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

// Keys of fp16 values differ only above these bits, which are 0, or all 1 in negative ones:
// a bound without them lies at most one value lower.
template <bool F32>
constexpr int LOW_BITS = F32 ? 0 : 13;

template <bool TOP>
struct LogprobSmem {
    float red[3][LP_WAVES];
    uint32_t wave_bound[LP_WAVES];
    uint64_t best[TOP ? LP_THREADS : 1];
    uint64_t pool[TOP ? LP_POOL : 1];
    uint64_t kept[TOP ? LOGPROB_MAX_TOP : 1];
    uint64_t bound;
    int count;
    int is_last;
};

__device__ __forceinline__ float wave_max_all(float v) {
    const LanePair p = swap32(half_max(v));
    return fmaxf(p.a, p.b);
}

// Z and E against a maximum m, differences in log2 units.  fp16 logits: m itself is in log2
// units, so that a difference is one fused multiply-add (the rounding of m log2 e is in
// every difference alike, the results' too, and cancels).  fp32: m is a logit, since a
// logit times log2 e need not be finite (the type's lowest value, a mask).
template <bool F32>
struct Sums {
    float m, z, e;
    static __device__ __forceinline__ float ref(float x) { return F32 ? x : x * LP_LOG2E; }
    static __device__ __forceinline__ float diff(float x, float m) {
        return F32 ? (x - m) * LP_LOG2E : __builtin_fmaf(x, LP_LOG2E, -m);
    }
    // Against `to`, which is finite; a maximum of -inf (nothing summed) weighs nothing.
    __device__ __forceinline__ void move(float to) {
        const float d = F32 ? (m - to) * LP_LOG2E : m - to;
        const float w = m == neg_inf() ? 0.f : fast_exp2(d);
        // (z may be NaN, which stays)
        e = w == 0.f ? 0.f * z : w * (e + z * d);
        z *= w;
        m = to;
    }
    // A logit against m (finite).
    __device__ __forceinline__ void add(float x) {
        const float d = diff(x, m);
        const float p = fast_exp2(d);
        z += p;
        e = __builtin_fmaf(p, fmaxf(d, -1024.f), e);      // (0 for -inf)
    }
};

// (m, z, e) of the lanes' sums, in every lane.
template <bool F32>
__device__ __forceinline__ Sums<F32> wave_sums(Sums<F32> s) {
    const float top = wave_max_all(s.m);
    s.move(top == neg_inf() ? 0.f : top);
    s.z = wave_sum_dpp(s.z);
    s.e = wave_sum_dpp(s.e);
    s.m = top;
    return s;
}

// A group's sums, in every lane, from its waves'.
template <bool F32, class Smem>
__device__ __forceinline__ Sums<F32> group_sums(Smem& sm, Sums<F32> s) {
    const int lane = threadIdx.x % WAVE, wv = threadIdx.x / WAVE;
    s = wave_sums(s);
    if (lane == 0) {
        sm.red[0][wv] = s.m;
        sm.red[1][wv] = s.z;
        sm.red[2][wv] = s.e;
    }
    __syncthreads();
    const int v = lane % LP_WAVES;
    s = {sm.red[0][v], sm.red[1][v], sm.red[2][v]};
    if (lane >= LP_WAVES) s = {neg_inf(), 0.f, 0.f};
    return wave_sums(s);
}

// The k-th largest of the wave's keys (0 where fewer than k lanes have one), its bits
// below LOW left 0.
template <int LOW>
__device__ __forceinline__ uint32_t wave_kth(uint32_t key, int k) {
    uint32_t ans = 0;
#pragma unroll
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t cand = ans | (1u << bit);
        if (__builtin_popcountll(__ballot(key >= cand)) >= k) ans = cand;
    }
    return ans;
}

// The largest of the waves' k-th largest keys, at least 1: no more than the k-th
// largest of all.  (Two barriers; sm.count is 0 after it.)
template <int LOW>
__device__ __forceinline__ uint32_t group_bound(LogprobSmem<true>& sm, uint32_t key, int k) {
    const uint32_t kth = wave_kth<LOW>(key, k);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) sm.wave_bound[threadIdx.x / WAVE] = kth;
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    uint32_t bound = 1;
#pragma unroll
    for (int v = 0; v < LP_WAVES; ++v) bound = sm.wave_bound[v] > bound ? sm.wave_bound[v] : bound;
    return bound;
}

// The k best of the n entries of sm.pool go to sm.kept in order (0: none), ranked by
// counting after all but a few have been dropped.
template <int LOW>
__device__ __forceinline__ void rank_pool(LogprobSmem<true>& sm, int n, int k) {
    const int tid = threadIdx.x;
    const uint64_t* list = sm.pool;
    if (n > WAVE) {
        uint32_t best = 0;
        for (int i = tid; i < n; i += LP_THREADS) {
            const uint32_t key = (uint32_t)(sm.pool[i] >> 32);
            best = key > best ? key : best;
        }
        const uint32_t bound = group_bound<LOW>(sm, best, k);
        for (int i = tid; i < n; i += LP_THREADS) {
            const uint64_t key = sm.pool[i];
            if ((uint32_t)(key >> 32) >= bound) {
                const int at = atomicAdd(&sm.count, 1);
                if (at < LP_THREADS) sm.best[at] = key;
            }
        }
        __syncthreads();
        if (sm.count <= LP_THREADS) {
            list = sm.best;
            n = sm.count;
        }
    }
    if (tid < k) sm.kept[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += LP_THREADS) {
        const uint64_t key = list[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) r += list[j] > key ? 1 : 0;
        if (r < k) sm.kept[r] = key;
    }
    __syncthreads();
}

// A part's sums s (in every lane), and its k best in sm.kept, to the row's results: at
// once, or by the last of the row's groups to arrive.
template <bool TOP, bool F32, class T>
__device__ __forceinline__ void finish(const LogprobParams& a, LogprobSmem<TOP>& sm, Sums<F32> s,
                                       const T* xr, int row, int part) {
    const int tid = threadIdx.x, lane = tid % WAVE, top = TOP ? a.top : 0;
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
        if (TOP && tid < top)
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
        // (every wave the same: a part a lane; the first ones requested ahead of the
        // entries)
        auto sums_of = [&](int p) {
            Sums<F32> t = {neg_inf(), 0.f, 0.f};
            if (p < a.parts) {
                const float* rp = recs + (int64_t)p * floats;
                t = {load_coherent(rp), load_coherent(rp + 1), load_coherent(rp + 2)};
            }
            return t;
        };
        s = sums_of(lane);
        if constexpr (TOP) {
            // rounds: the kept ones so far, then as many parts' as fit
            const int round = (LP_POOL - LOGPROB_MAX_TOP) / top;
            for (int p0 = 0; p0 < a.parts; p0 += round) {
                const int np = a.parts - p0 < round ? a.parts - p0 : round;
                const int had = p0 == 0 ? 0 : top;
                if (tid < had) sm.pool[tid] = sm.kept[tid];
                // (every part's best, then every part's second, ...: a wave's entries are
                // alike in rank, and the first wave's bound is a good one)
                for (int i = tid; i < np * top; i += LP_THREADS)
                    sm.pool[had + i] = load_coherent(
                        (const uint64_t*)(recs + (int64_t)(p0 + i % np) * floats + 4) + i / np);
                __syncthreads();
                // (absent entries are 0 and never rank before a present one)
                rank_pool<LOW_BITS<F32>>(sm, had + np * top, top);
            }
        }
        s = wave_sums(s);
        for (int p0 = WAVE; p0 < a.parts; p0 += WAVE) {
            Sums<F32> t = wave_sums(sums_of(p0 + lane));
            const float m = fmaxf(s.m, t.m), to = m == neg_inf() ? 0.f : m;
            s.move(to);
            t.move(to);
            s = {m, s.z + t.z, s.e + t.e};
        }
    }

    // (a row of -inf only: m -inf, z 0)
    const float mr = s.m == neg_inf() ? 0.f : s.m;
    const float lz = __builtin_amdgcn_logf(s.z);                   // log2
    auto logp = [&](float v) {
        if (v == neg_inf() && s.z == s.z) return neg_inf();
        return F32 ? (v - mr) - lz * LP_LN2 : (Sums<F32>::diff(v, mr) - lz) * LP_LN2;
    };
    if (tid == 0) {
        const int64_t tok = a.tokens[(int64_t)row * a.s_tok];
        a.logprob[row] = tok >= 0 && tok < a.n ? logp((float)xr[tok]) : 0.f;
        a.entropy[row] = s.z == 0.f ? 0.f : (lz - s.e / s.z) * LP_LN2;
    }
    if (TOP && tid < top) {
        const uint64_t key = sm.kept[tid];
        a.top_val[(int64_t)row * top + tid] = logp(key_value((uint32_t)(key >> 32)));
        a.top_id[(int64_t)row * top + tid] = (uint32_t)~(uint32_t)key;
    }
}

template <bool F32, bool TOP, int HELD>
__global__ __launch_bounds__(LP_THREADS) void logprob_kernel(const LogprobParams a) {
    constexpr int VEC = F32 ? 4 : 8, CHUNKS = HELD / VEC, PART = LP_THREADS * HELD;
    using T = std::conditional_t<F32, float, half_t>;
    typedef T tv __attribute__((ext_vector_type(VEC)));
    __shared__ LogprobSmem<TOP> sm;
    const int tid = threadIdx.x;
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
    tv mx = x[0];
#pragma unroll
    for (int k = 1; k < CHUNKS; ++k) mx = __builtin_elementwise_max(mx, x[k]);
    float best = (float)mx[0];
#pragma unroll
    for (int v = 1; v < VEC; ++v) best = fmaxf(best, (float)mx[v]);

    const float ref = Sums<F32>::ref(best);
    Sums<F32> s = {ref == neg_inf() ? 0.f : ref, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) s.add((float)x[k][v]);
    s.m = ref;

    // (the maximum ignores NaN, which ranks first: a thread whose sum is NaN, by one or by
    // an infinity, counts as holding the largest, a bound made of such threads takes in
    // all)
    const bool nan = s.z != s.z;
    s = group_sums(sm, s);
    if constexpr (TOP) {
        bool any = false;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int i0 = base + k * STEP;
            any = any || (i0 + VEC > 0 && i0 < a.n);
        }
        const uint32_t mine = nan ? 0xFFFFFFFFu : any ? value_key(best) : 0;
        const uint32_t bound = group_bound<LOW_BITS<F32>>(sm, mine, top);
        // The entries at or over the bound to the pool (NaN among them; where the bound
        // stands for none, all): a thread counts its own, so it asks for its place once.
        if (mine >= bound) {
            const T value = (T)key_value(bound);         // (of one of the logits, or NaN)
            uint64_t hits = 0;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                const int i0 = base + k * STEP;
                uint32_t hit = 0;
#pragma unroll
                for (int v = 0; v < VEC; ++v) hit |= x[k][v] < value ? 0u : 1u << v;
                const int from = i0 < 0 ? -i0 : 0, to = a.n - i0 < VEC ? a.n - i0 : VEC;
                hit &= to > from ? (1u << to) - (1u << from) : 0u;
                hits |= (uint64_t)hit << (k * VEC);
            }
            int at = atomicAdd(&sm.count, __builtin_popcountll(hits));
            // (read again, from a cache: a register cannot be picked by a lane's number)
            for (; hits && at < LP_POOL; hits &= hits - 1, ++at) {
                const int j = __builtin_ctzll(hits);
                const uint32_t i = base + j / VEC * STEP + j % VEC;
                sm.pool[at] = ((uint64_t)value_key((float)xr[i]) << 32) | ~i;
            }
        }
        __syncthreads();
        if (sm.count > LP_POOL) {
            // Ties: the bound as the k-th largest of the threads' best (value, index)
            // pairs.  Only the k threads whose best reaches it hold entries over it.
            auto entry = [&](int k, int v) -> uint64_t {
                const int i = base + k * STEP + v;
                if (i < 0 || i >= a.n) return 0;
                return ((uint64_t)value_key((float)x[k][v]) << 32) | (uint32_t)~i;
            };
            uint64_t pair = 0;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) pair = entry(k, v) > pair ? entry(k, v) : pair;
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
            const uint64_t least = sm.bound;
            if (pair >= least)
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        if (entry(k, v) >= least) sm.pool[atomicAdd(&sm.count, 1)] = entry(k, v);
            __syncthreads();
        }
        rank_pool<LOW_BITS<F32>>(sm, sm.count, top);
    }
    finish<TOP, F32>(a, sm, s, xr, row, part);
}

// Many logits and no alternatives: a group streams its part, so there are few parts to
// hand over, each thread's sums moving along with its maximum.
constexpr int LP_AHEAD = 4;          // chunks a thread takes a step; the next ones on their way

template <bool F32>
__global__ __launch_bounds__(LP_THREADS) void logprob_stream_kernel(const LogprobParams a) {
    constexpr int VEC = F32 ? 4 : 8, STEP = LP_THREADS * VEC;
    using T = std::conditional_t<F32, float, half_t>;
    typedef T tv __attribute__((ext_vector_type(VEC)));
    __shared__ LogprobSmem<false> sm;
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const T* xr = (const T*)a.x + (int64_t)row * a.sx;
    const int off = (int)(((uintptr_t)xr % 16) / sizeof(T));
    const int lo = part * a.part_len - off, hi = lo + a.part_len < a.n ? lo + a.part_len : a.n;
    Sums<F32> s = {neg_inf(), 0.f, 0.f};
    auto add = [&](const tv (&x)[LP_AHEAD]) {
        tv mx = x[0];
#pragma unroll
        for (int k = 1; k < LP_AHEAD; ++k) mx = __builtin_elementwise_max(mx, x[k]);
        float best = (float)mx[0];
#pragma unroll
        for (int v = 1; v < VEC; ++v) best = fmaxf(best, (float)mx[v]);
        best = fmaxf(s.m, Sums<F32>::ref(best));
        const float to = best == neg_inf() ? 0.f : best;
        if (best != s.m) s.move(to);
        s.m = to;
#pragma unroll
        for (int k = 0; k < LP_AHEAD; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) s.add((float)x[k][v]);
        s.m = best;
    };
    tv x[2][LP_AHEAD];
    // a step that the row's start or the part's end cuts
    auto cut = [&](int from) {
#pragma unroll
        for (int k = 0; k < LP_AHEAD; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int i = from + tid * VEC + k * STEP + v;
                x[0][k][v] = i >= 0 && i < hi ? xr[i] : (T)neg_inf();
            }
        add(x[0]);
    };
    auto load = [&](tv (&to)[LP_AHEAD], int from) {
#pragma unroll
        for (int k = 0; k < LP_AHEAD; ++k)
            to[k] = stream_load((const tv*)(xr + from + tid * VEC + k * STEP));
    };
    constexpr int ALL = LP_AHEAD * STEP;
    int at = lo;
    if (at < 0) {
        cut(at);
        at += ALL;
    }
    if (at + ALL <= hi) {
        load(x[0], at);
        while (true) {
            const bool one = at + 2 * ALL <= hi;
            if (one) load(x[1], at + ALL);
            add(x[0]);
            at += ALL;
            if (!one) break;
            const bool two = at + 2 * ALL <= hi;
            if (two) load(x[0], at + ALL);
            add(x[1]);
            at += ALL;
            if (!two) break;
        }
    }
    if (at < hi) cut(at);
    finish<false, F32>(a, sm, group_sums(sm, s), xr, row, part);
}

// How a call is split: held parts of LP_THREADS times `held` logits, or (held 0) streamed
// ones of part_len.
struct LogprobPlan {
    int held, parts, part_len;
};
static LogprobPlan plan(int rows, int n, int top) {
    // (a row that does not start on 16 bytes takes up to 7 entries more)
    const int64_t all = (int64_t)n + 7;
    auto count = [&](int64_t len) { return (int)((all + len - 1) / len); };
    const int64_t longs = LP_THREADS * LP_LONG;
    if (rows * (int64_t)count(longs) <= LP_FEW)
        return {LP_SHORT, count(LP_THREADS * LP_SHORT), LP_THREADS * LP_SHORT};
    if (top) return {LP_LONG, count(longs), (int)longs};
    // none of less than a held part
    int64_t len = all / ((LP_GROUPS + rows - 1) / rows);
    len = (len + longs - 1) / longs * longs;
    return {0, count(len), (int)len};
}

int logprob_parts(int rows, int n, int top) { return plan(rows, n, top).parts; }

template <bool F32, bool TOP>
static void launch_held(const LogprobParams& a, int held, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)a.rows * a.parts)), block(LP_THREADS);
    if (held == LP_SHORT)
        hipLaunchKernelGGL((logprob_kernel<F32, TOP, LP_SHORT>), grid, block, 0, stream, a);
    else if constexpr (TOP)
        hipLaunchKernelGGL((logprob_kernel<F32, TOP, LP_LONG>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL(logprob_stream_kernel<F32>, grid, block, 0, stream, a);
}

hipError_t launch_token_logprobs(const LogprobParams& a, int fp32, hipStream_t stream) {
    const LogprobPlan p = plan(a.rows, a.n, a.top);
    LogprobParams d = a;
    d.part_len = p.part_len;
    if (fp32 && a.top) launch_held<true, true>(d, p.held, stream);
    else if (fp32) launch_held<true, false>(d, p.held, stream);
    else if (a.top) launch_held<false, true>(d, p.held, stream);
    else launch_held<false, false>(d, p.held, stream);
    return hipGetLastError();
}

}  // namespace ls

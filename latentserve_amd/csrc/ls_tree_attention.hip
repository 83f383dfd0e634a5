// Attention of a tree of drafted tokens over the paged fp16 cache.
//
// A sequence's N newest tokens are the nodes of a tree; node i, with n_rep query rows a
// KV head, sees the tokens before the tree and the nodes its mask names:
//   out = softmax(q K^T scale) V over what the row sees.
//
// All rows of a KV head share its keys, so the products are made transposed:
// S^T = K Q^T and O^T = V^T P^T (32x32x16 MFMA).  Then a lane holds one row (lane % 32)
// and, of each 32 keys, the 16 whose number has bit 2 equal to lane / 32: a row's maximum
// and sum are made inside a lane and one exchange with its other half, a rescale is one
// factor a lane, and the weights of 16 keys are already the B operand of the second
// product (whose k order is free as long as V's is the same).
//
// K and V go to LDS by direct loads, whole rows of 256 bytes (16 lanes a row): K's 16-byte
// piece p of key r at place p ^ (r % 16), V's 32-byte unit u of key r at u ^ (r % 8), so
// that neither the row reads of K nor the transposing reads of V meet in a bank.
#include "ls_common.h"
#include "ls_tree.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __fp16 g4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

namespace {

// A weight is 2^(x - m + TOP) with x - m <= LAZY: at most 2^15, which fp16 holds, and of
// full precision down to 2^-21 of the running maximum's.
constexpr float TREE_TOP = 7.f, TREE_LAZY = 8.f;

__device__ __forceinline__ f16v mfma3216(u4 a, u4 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

__device__ __forceinline__ void load_to_lds(const char* src, char* dst) {
    __builtin_amdgcn_global_load_lds(
        (const void __attribute__((address_space(1)))*)src,
        (void __attribute__((address_space(3)))*)dst, 16, 0, 0);
}

__device__ __forceinline__ u2 read_transposed(const char* p) {
    return __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((g4 __attribute__((address_space(3)))*)p));
}

// Where a lane reads a tile's K and V, in bytes (every other offset is a constant).
struct LanePlaces {
    int k[8], v[4];
};
__device__ __forceinline__ LanePlaces lane_places(int lane) {
    LanePlaces p;
    const int key = lane & 31, half = lane >> 5;
#pragma unroll
    for (int s = 0; s < 8; ++s) p.k[s] = key * 256 + 16 * ((2 * s + half) ^ (key & 15));
    const int quarter = lane >> 4, r = 4 * (quarter >> 1) + ((lane & 15) >> 2);
#pragma unroll
    for (int c = 0; c < 4; ++c) p.v[c] = r * 256 + 32 * ((2 * c + (quarter & 1)) ^ r) + 8 * (lane & 3);
    return p;
}

struct RowState {
    f16v acc[4];                          // O^T: channel 32 c + 8 (i / 4) + 4 half + i % 4
    float m, l;                           // running maximum (log2 units), this half's sum
};

__device__ __forceinline__ void clear(RowState& st) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.acc[c][i] = 0.f;
    st.m = neg_inf();
    st.l = 0.f;
}

// The 32 bits of what `row` sees of keys key0 .. key0 + 31 (bit: key - key0), for a tile
// that meets the tree or the end.  `ok`: keys that exist.
__device__ __forceinline__ uint32_t seen_bits(const TreeParams& a, const uint64_t* row_mask, int node,
                                              int64_t rel0, int nodes) {
    // keys of the context
    if (rel0 <= -32) return ~0u;
    uint32_t ctx = 0;
    int from = 0;                         // first node of the window
    if (rel0 < 0) {
        ctx = (1u << (int)(-rel0)) - 1;
        from = 0;
    } else {
        from = (int)(rel0 < TREE_MAX_NODES ? rel0 : TREE_MAX_NODES);
    }
    uint64_t w;
    if (row_mask) {
        const int i = from >> 6, s = from & 63;
        w = i < a.words ? row_mask[i] >> s : 0;
        if (s > 32 && i + 1 < a.words) w |= row_mask[i + 1] << (64 - s);
    } else {
        const int n = node + 1 - from;
        w = n <= 0 ? 0 : n >= 32 ? 0xFFFFFFFFull : (1ull << n) - 1;
    }
    const int left = nodes - from;        // nodes that exist, from the window's first
    uint32_t t = (uint32_t)w;
    if (left < 32) t &= left <= 0 ? 0u : (1u << left) - 1;
    return rel0 < 0 ? (t << (int)(-rel0)) | ctx : t;
}

// Scores of a tile of 32 KB keys for the wave's 32 rows.
template <int KB>
__device__ __forceinline__ void scores_of(const char* kt, const LanePlaces& at, const u4 (&q)[8],
                                          f16v (&s)[KB]) {
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[z][i] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int z = 0; z < KB; ++z)
            s[z] = mfma3216(*(const u4*)(kt + at.k[j] + z * 8192), q[j], s[z]);
}

template <int KB>
__device__ __forceinline__ void mask_scores(f16v (&s)[KB], const uint32_t (&bits)[KB], int half) {
#pragma unroll
    for (int z = 0; z < KB; ++z) {
        const uint32_t b = bits[z] >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[z][i] = (b >> (8 * (i / 4) + i % 4)) & 1 ? s[z][i] : neg_inf();
    }
}

// Softmax weights of the tile as fp16 pairs, the state's maximum and sum brought up to date.
template <int KB>
__device__ __forceinline__ void weights_of(const f16v (&s)[KB], RowState& st, float scale2,
                                           u4 (&p)[2 * KB]) {
    float top = neg_inf();
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[z][i]);
    const LanePair o = swap32(top);
    const float m_new = fmaxf(st.m, fmaxf(o.a, o.b) * scale2);
    // (wave-uniform; weights stay below 2^15 as long as nothing outgrows the maximum by more)
    if (__any(m_new > st.m + TREE_LAZY)) {
        const float alpha = fast_exp2(st.m - (m_new == neg_inf() ? 0.f : m_new));
        st.l *= alpha;
#pragma unroll
        for (int c = 0; c < 4; ++c) st.acc[c] *= alpha;
        st.m = m_new;
    }
    const float off = TREE_TOP - (st.m == neg_inf() ? 0.f : st.m);
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float w0 = fast_exp2(__builtin_fmaf(s[z][i], scale2, off));
            const float w1 = fast_exp2(__builtin_fmaf(s[z][i + 1], scale2, off));
            st.l += w0 + w1;
            const h2 w = {(half_t)w0, (half_t)w1};
            p[2 * z + i / 8][i / 2 % 4] = __builtin_bit_cast(uint32_t, w);
        }
}

// V^T of 16 keys (step j of the tile) and 32 channels (c).
__device__ __forceinline__ u4 values_of(const char* vt, const LanePlaces& at, int j, int c) {
    const u2 a = read_transposed(vt + at.v[c] + j * 4096);
    const u2 b = read_transposed(vt + at.v[c] + j * 4096 + 2048);
    return (u4){a.x, a.y, b.x, b.y};
}

template <int KB>
__device__ __forceinline__ void add_values(const char* vt, const LanePlaces& at, RowState& st,
                                           const u4 (&p)[2 * KB]) {
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) st.acc[c] = mfma3216(values_of(vt, at, j, c), p[j], st.acc[c]);
}

// Halves of a V operand's keys 16 j + 4 half + (0..3) and + 8 cleared where `keep` (bits of the
// 32 keys) has a 0.
__device__ __forceinline__ u4 keep_keys(u4 v, uint32_t keep, int j, int half) {
    const uint32_t b = keep >> (16 * (j & 1) + 4 * half);
    auto pair = [&](int i) {
        return ((b >> i) & 1 ? 0xFFFFu : 0u) | ((b >> (i + 1)) & 1 ? 0xFFFF0000u : 0u);
    };
    v.x &= pair(0);
    v.y &= pair(2);
    v.z &= pair(8);
    v.w &= pair(10);
    return v;
}
__device__ __forceinline__ bool finite(uint32_t w) {
    return (w & 0x7C00u) != 0x7C00u && (w & 0x7C000000u) != 0x7C000000u;
}

// The same for a 32-key block that meets the tree or the end.  bits: what the lane's row sees
// of it; live: the keys that exist (the same in every lane): other V rows count as zeros.
// A key that exists may be hidden from a row and hold an infinity or a NaN, which a
// weight of 0 does not remove: such a block's products are made a row at a time, of the
// keys that the row sees.
__device__ __forceinline__ void add_values_masked(const char* vt, const LanePlaces& at, RowState& st,
                                                  const u4 (&p)[2], uint32_t bits, uint32_t live,
                                                  int half) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const u4 v = keep_keys(values_of(vt, at, j, c), live, j, half);
            odd |= !(finite(v.x) && finite(v.y) && finite(v.z) && finite(v.w));
        }
    asm volatile("" ::: "memory");            // (read again below: not kept in registers)
    if (!__any(odd)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                st.acc[c] = mfma3216(keep_keys(values_of(vt, at, j, c), live, j, half), p[j], st.acc[c]);
        return;
    }
    const int row = __lane_id() & 31;
    for (int x = 0; x < 32; ++x) {
        const uint32_t seen = (uint32_t)__builtin_amdgcn_readlane((int)bits, x) & live;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            f16v y;
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                y = mfma3216(keep_keys(values_of(vt, at, j, c), seen, j, half), p[j], y);
#pragma unroll
            for (int i = 0; i < 16; ++i) st.acc[c][i] = row == x ? st.acc[c][i] + y[i] : st.acc[c][i];
        }
        asm volatile("" ::: "memory");
    }
}

// ---- the run of a group -------------------------------------------------------------

struct Unit {
    int b, h, start;                      // sequence, KV head, place of its first step
    int len, steps;
};

__device__ __forceinline__ int length_of(const TreeParams& a, int b) {
    const int n = a.lens[b];
    return n > 0 ? n : 0;
}
// Keys that the table covers, and the steps they take (one where there is none).
__device__ __forceinline__ int keys_of(const TreeParams& a, int len) {
    const int64_t most = (int64_t)a.max_pages * PAGE;
    return (int)(len < most ? len : most);
}
__device__ __forceinline__ int steps_of(const TreeParams& a, int len, int step_keys) {
    const int n = keys_of(a, len);
    return n > 0 ? (n - 1) / step_keys + 1 : 1;
}

// The total of all units' places, and (find) the unit that place u0 lies in.
__device__ __forceinline__ int total_places(const TreeParams& a, int step_keys, int lane) {
    int mine = 0;
    for (int b = lane; b < a.B; b += WAVE)
        mine += (steps_of(a, length_of(a, b), step_keys) + a.extra) * a.H;
    // (each half's lanes, then the halves; whole numbers below 2^31)
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) mine += __shfl_xor(mine, d);
    return __builtin_amdgcn_readfirstlane(mine);
}
__device__ __forceinline__ Unit find_unit(const TreeParams& a, int step_keys, int lane, int u0) {
    Unit u = {0, 0, 0, 0, 1};
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += WAVE) {
        const int b = b0 + lane;
        const int len = b < a.B ? length_of(a, b) : 0;
        const int n = b < a.B ? (steps_of(a, len, step_keys) + a.extra) * a.H : 0;
        int incl = n;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        const uint64_t hit = __ballot(b < a.B && u0 < before + incl);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            u.b = b0 + src;
            u.len = __builtin_amdgcn_readlane(len, src);
            u.steps = steps_of(a, u.len, step_keys);
            const int first = before + __builtin_amdgcn_readlane(incl - n, src);
            u.h = __builtin_amdgcn_readfirstlane((u0 - first) / (u.steps + a.extra));
            u.start = first + u.h * (u.steps + a.extra) + a.extra;
            return u;
        }
        before += __builtin_amdgcn_readlane(incl, WAVE - 1);
    }
    u.b = a.B;
    return u;
}
__device__ __forceinline__ void next_unit(const TreeParams& a, int step_keys, Unit& u) {
    u.start += u.steps + a.extra;
    if (++u.h < a.H) return;
    u.h = 0;
    if (++u.b >= a.B) return;
    u.len = length_of(a, u.b);
    u.steps = steps_of(a, u.len, step_keys);
}

// WR row groups of 32 rows by 8 / WR key groups.
// SCORES: the scores are stored too (one tile of rows).
template <int WR, int KB, bool SCORES>
__global__ __launch_bounds__(WAVE* TREE_NW) __attribute__((amdgpu_waves_per_eu(2)))
void tree_kernel(const TreeParams a) {
    constexpr int WK = TREE_NW / WR, KEYS = 32 * KB, STEP = KEYS * WK;
    constexpr int TILE = KEYS * 256;                       // bytes of K, and of V
    constexpr bool TWO = WR > 1;                           // two buffers; one wave's tile: one
    __shared__ __attribute__((aligned(1024))) char k0_[WK * TILE];
    __shared__ __attribute__((aligned(1024))) char v0_[WK * TILE];
    __shared__ __attribute__((aligned(1024))) char k1_[TWO ? WK * TILE : 16];
    __shared__ __attribute__((aligned(1024))) char v1_[TWO ? WK * TILE : 16];
    __shared__ float2 ml_[TREE_NW][32];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int rg = wave % WR, kg = wave / WR, half = lane >> 5;
    const int v = xcd_major(blockIdx.x, gridDim.x);
    const int g = __builtin_amdgcn_readfirstlane(v / a.row_tiles), rt = v - g * a.row_tiles;

    const int total = total_places(a, STEP, lane);
    const int per = __builtin_amdgcn_readfirstlane((total + a.groups - 1) / a.groups);
    const int64_t lo = (int64_t)g * per;
    if (lo >= total) return;
    const int u0 = (int)lo, u1 = total - u0 < per ? total : u0 + per;

    const LanePlaces at = lane_places(lane);
    const int R = a.N * a.NR;
    const int row = (rt * WR + rg) * 32 + (lane & 31);
    const bool is_row = row < R;
    const int node = is_row ? row / a.NR : 0, rep = is_row ? row - node * a.NR : 0;

    // this wave's part of a tile's loads: LOADS instructions of four rows, K and V each
    constexpr int LOADS = KEYS / 4 / WR;
    int src_k[LOADS], src_v[LOADS];                        // bytes inside a (page, head)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (rg * LOADS + i) * 4 + (lane >> 4), pp = lane & 15;
        src_k[i] = (int)((r & 15) * a.sp_t) + 16 * (pp ^ (r & 15));
        src_v[i] = (int)((r & 15) * a.sp_t) + 32 * ((pp >> 1) ^ (r & 7)) + 16 * (pp & 1);
    }

    Unit u = find_unit(a, STEP, lane, u0);
    for (; u.b < a.B && u.start - a.extra < u1; next_unit(a, STEP, u)) {
        const int s0 = u0 > u.start ? u0 - u.start : 0;
        const int s1 = u1 - u.start < u.steps ? u1 - u.start : u.steps;
        if (s0 >= s1) continue;                            // (only what starting counts as)
        const int keys = keys_of(a, u.len);
        const int ctx = u.len > a.N ? u.len - a.N : 0;
        int nodes = a.N;
        if (a.counts) {
            const int n = a.counts[u.b];
            nodes = n < nodes ? (n > 0 ? n : 0) : nodes;
        }
        nodes = nodes < u.len ? nodes : u.len;
        const bool seeing = is_row && node < nodes;
        const uint64_t* row_mask =
            a.masks && is_row ? a.masks + ((int64_t)u.b * a.N + node) * a.words : nullptr;
        const int32_t* table = a.tables + u.b * a.st_b;
        const int pages = (keys + PAGE - 1) / PAGE;

        u4 q[8];
        {
            const half_t* p = a.q + u.b * a.sq_b + node * a.sq_n + u.h * a.sq_h + rep * a.sq_r + 8 * half;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = is_row ? *(const u4*)(p + 16 * j) : (u4){0, 0, 0, 0};
        }
        RowState st;
        clear(st);

        // block of page `lane` of a step's tile, -1: none
        auto ids_of = [&](int step) {
            const int64_t page = ((int64_t)step * WK + kg) * (KEYS / PAGE) + lane;
            int id = -1;
            if (lane < KEYS / PAGE && page < pages) {
                id = table[page];
                if ((unsigned)id >= (unsigned)a.num_blocks) id = -1;
            }
            return id;
        };
        auto bad_of = [&](int ids) {
            return (uint32_t)__ballot(lane < KEYS / PAGE && ids < 0);
        };
        // a page outside the pool is read as zeros
        auto load = [&](int z, int ids, char* t) {
            constexpr int SAME = LOADS < 4 ? LOADS : 4;    // instructions of one page
#pragma unroll
            for (int i0 = 0; i0 < LOADS; i0 += SAME) {
                const int first = (rg * LOADS + i0) * 4;
                const int id = __builtin_amdgcn_readlane(ids, first / PAGE);
                if (id >= 0) {
                    const char* from = a.pool[z] + id * a.sp_b + u.h * a.sp_h;
#pragma unroll
                    for (int i = i0; i < i0 + SAME; ++i)
                        load_to_lds(from + (z ? src_v[i] : src_k[i]), t + (first + 4 * (i - i0)) * 256);
                } else {
#pragma unroll
                    for (int i = 0; i < SAME; ++i)
                        *(u4*)(t + (first + 4 * i) * 256 + lane * 16) = (u4){0, 0, 0, 0};
                }
            }
        };
        // a block's scores, in log2 units
        auto store_scores = [&](const f16v& s, int64_t k0) {
            if (!is_row) return;
            float* to = a.scores + ((int64_t)(u.b * a.H + u.h) * R + row) * a.score_len + k0 + 4 * half;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const f4 x = {s[4 * n] * a.scale2, s[4 * n + 1] * a.scale2, s[4 * n + 2] * a.scale2,
                              s[4 * n + 3] * a.scale2};
                *(f4*)(to + 8 * n) = x;
            }
        };
        // keys of the context only; bad: pages of the tile that are not there
        auto mask_pages = [&](f16v (&s)[KB], uint32_t bad) {
            uint32_t bits[KB];
#pragma unroll
            for (int z = 0; z < KB; ++z)
                bits[z] = ((bad >> (2 * z)) & 1 ? 0u : 0xFFFFu) |
                          ((bad >> (2 * z + 1)) & 1 ? 0u : 0xFFFF0000u);
            mask_scores<KB>(s, bits, half);
        };
        // a tile that meets the tree or the end, a block at a time
        auto compute_masked = [&](int step, uint32_t bad, const char* kt, const char* vt) {
            for (int z = 0; z < KB; ++z) {
                const int64_t k0 = ((int64_t)step * WK + kg) * KEYS + 32 * z;
                const int64_t left = (ctx + nodes < keys ? ctx + nodes : keys) - k0;
                if (left <= 0) return;
                uint32_t live = left >= 32 ? ~0u : (1u << (int)left) - 1;
                if ((bad >> (2 * z)) & 1) live &= 0xFFFF0000u;
                if ((bad >> (2 * z + 1)) & 1) live &= 0x0000FFFFu;
                const uint32_t bits[1] = {
                    seeing ? seen_bits(a, row_mask, node, k0 - ctx, nodes) & live : 0u};
                f16v s[1];
                u4 p[2];
                scores_of<1>(kt + z * 8192, at, q, s);
                mask_scores<1>(s, bits, half);
                if constexpr (SCORES) store_scores(s[0], k0);
                weights_of<1>(s, st, a.scale2, p);
                add_values_masked(vt + z * 8192, at, st, p, bits[0], live, half);
            }
        };

        char* const kt0 = k0_ + kg * TILE;
        char* const vt0 = v0_ + kg * TILE;
        // steps of the context alone, then the others
        const int sf = s1 < ctx / STEP ? s1 : (s0 > ctx / STEP ? s0 : ctx / STEP);
        int ids = ids_of(s0);
        if constexpr (TWO) {
            char* const kt1 = k1_ + kg * TILE;
            char* const vt1 = v1_ + kg * TILE;
            uint32_t bad = bad_of(ids);
            load(0, ids, kt0);
            load(1, ids, vt0);
            ids = s0 + 1 < s1 ? ids_of(s0 + 1) : -1;
            // a step's loads have come and everyone is done with the step before: the next
            // one's go out
            auto turn = [&](int step, char* kn, char* vn) {
                wait_vm_lds<0>();
                __syncthreads();
                const uint32_t now = bad;
                if (step + 1 < s1) {
                    bad = bad_of(ids);
                    load(0, ids, kn);
                    load(1, ids, vn);
                    if (step + 2 < s1) ids = ids_of(step + 2);
                }
                return now;
            };
            auto compute = [&](uint32_t now, const char* kt, const char* vt) {
                f16v s[KB];
                u4 p[2 * KB];
                scores_of<KB>(kt, at, q, s);
                if (now) mask_pages(s, now);
                weights_of<KB>(s, st, a.scale2, p);
                add_values<KB>(vt, at, st, p);
            };
            int step = s0;
            while (step < sf) {
                uint32_t now = turn(step, kt1, vt1);
                compute(now, kt0, vt0);
                if (++step >= sf) break;
                now = turn(step, kt0, vt0);
                compute(now, kt1, vt1);
                ++step;
            }
            for (; step < s1; ++step) {
                const bool odd = (step - s0) & 1;
                const uint32_t now = odd ? turn(step, kt0, vt0) : turn(step, kt1, vt1);
                compute_masked(step, now, odd ? kt1 : kt0, odd ? vt1 : vt0);
            }
        } else {
            // one buffer of a wave's own, K and V in turn: each is requested again as soon as
            // it has been read
            auto reads_done = [&] {
                __builtin_amdgcn_s_waitcnt(0xC07F);        // lgkmcnt 0
                asm volatile("" ::: "memory");
            };
            uint32_t bad = bad_of(ids);
            load(0, ids, kt0);
            load(1, ids, vt0);
            int step = s0;
            for (; step < sf; ++step) {
                const bool more = step + 1 < s1;
                int next = -1;
                if (more) next = ids_of(step + 1);
                wait_vm_lds<0>();
                f16v s[KB];
                u4 p[2 * KB];
                scores_of<KB>(kt0, at, q, s);
                if (bad) mask_pages(s, bad);
                reads_done();
                if (more) load(0, next, kt0);
                weights_of<KB>(s, st, a.scale2, p);
                add_values<KB>(vt0, at, st, p);
                reads_done();
                if (more) load(1, next, vt0);
                if constexpr (SCORES) store_scores(s[0], ((int64_t)step * WK + kg) * KEYS);
                ids = next;
                bad = bad_of(next);
            }
            for (; step < s1; ++step) {
                wait_vm_lds<0>();
                reads_done();
                compute_masked(step, bad, kt0, vt0);
                reads_done();
                if (step + 1 < s1) {
                    ids = ids_of(step + 1);
                    bad = bad_of(ids);
                    load(0, ids, kt0);
                    load(1, ids, vt0);
                }
            }
        }

        // ---- the key groups' results made one, then the output or a record ----
        const bool whole = s0 == 0 && s1 == u.steps;
        const LanePair lp = swap32(st.l);
        float l = lp.a + lp.b, m = st.m;
        constexpr int QUADS = 16 / WK;                     // of 16 channel quads, this wave's
        f4 y[QUADS];
        if constexpr (WK > 1) {
            // 16 KB a wave, over the tiles' arrays
            constexpr int PER = (TWO ? WK * TILE : WK * TILE) / 16384;
            auto place = [&](int w) -> char* {
                char* arr = w / PER == 0 ? k0_ : w / PER == 1 ? v0_ : w / PER == 2 ? k1_ : v1_;
                return arr + (w % PER) * 16384;
            };
            __syncthreads();
            char* mine = place(wave);
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                const f4 x = {st.acc[n / 4][4 * (n % 4)], st.acc[n / 4][4 * (n % 4) + 1],
                              st.acc[n / 4][4 * (n % 4) + 2], st.acc[n / 4][4 * (n % 4) + 3]};
                *(f4*)(mine + n * 1024 + lane * 16) = x;
            }
            if (half == 0) ml_[wave][lane] = make_float2(m, l);
            __syncthreads();
            float top = neg_inf();
#pragma unroll
            for (int k = 0; k < WK; ++k) top = fmaxf(top, ml_[k * WR + rg][lane & 31].x);
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < QUADS; ++n) y[n] = (f4){0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < WK; ++k) {
                const float2 o = ml_[k * WR + rg][lane & 31];
                const float w = o.x == neg_inf() ? 0.f : fast_exp2(o.x - top);
                // (a part that saw nothing holds zeros)
                sum += w * o.y;
                const char* from = place(k * WR + rg);
#pragma unroll
                for (int n = 0; n < QUADS; ++n)
                    y[n] += *(const f4*)(from + (kg * QUADS + n) * 1024 + lane * 16) * w;
            }
            m = top;
            l = sum;
            __syncthreads();                               // (before the next unit's loads)
        } else {
#pragma unroll
            for (int n = 0; n < QUADS; ++n)
                y[n] = (f4){st.acc[n / 4][4 * (n % 4)], st.acc[n / 4][4 * (n % 4) + 1],
                            st.acc[n / 4][4 * (n % 4) + 2], st.acc[n / 4][4 * (n % 4) + 3]};
            __syncthreads();
        }
        if (whole) {
            const float inv = seeing && l != 0.f ? 1.f / l : 0.f;
            if (is_row) {
                half_t* o = a.out + u.b * a.so_b + node * a.so_n + u.h * a.so_h + rep * a.so_r;
#pragma unroll
                for (int n = 0; n < QUADS; ++n) {
                    const int quad = kg * QUADS + n;
                    h4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = seeing ? (half_t)(y[n][e] * inv) : (half_t)0.f;
                    *(h4*)(o + 8 * quad + 4 * half) = x;
                }
                if (a.lse && kg == 0 && half == 0)
                    a.lse[((int64_t)(u.b * a.N + node) * a.H + u.h) * a.NR + rep] =
                        seeing && m != neg_inf()
                            ? (m - TREE_TOP + __builtin_amdgcn_logf(l)) * 0.69314718055994531f
                            : neg_inf();
            }
        } else {
            float* rec = a.work + ((((int64_t)g * 2 + (s0 == 0)) * a.row_tiles + rt) * WR + rg) * TREE_RECORD;
#pragma unroll
            for (int n = 0; n < QUADS; ++n) *(f4*)(rec + (kg * QUADS + n) * 256 + lane * 4) = y[n];
            if (kg == 0 && half == 0) *(float2*)(rec + 4096 + 2 * lane) = make_float2(m, l);
        }
        if (s0 == 0 && rt == 0 && threadIdx.x == 0)
            a.info[u.b * a.H + u.h] = make_int2(u.start / per, (u.start + u.steps - 1) / per);
    }
}

// Records of a unit made its output: a workgroup a (unit, 32 rows, CQ channel quads), its
// waves take the records in turn.
constexpr int COMBINE_NW = 8;
template <int CQ>
__global__ __launch_bounds__(WAVE* COMBINE_NW) void tree_combine_kernel(const TreeParams a, int wr) {
    __shared__ float sums[COMBINE_NW][CQ * 4 + 2][WAVE];
    const int parts = 16 / CQ, blocks = gridDim.y / parts;
    const int unit = blockIdx.x, rb = blockIdx.y / parts, part = blockIdx.y % parts;
    (void)blocks;
    const int2 gs = a.info[unit];
    if (gs.x == gs.y) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int rt = rb / wr, rg = rb % wr, count = gs.y - gs.x + 1;
    auto record = [&](int k) {
        const int64_t slot = (int64_t)(gs.x + k) * 2 + (k == 0);
        return a.work + ((slot * a.row_tiles + rt) * wr + rg) * TREE_RECORD;
    };
    float m = neg_inf(), l = 0.f;
    f4 y[CQ];
#pragma unroll
    for (int n = 0; n < CQ; ++n) y[n] = (f4){0.f, 0.f, 0.f, 0.f};
    for (int k = wave; k < count; k += COMBINE_NW) {
        const float* rec = record(k);
        const float2 o = *(const float2*)(rec + 4096 + 2 * (lane & 31));
        f4 x[CQ];
#pragma unroll
        for (int n = 0; n < CQ; ++n) x[n] = *(const f4*)(rec + (part * CQ + n) * 256 + lane * 4);
        const float top = fmaxf(m, o.x), use = top == neg_inf() ? 0.f : top;
        const float keep = fast_exp2(m - use), w = fast_exp2(o.x - use);
        l = l * keep + o.y * w;
#pragma unroll
        for (int n = 0; n < CQ; ++n) y[n] = y[n] * keep + x[n] * w;
        m = top;
    }
#pragma unroll
    for (int n = 0; n < CQ; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][4 * n + e][lane] = y[n][e];
    sums[wave][CQ * 4][lane] = m;
    sums[wave][CQ * 4 + 1][lane] = l;
    __syncthreads();
    // wave w finishes quad w
    if (wave >= CQ) return;
    float top = neg_inf(), total = 0.f;
    for (int w = 0; w < COMBINE_NW; ++w) top = fmaxf(top, sums[w][CQ * 4][lane]);
    const float use = top == neg_inf() ? 0.f : top;
    f4 z = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < COMBINE_NW; ++w) {
        const float f = fast_exp2(sums[w][CQ * 4][lane] - use);
        total += f * sums[w][CQ * 4 + 1][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += f * sums[w][4 * wave + e][lane];
    }
    const int row = rb * 32 + (lane & 31), half = lane >> 5;
    if (row >= a.N * a.NR) return;
    const int node = row / a.NR, rep = row - node * a.NR, b = unit / a.H, h = unit - b * a.H;
    int nodes = a.N;
    if (a.counts) {
        const int n = a.counts[b];
        nodes = n < nodes ? (n > 0 ? n : 0) : nodes;
    }
    const int len = length_of(a, b);
    nodes = nodes < len ? nodes : len;
    const bool seeing = node < nodes;
    const float inv = seeing && total != 0.f ? 1.f / total : 0.f;
    h4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = seeing ? (half_t)(z[e] * inv) : (half_t)0.f;
    *(h4*)(a.out + b * a.so_b + node * a.so_n + h * a.so_h + rep * a.so_r + 8 * (part * CQ + wave) +
           4 * half) = x;
    if (a.lse && part == 0 && wave == 0 && half == 0)
        a.lse[((int64_t)(b * a.N + node) * a.H + h) * a.NR + rep] =
            seeing && top != neg_inf()
                ? (top - TREE_TOP + __builtin_amdgcn_logf(total)) * 0.69314718055994531f
                : neg_inf();
}

template <int WR, int KB, bool SCORES>
hipError_t launch(const TreeParams& a, hipStream_t stream) {
    tree_kernel<WR, KB, SCORES>
        <<<dim3(a.groups * a.row_tiles), dim3(WAVE * TREE_NW), 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int blocks = (a.N * a.NR + 31) / 32;
    tree_combine_kernel<4><<<dim3(a.B * a.H, blocks * 4), dim3(WAVE * COMBINE_NW), 0, stream>>>(a, WR);
    return hipGetLastError();
}

}  // namespace

constexpr int TREE_CUS = 256;

TreeShape tree_shape(int batch, int kv_heads, int rows, int64_t keys_bound) {
    TreeShape s;
    s.wr = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
    s.kb = s.wr >= 4 ? 2 : 1;
    s.row_tiles = (rows + 32 * s.wr - 1) / (32 * s.wr);
    const int64_t step = 32 * s.kb * (TREE_NW / s.wr);
    const int64_t units = (int64_t)batch * kv_heads;
    const int64_t places = units * ((keys_bound + step - 1) / step + TREE_EXTRA);
    int64_t most = (TREE_CUS + s.row_tiles - 1) / s.row_tiles;
    const int64_t useful = (places + 1) / 2;               // (two steps a run at least)
    s.groups = (int)(most < useful ? most : useful);
    if (s.groups < 1) s.groups = 1;
    return s;
}

size_t tree_record_bytes(const TreeShape& s) {
    return (size_t)s.groups * 2 * s.row_tiles * s.wr * TREE_RECORD * sizeof(float);
}

hipError_t launch_tree_attention(const TreeParams& p, const TreeShape& s, hipStream_t stream) {
    TreeParams a = p;
    a.groups = s.groups;
    a.row_tiles = s.row_tiles;
    a.extra = TREE_EXTRA;
    if (a.scores) return launch<1, 1, true>(a, stream);
    switch (s.wr) {
        case 1: return launch<1, 1, false>(a, stream);
        case 2: return launch<2, 1, false>(a, stream);
        case 4: return launch<4, 2, false>(a, stream);
        default: return launch<8, 2, false>(a, stream);
    }
}

}  // namespace ls

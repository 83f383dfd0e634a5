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

// (buffer loads: after a global load to LDS the compiler waits for all LDS reads where it
// needs one)
typedef void __attribute__((address_space(3)))* lds_ptr;
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t off, int soff, char* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)dst, 16, off, soff, 0, 0);
}

__device__ __forceinline__ u2 read_transposed(const char* p) {
    return __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((g4 __attribute__((address_space(3)))*)p));
}

// Where a lane reads a tile's K and V, and what it loads of it, in bytes.  A tile starts
// on 1 KB and a row is 256 bytes, so a swizzled place inside a row is one exclusive or:
//   K of step j:         k ^ (32 j)        (piece 2 j + half of key lane % 32)
//   V of channels 32 c:  v ^ (64 c)        (see values_of)
//   loads i of a page:   (4 i + lane / 16) rows, pieces k_in ^ (64 i), v_in ^ (128 (i % 2))
struct LanePlaces {
    uint32_t k, v, k_in, v_in;
};
__device__ __forceinline__ LanePlaces lane_places(int lane) {
    LanePlaces p;
    const int key = lane & 31, half = lane >> 5, quarter = lane >> 4, pp = lane & 15;
    const int r = 4 * (quarter >> 1) + ((lane & 15) >> 2);
    p.k = key * 256 + 16 * (half ^ (key & 15));
    p.v = r * 256 + 32 * ((quarter & 1) ^ r) + 8 * (lane & 3);
    p.k_in = 16 * (pp ^ quarter);
    p.v_in = 32 * ((pp >> 1) ^ quarter) + 16 * (pp & 1);
    return p;
}
// The same value, made anew where it is used: what follows from it is computed there, not
// kept in registers through the loop.
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

struct RowState {
    f16v acc[4];                          // O^T: channel 32 c + 8 (i / 4) + 4 half + i % 4
    float m, l;                           // running maximum (log2 units), this half's sum
};

// Keeps the sums in one set of registers where branches join (the compiler otherwise takes them
// apart there and copies all 64, in every step).
__device__ __forceinline__ void pin(RowState& st) {
    asm volatile("" : "+v"(st.acc[0]), "+v"(st.acc[1]), "+v"(st.acc[2]), "+v"(st.acc[3]));
}

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

// What the scheduler is to keep: `first` LDS reads ahead, then one product and `per`
// reads in turn (left to itself it reads an operand and waits for it, product by product).
template <int FIRST, int PER, int READS, int PRODUCTS>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (FIRST + i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
}

// Scores of a tile of 32 KB keys for the wave's 32 rows.
template <int KB>
__device__ __forceinline__ void scores_of(const char* kt, const LanePlaces& at, const u4 (&q)[8],
                                          f16v (&s)[KB]) {
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[z][i] = 0.f;
    u4 k[8][KB];
    const uint32_t lane_k = here(at.k);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int z = 0; z < KB; ++z) k[j][z] = *(const u4*)(kt + (lane_k ^ (32 * j)) + z * 8192);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int z = 0; z < KB; ++z) s[z] = mfma3216(k[j][z], q[j], s[z]);
    reads_ahead<4, 1, 8 * KB, 8 * KB>();
    __builtin_amdgcn_sched_barrier(0);
}

template <int KB>
__device__ __forceinline__ void mask_scores(f16v (&s)[KB], const uint32_t (&bits)[KB], int half) {
    const uint32_t shift = here(4 * half);
#pragma unroll
    for (int z = 0; z < KB; ++z) {
        const uint32_t b = bits[z] >> shift;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[z][i] = (b >> (8 * (i / 4) + i % 4)) & 1 ? s[z][i] : neg_inf();
    }
}

// The row's maximum with the tile's scores, in log2 units.
template <int KB>
__device__ __forceinline__ float top_of(const f16v (&s)[KB], const RowState& st, float scale2) {
    float top = neg_inf();
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[z][i]);
    const LanePair o = swap32(top);
    return fmaxf(st.m, fmaxf(o.a, o.b) * scale2);
}
// Whether weights could pass 2^15: a score outgrew the maximum (the same in every lane).
__device__ __forceinline__ bool outgrown(const RowState& st, float top) {
    return __any(top > st.m + TREE_LAZY);
}
__device__ __forceinline__ void rescale(RowState& st, float top) {
    const float alpha = fast_exp2(st.m - (top == neg_inf() ? 0.f : top));
    st.l *= alpha;
#pragma unroll
    for (int c = 0; c < 4; ++c) st.acc[c] *= alpha;
    st.m = top;
    pin(st);
}

// Softmax weights of the tile as fp16 pairs, and their sum.
template <int KB>
__device__ __forceinline__ void weights_of(const f16v (&s)[KB], RowState& st, float scale2,
                                           u4 (&p)[2 * KB]) {
    const float off = TREE_TOP - (st.m == neg_inf() ? 0.f : st.m);
    float l[4] = {0.f, 0.f, 0.f, 0.f};        // (four sums: shorter chains)
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float w0 = fast_exp2(__builtin_fmaf(s[z][i], scale2, off));
            const float w1 = fast_exp2(__builtin_fmaf(s[z][i + 1], scale2, off));
            l[i % 4] += w0;
            l[i % 4 + 1] += w1;
            const h2 w = {(half_t)w0, (half_t)w1};
            p[2 * z + i / 8][i / 2 % 4] = __builtin_bit_cast(uint32_t, w);
        }
    st.l += (l[0] + l[1]) + (l[2] + l[3]);
}

// V^T of 16 keys (step j of the tile) and 32 channels (c).
__device__ __forceinline__ u4 values_of(const char* vt, uint32_t lane_v, int j, int c) {
    const u2 a = read_transposed(vt + (lane_v ^ (64 * c)) + j * 4096);
    const u2 b = read_transposed(vt + (lane_v ^ (64 * c)) + j * 4096 + 2048);
    return (u4){a.x, a.y, b.x, b.y};
}

template <int KB>
__device__ __forceinline__ void add_values(const char* vt, const LanePlaces& at, RowState& st,
                                           const u4 (&p)[2 * KB]) {
    u4 v[2 * KB][4];
    const uint32_t lane_v = here(at.v);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[j][c] = values_of(vt, lane_v, j, c);
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) st.acc[c] = mfma3216(v[j][c], p[j], st.acc[c]);
    reads_ahead<10, 2, 16 * KB, 8 * KB>();
    __builtin_amdgcn_sched_barrier(0);
}

// Halves of a V operand's keys 16 j + 4 half + (0..3) and + 8 cleared where `keep` (bits of the
// 32 keys) has a 0.
__device__ __forceinline__ u4 keep_keys(u4 v, uint32_t keep, int j, int half) {
    const uint32_t b = keep >> here(16 * (j & 1) + 4 * half);
    auto pair = [&](int i) {
        return ((b >> i) & 1 ? 0xFFFFu : 0u) | ((b >> (i + 1)) & 1 ? 0xFFFF0000u : 0u);
    };
    v.x &= pair(0);
    v.y &= pair(2);
    v.z &= pair(8);
    v.w &= pair(10);
    return v;
}
// V rows of a 32-key block whose keys do not exist (not `live`) become zeros in LDS: what lies
// there may be anything, and a weight of 0 removes no NaN.  (Waves that share the block all
// write the same zeros.)
__device__ __forceinline__ void clear_values(char* vt, uint32_t live, int lane_) {
    const uint32_t lane = here(lane_);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!((live >> (4 * i + (lane >> 4))) & 1)) *(u4*)(vt + i * 1024 + lane * 16) = (u4){0, 0, 0, 0};
}

// The largest magnitude of an operand's halves so far, as bits (an infinity or a NaN: 0x7C00 and
// more).
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ us2 magnitude(us2 m, u4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, v[i] & 0x7FFF7FFFu));
    return m;
}

// Whether V of a tile holds an infinity or a NaN.
template <int KB>
__device__ __forceinline__ bool odd_values(const char* vt, const LanePlaces& at) {
    const uint32_t lane_v = here(at.v);
    us2 m = {0, 0};
#pragma unroll 1
    for (int j = 0; j < 2 * KB; ++j) {
        u4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = values_of(vt + j * 4096, lane_v, 0, c);
#pragma unroll
        for (int c = 0; c < 4; ++c) m = magnitude(m, v[c]);
    }
    return __any(m.x >= 0x7C00 || m.y >= 0x7C00);
}

// A tile whose V holds an infinity or a NaN, which some rows see and others do not: products a
// row at a time, of the keys that the row sees.  bits: what the lane's row sees.
template <int KB>
__device__ __forceinline__ void add_values_by_row(const char* vt, const LanePlaces& at, RowState& st,
                                                  const u4 (&p)[2 * KB], const uint32_t (&bits)[KB],
                                                  int half) {
    const int row = (int)here(__lane_id()) & 31;
    // (loops that stay loops: this is rare, and registers are the common path's)
#pragma unroll 1
    for (int z = 0; z < KB; ++z) {
        const u4 p0 = z ? p[2 * KB - 2] : p[0], p1 = z ? p[2 * KB - 1] : p[1];
        const uint32_t b = z ? bits[KB - 1] : bits[0];
#pragma unroll 1
        for (int x = 0; x < 32; ++x) {
            const uint32_t seen = (uint32_t)__builtin_amdgcn_readlane((int)b, x);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t lane_v = here(at.v);
                f16v y;
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = 0.f;
                y = mfma3216(keep_keys(values_of(vt + z * 8192, lane_v, 0, c), seen, 0, half), p0, y);
                y = mfma3216(keep_keys(values_of(vt + z * 8192, lane_v, 1, c), seen, 1, half), p1, y);
#pragma unroll
                for (int i = 0; i < 16; ++i) st.acc[c][i] += row == x ? y[i] : 0.f;
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" ::: "memory");        // (one quarter's registers at a time)
            }
        }
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

// Inclusive prefix sum over the wave's lanes, and its total (row shifts inside 16 lanes, whose
// missing sources add 0, then the rows' totals).
template <int CTRL>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ int scan(int x, int lane, int& total) {
    x = dpp_add<0x118>(dpp_add<0x114>(dpp_add<0x112>(dpp_add<0x111>(x))));
    const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = __builtin_amdgcn_readlane(x, 31),
              r2 = __builtin_amdgcn_readlane(x, 47), r3 = __builtin_amdgcn_readlane(x, 63);
    total = r0 + r1 + r2 + r3;
    const int row = lane >> 4;
    return x + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}

// Which steps of which units group g takes.
//
// Units no more than groups (one sequence a lane): a group has a part of one unit, so it
// starts and joins once.  Parts are as long as the groups suffice for: the smallest length
// `per` whose parts, ceil(steps / per) a unit, are no more than the groups; a unit's parts
// are then made even.
//
// More units: all units' steps in a row, each unit's behind `extra` places that starting on
// it counts as, cut into even runs; a group's run may end one unit and start others.
struct Runs {
    bool dealt;
    int per;                              // of a run
    int u0, u1;                           // the run (dealt: the unit's steps s0, s1)
    int first, last;                      // dealt: the unit's groups
};
__device__ __forceinline__ Unit find_run(const TreeParams& a, int step_keys, int lane, int g, Runs& r) {
    Unit u = {a.B, 0, 0, 0, 1};
    const int units = a.B * a.H;
    r.dealt = a.B <= WAVE && units <= a.groups;
    if (r.dealt) {
        const int len = lane < a.B ? length_of(a, lane) : 0;
        const int steps = lane < a.B ? steps_of(a, len, step_keys) : 0;
        int total;
        scan(steps, lane, total);
        total *= a.H;
        // parts of length per: at most total / per + units
        int lo = (total + a.groups - 1) / a.groups, hi = total;
        if (a.groups > units) hi = (total + a.groups - units - 1) / (a.groups - units);
        lo = __builtin_amdgcn_readfirstlane(lo < 1 ? 1 : lo);
        hi = __builtin_amdgcn_readfirstlane(hi < lo ? lo : hi);
        auto parts_of = [&](int per) {
            // (an estimate by the reciprocal, put right)
            int n = (int)((float)steps * __builtin_amdgcn_rcpf((float)per));
            n += n * per < steps ? 1 : 0;
            n += n * per < steps ? 1 : 0;
            return n;
        };
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            int sum;
            scan(parts_of(mid), lane, sum);
            if (sum * a.H <= a.groups)
                hi = mid;
            else
                lo = mid + 1;
        }
        const int n = parts_of(lo);
        int all;
        const int incl = scan(n * a.H, lane, all);
        if (g >= all) return u;
        const int src = __builtin_ctzll(__ballot(g < incl));
        const int parts = __builtin_amdgcn_readlane(n, src);
        const int at = g - __builtin_amdgcn_readlane(incl - n * a.H, src);
        u.b = src;
        u.len = __builtin_amdgcn_readlane(len, src);
        u.steps = __builtin_amdgcn_readlane(steps, src);
        u.h = __builtin_amdgcn_readfirstlane(at / parts);
        const int part = at - u.h * parts;
        const int even = __builtin_amdgcn_readfirstlane(u.steps / parts), more = u.steps - even * parts;
        r.u0 = part * even + (part < more ? part : more);
        r.u1 = r.u0 + even + (part < more ? 1 : 0);
        r.first = g - part;
        r.last = r.first + parts - 1;
        return u;
    }
    // (two passes over the lengths: the total, then where the run starts)
    int total = 0;
    for (int b0 = 0; b0 < a.B; b0 += WAVE) {
        const int b = b0 + lane;
        int sum;
        scan(b < a.B ? (steps_of(a, length_of(a, b), step_keys) + a.extra) * a.H : 0, lane, sum);
        total += sum;
    }
    r.per = __builtin_amdgcn_readfirstlane((total + a.groups - 1) / a.groups);
    const int64_t from = (int64_t)g * r.per;
    if (from >= total) return u;
    r.u0 = (int)from;
    r.u1 = total - r.u0 < r.per ? total : r.u0 + r.per;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += WAVE) {
        const int b = b0 + lane;
        const int len = b < a.B ? length_of(a, b) : 0;
        const int n = b < a.B ? (steps_of(a, len, step_keys) + a.extra) * a.H : 0;
        int sum;
        const int incl = scan(n, lane, sum);
        if (r.u0 < before + sum) {
            const int src = __builtin_ctzll(__ballot(r.u0 < before + incl));
            u.b = b0 + src;
            u.len = __builtin_amdgcn_readlane(len, src);
            u.steps = steps_of(a, u.len, step_keys);
            const int first = before + __builtin_amdgcn_readlane(incl - n, src);
            u.h = __builtin_amdgcn_readfirstlane((r.u0 - first) / (u.steps + a.extra));
            u.start = first + u.h * (u.steps + a.extra) + a.extra;
            return u;
        }
        before += sum;
    }
    return u;
}
// The next unit of a run (false: none).
__device__ __forceinline__ bool next_unit(const TreeParams& a, int step_keys, const Runs& r, Unit& u) {
    if (r.dealt) return false;
    u.start += u.steps + a.extra;
    if (++u.h == a.H) {
        u.h = 0;
        if (++u.b >= a.B) return false;
        u.len = length_of(a, u.b);
        u.steps = steps_of(a, u.len, step_keys);
    }
    return u.start - a.extra < r.u1;
}

// NW waves: WR row groups of 32 rows by NW / WR key groups.
// SCORES: the scores are stored too (one tile of rows).
// (Bounds of eight waves for four too: with more than 256 registers to give, the compiler
// keeps the sums in the accumulation registers and moves them for every other use.)
template <int NW, int WR, int KB, bool SCORES>
__global__ __launch_bounds__(WAVE * 8) __attribute__((amdgpu_waves_per_eu(2)))
void tree_kernel(const TreeParams a) {
    constexpr int WK = NW / WR, KEYS = 32 * KB, STEP = KEYS * WK;
    constexpr int TILE = KEYS * 256;                       // bytes of K, and of V
    __shared__ __attribute__((aligned(1024))) char k0_[WK * TILE];
    __shared__ __attribute__((aligned(1024))) char v0_[WK * TILE];
    __shared__ __attribute__((aligned(1024))) char k1_[WK * TILE];
    __shared__ __attribute__((aligned(1024))) char v1_[WK * TILE];
    __shared__ float2 ml_[NW][32];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int rg = wave % WR, kg = wave / WR, half = lane >> 5;
    const int v = xcd_major(blockIdx.x, gridDim.x);
    const int g = __builtin_amdgcn_readfirstlane(v / a.row_tiles), rt = v - g * a.row_tiles;

    Runs run;
    Unit u = find_run(a, STEP, lane, g, run);
    if (u.b >= a.B) return;                                // (every wave alike, before any barrier)

    const LanePlaces at = lane_places(lane);
    const int R = a.N * a.NR;
    // the lane's row, worked out where it is used (in registers it would cost the loop some)
    struct Row {
        int node, rep;
        bool is;
    };
    auto row_of = [&] {
        const int row = (rt * WR + rg) * 32 + (int)here(lane & 31);
        Row o;
        o.is = row < R;
        o.node = o.is ? row / a.NR : 0;
        o.rep = o.is ? row - o.node * a.NR : 0;
        return o;
    };

    // this wave's part of a tile's loads: LOADS instructions of four rows, K and V each
    constexpr int LOADS = KEYS / 4 / WR;
    const uint32_t row_in = (uint32_t)(lane >> 4) * (uint32_t)a.sp_t;

    do {
        int s0 = run.u0, s1 = run.u1;
        if (!run.dealt) {
            s0 = s0 > u.start ? s0 - u.start : 0;
            s1 = s1 - u.start < u.steps ? s1 - u.start : u.steps;
            if (s0 >= s1) continue;                        // (only what starting counts as)
        }
        const int keys = keys_of(a, u.len);
        const int ctx = u.len > a.N ? u.len - a.N : 0;
        int nodes = a.N;
        if (a.counts) {
            const int n = a.counts[u.b];
            nodes = n < nodes ? (n > 0 ? n : 0) : nodes;
        }
        nodes = nodes < u.len ? nodes : u.len;
        const int32_t* table = a.tables + u.b * a.st_b;
        const int pages = (keys + PAGE - 1) / PAGE, last_page = pages > 0 ? pages - 1 : 0;

        u4 q[8];
        RowState st;

        // Blocks of a step's tile, a lane a page (past the sequence's last page, it again: keys
        // there do not count).
        auto ids_of = [&](int step) {
            int i = (int)here(lane);
            i = (step * WK + kg) * (KEYS / PAGE) + (i < KEYS / PAGE ? i : KEYS / PAGE - 1);
            return table[i < pages ? i : last_page];
        };
        // its pages that are not in the pool
        auto bad_of = [&](int ids) {
            return (uint32_t)__ballot((unsigned)ids >= (unsigned)a.num_blocks) & ((1u << (KEYS / PAGE)) - 1);
        };
        // (a page outside the pool is not requested: what its rows hold then counts as nothing)
        auto load = [&](int z, int ids, char* t) {
            constexpr int SAME = LOADS < 4 ? LOADS : 4;    // instructions of one page
            const uint32_t row = here(row_in), k_in = here(at.k_in), v_in = here(at.v_in);
#pragma unroll
            for (int i0 = 0; i0 < LOADS; i0 += SAME) {
                const int first = (rg * LOADS + i0) * 4;
                const int id = __builtin_amdgcn_readlane(ids, first / PAGE);
                const bool in = (unsigned)id < (unsigned)a.num_blocks;
                const __amdgpu_buffer_rsrc_t from =
                    page_rsrc(a.pool[z] + (in ? id : 0) * a.sp_b + u.h * a.sp_h, in);
#pragma unroll
                for (int i = 0; i < SAME; ++i) {
                    const int n = LOADS < 4 ? (rg * LOADS + i) & 3 : i;       // of the page's four
                    const uint32_t off = z ? v_in ^ (128 * (n & 1)) : k_in ^ (64 * n);
                    load_to_lds(from, row + off, 4 * n * (int)a.sp_t, t + (first + 4 * i) * 256);
                }
            }
        };
        // a block's scores, in log2 units
        auto store_scores = [&](const f16v& s, int64_t k0) {
            if ((lane & 31) >= R || k0 >= keys) return;
            float* to = a.scores + ((int64_t)(u.b * a.H + u.h) * R + (lane & 31)) * a.score_len + k0 + 4 * half;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const f4 x = {s[4 * n] * a.scale2, s[4 * n + 1] * a.scale2, s[4 * n + 2] * a.scale2,
                              s[4 * n + 3] * a.scale2};
                *(f4*)(to + 8 * n) = x;
            }
        };
        // What the row sees of a step's tile (bits), and which of its keys exist (live, the same in
        // every lane).  Steps of the context alone, with all their pages, need neither.
        uint32_t bits[KB], live[KB];
        auto look = [&](int step, uint32_t bad) {
            const Row row = row_of();
            const bool seeing = row.is && row.node < nodes;
            const uint64_t* row_mask =
                a.masks ? a.masks + ((int64_t)u.b * a.N + row.node) * a.words : nullptr;
#pragma unroll
            for (int z = 0; z < KB; ++z) {
                const int64_t k0 = ((int64_t)step * WK + kg) * KEYS + 32 * z;
                const int64_t left = (ctx + nodes < keys ? ctx + nodes : keys) - k0;
                uint32_t l = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << (int)left) - 1;
                if ((bad >> (2 * z)) & 1) l &= 0xFFFF0000u;
                if ((bad >> (2 * z + 1)) & 1) l &= 0x0000FFFFu;
                live[z] = l;
                bits[z] = seeing && l ? seen_bits(a, row_mask, row.node, k0 - ctx, nodes) & l : 0u;
            }
        };
        // A step's products; false, with nothing done, where V holds an infinity or a NaN that a row
        // may not see.
        auto add_step = [&](int step, bool masked, const char* kt, char* vt) {
            f16v s[KB];
            u4 p[2 * KB];
            scores_of<KB>(kt, at, q, s);
            if (masked) {
                mask_scores<KB>(s, bits, half);
#pragma unroll 1
                for (int z = 0; z < KB; ++z) clear_values(vt + z * 8192, z ? live[KB - 1] : live[0], lane);
                if (odd_values<KB>(vt, at)) return false;
            }
            if constexpr (SCORES) store_scores(s[0], ((int64_t)step * WK + kg) * KEYS);
            const float top = top_of<KB>(s, st, a.scale2);
            if (outgrown(st, top)) rescale(st, top);
            pin(st);
            weights_of<KB>(s, st, a.scale2, p);
            add_values<KB>(vt, at, st, p);
            return true;
        };
        auto add_step_by_row = [&](int step, const char* kt, const char* vt) {
            f16v s[KB];
            u4 p[2 * KB];
            scores_of<KB>(kt, at, q, s);
            mask_scores<KB>(s, bits, half);
            if constexpr (SCORES) store_scores(s[0], ((int64_t)step * WK + kg) * KEYS);
            const float top = top_of<KB>(s, st, a.scale2);
            if (outgrown(st, top)) rescale(st, top);
            pin(st);
            weights_of<KB>(s, st, a.scale2, p);
            add_values_by_row<KB>(vt, at, st, p, bits, half);
        };

        char* const kt0 = k0_ + kg * TILE;
        char* const vt0 = v0_ + kg * TILE;
        // steps of the context alone, then the others
        const int plain = (ctx < keys ? ctx : keys) / STEP;
        const int sf = s1 < plain ? s1 : plain;
        int ids = ids_of(s0);
        {
            // (a lane past the last row takes the first one's: its results go nowhere)
            const Row row = row_of();
            const half_t* p = a.q + u.b * a.sq_b + row.node * a.sq_n + u.h * a.sq_h +
                              row.rep * a.sq_r + 8 * half;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = *(const u4*)(p + 16 * j);
        }
        clear(st);

        uint32_t bad = bad_of(ids);
        load(0, ids, kt0);
        load(1, ids, vt0);
        // (A step of infinities leaves the loop for its products by row and comes back: as a branch
        // inside it, it would cost every step copies of the sums.)
        char* const kt1 = k1_ + kg * TILE;
        char* const vt1 = v1_ + kg * TILE;
        ids = s0 + 1 < s1 ? ids_of(s0 + 1) : 0;
        bool masked;
        // a step's loads have come and everyone is done with the step before: the next
        // one's go out
        auto turn = [&](int step, char* kn, char* vn) {
            masked = step >= sf || bad != 0;
            if (masked) look(step, bad);               // (its loads come with the tile's)
            wait_vm_lds<0>();
            if constexpr (WR > 1) {
                __syncthreads();
            } else {                                       // (a tile of the wave's own)
                __builtin_amdgcn_s_waitcnt(0xC07F);        // lgkmcnt 0
                asm volatile("" ::: "memory");
            }
            if (step + 1 < s1) {
                bad = bad_of(ids);
                load(0, ids, kn);
                load(1, ids, vn);
                if (step + 2 < s1) ids = ids_of(step + 2);
            }
        };
        int step = s0;
        bool second = false;                           // which buffers hold the step
        while (true) {
            while (true) {
                if (!second) {
                    turn(step, kt1, vt1);
                    if (!add_step(step, masked, kt0, vt0)) break;
                    second = true;
                    if (++step >= s1) break;
                }
                turn(step, kt0, vt0);
                if (!add_step(step, masked, kt1, vt1)) break;
                second = false;
                if (++step >= s1) break;
            }
            if (step >= s1) break;
            add_step_by_row(step, second ? kt1 : kt0, second ? vt1 : vt0);
            second = !second;
            if (++step >= s1) break;
        }

        // ---- the key groups' results made one, then the output or a record ----
        const bool whole = s0 == 0 && s1 == u.steps;
        const LanePair lp = swap32(st.l);
        float l = lp.a + lp.b, m = st.m;
        constexpr int QUADS = 16 / WK;                     // of 16 channel quads, this wave's
        f4 y[QUADS];
        if constexpr (WK > 1) {
            // 16 KB a wave, over the tiles' arrays
            constexpr int PER = WK * TILE / 16384;
            auto place = [&](int w) -> char* {
                char* arr = w / PER == 0 ? k0_ : w / PER == 1 ? v0_ : w / PER == 2 ? k1_ : v1_;
                return arr + (w % PER) * 16384;
            };
            __syncthreads();
            char* mine = place(wave);
            const uint32_t lane16 = here(lane * 16);
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                const f4 x = {st.acc[n / 4][4 * (n % 4)], st.acc[n / 4][4 * (n % 4) + 1],
                              st.acc[n / 4][4 * (n % 4) + 2], st.acc[n / 4][4 * (n % 4) + 3]};
                *(f4*)(mine + n * 1024 + lane16) = x;
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
                    y[n] += *(const f4*)(from + (kg * QUADS + n) * 1024 + lane16) * w;
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
        const Row row = row_of();
        if (whole) {
            const bool seeing = row.is && row.node < nodes;
            const float inv = seeing && l != 0.f ? 1.f / l : 0.f;
            if (row.is) {
                half_t* o = a.out + u.b * a.so_b + row.node * a.so_n + u.h * a.so_h + row.rep * a.so_r;
#pragma unroll
                for (int n = 0; n < QUADS; ++n) {
                    const int quad = kg * QUADS + n;
                    h4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = seeing ? (half_t)(y[n][e] * inv) : (half_t)0.f;
                    *(h4*)(o + 8 * quad + 4 * half) = x;
                }
                if (a.lse && kg == 0 && half == 0)
                    a.lse[((int64_t)(u.b * a.N + row.node) * a.H + u.h) * a.NR + row.rep] =
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
            a.info[u.b * a.H + u.h] =
                run.dealt ? make_int2(run.first, run.last)
                          : make_int2(u.start / run.per, (u.start + u.steps - 1) / run.per);
    } while (next_unit(a, STEP, run, u));
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

template <int NW, int WR, int KB, bool SCORES>
hipError_t launch(const TreeParams& a, hipStream_t stream) {
    tree_kernel<NW, WR, KB, SCORES><<<dim3(a.groups * a.row_tiles), dim3(WAVE * NW), 0, stream>>>(a);
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
    s.nw = s.wr == 1 ? 4 : 8;
    s.kb = s.wr >= 4 ? 2 : 1;
    s.row_tiles = (rows + 32 * s.wr - 1) / (32 * s.wr);
    const int64_t step = 32 * s.kb * (s.nw / s.wr);
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
    if (a.scores) return launch<4, 1, 1, true>(a, stream);
    switch (s.wr) {
        case 1: return launch<4, 1, 1, false>(a, stream);
        case 2: return launch<8, 2, 1, false>(a, stream);
        case 4: return launch<8, 4, 2, false>(a, stream);
        default: return launch<8, 8, 2, false>(a, stream);
    }
}

}  // namespace ls

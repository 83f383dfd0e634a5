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
// piece p of key r at place p ^ (r % 16), V's 32-byte units swapped by row too, so that
// neither the row reads of K nor the transposing reads of V meet in a bank.
//
// Bound by K's and V's bytes up to about 100 rows (16 sequences of 16K, 2 heads: 12 rows with
// scores 52 us, 5.2 TB/s; 96 rows 56 us), then by the products and exponentials, which a
// SIMD's two waves do one after the other for the most part (198 rows: 2.2 us a step of 64 keys,
// the matrix units busy 38 % of the time, the vector units 43 %).
#include "ls_common.h"
#include "ls_tree.h"
#include "ls_tree_load.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __fp16 g4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

namespace {

// A weight is 2^(x - m + TOP) with x - m <= LAZY: at most 2^15, which fp16 holds, and of
// full precision down to 2^-21 of the running maximum's.  It is rounded to fp16 for the second
// product, as in the framework's decode, since the matrix units take V's type on both sides: at
// most 2^-11 of a weight, as much as the output's own rounding.  Against 64 bits, 16 sequences of
// 16K, outputs are off by 2.9e-4 of their size (2.1e-4 with weights of 32 bits).  The sums and the
// log-sum-exp are of the unrounded ones.
constexpr float TREE_TOP = 7.f, TREE_LAZY = 8.f;

__device__ __forceinline__ u2 read_transposed(const char* p) {
    return __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((g4 __attribute__((address_space(3)))*)p));
}

// Products are of ROWS rows: 32 (32x32x16), or 16 (16x16x32) where a head has no more, for half
// the arithmetic.  A lane holds row lane % ROWS, its part h = lane / ROWS of HB.
template <int ROWS>
struct Form;
template <>
struct Form<32> {
    typedef f16v Acc;
    static constexpr int PARTS = 4;       // of the channels, an accumulator each
    static __device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};
template <>
struct Form<16> {
    typedef f4 Acc;
    static constexpr int PARTS = 8;
    static __device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};

// Where a lane reads a tile's K and V, and what it loads of it, in bytes.  A tile starts
// on 1 KB and a row is 256 bytes, so a swizzled place inside a row is one exclusive or:
//   K of step j:         k ^ (16 HB j)     (piece HB j + h of key lane % ROWS)
//   V of part c:         v ^ (256 / PARTS c)
//   loads i of a page:   (4 i + lane / 16) rows, pieces k_in ^ (64 i), v_in ^ v_turn(i)
// V's unit u of row r lies at u ^ v_swap(r): a transposing read's 32 lanes take eight units
// (of four rows, or of eight), which then lie in all eight places of a row's 256 bytes.
struct LanePlaces {
    uint32_t k, v, k_in, v_in;
};
template <int ROWS>
constexpr __device__ __forceinline__ int v_swap(int r) { return ROWS == 32 ? 2 * (r & 3) : r & 7; }
template <int ROWS>
constexpr __device__ __forceinline__ int v_turn(int i) { return ROWS == 32 ? 0 : 128 * (i & 1); }
template <int ROWS>
__device__ __forceinline__ LanePlaces lane_places(int lane) {
    LanePlaces p;
    const int key = lane % ROWS, h = lane / ROWS, quarter = lane >> 4, pp = lane & 15;
    p.k = key * 256 + 16 * (h ^ (key & 15));
    // a transposing read's 16 lanes take four keys' 16 channels and get a channel's four keys
    const int r = 4 * h + ((lane & 15) >> 2), unit = ROWS == 32 ? quarter & 1 : 0;
    p.v = r * 256 + 32 * (unit ^ v_swap<ROWS>(r)) + 8 * (lane & 3);
    p.k_in = 16 * (pp ^ quarter);
    p.v_in = 32 * ((pp >> 1) ^ v_swap<ROWS>(quarter)) + 16 * (pp & 1);
    return p;
}
// The same value, made anew where it is used: what follows from it is computed there, not
// kept in registers through the loop.
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Of ROWS rows and 32 KB keys a tile.
template <int ROWS, int KB>
struct Tile {
    typedef Form<ROWS> F;
    typedef typename F::Acc Acc;
    static constexpr int HB = 64 / ROWS, PARTS = F::PARTS;
    static constexpr int STEPS = 16 / HB;               // of the first product (128 channels)
    static constexpr int SN = ROWS / 2;                 // scores a lane and 32 keys
    static constexpr int NP = KB * SN / 8;              // steps of the second product
    static constexpr int EL = sizeof(Acc) / 4;
    static constexpr int QUADS = ROWS / 2;              // four adjacent channels each

    u4 q[STEPS];
    Acc acc[PARTS];                                     // O^T
    float m, l;                                         // maximum (log2 units), this part's sum
    float s[KB][SN];                                    // scores: see key_of
    u4 p[NP];                                           // weights, fp16
    LanePlaces at;
    int h;                                              // lane / ROWS

    // the key of score i, and the channel of quad n's first value, but for 4 h
    static constexpr int key_of(int i) { return 128 / SN * (i / 4) + i % 4; }
    static constexpr int channel_of(int n) { return 128 / QUADS * n; }
    __device__ __forceinline__ f4 quad(int n) const {
        const Acc& x = acc[4 * n / EL];
        const int i = 4 * n % EL;
        return (f4){x[i], x[i + 1], x[i + 2], x[i + 3]};
    }

    // Keeps the sums in one set of registers where branches join (the compiler otherwise takes
    // them apart there and copies all of them, in every step).
    __device__ __forceinline__ void pin() {
        if constexpr (PARTS == 4)
            asm volatile("" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]));
        else
            asm volatile("" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]), "+v"(acc[4]),
                              "+v"(acc[5]), "+v"(acc[6]), "+v"(acc[7]));
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < PARTS; ++c)
#pragma unroll
            for (int i = 0; i < EL; ++i) acc[c][i] = 0.f;
        m = neg_inf();
        l = 0.f;
    }

    // What the scheduler is to keep: `FIRST` LDS reads ahead, then one product and `PER`
    // reads in turn (left to itself it reads an operand and waits for it, product by product).
    template <int FIRST, int PER, int READS, int PRODUCTS>
    static __device__ __forceinline__ void reads_ahead() {
        __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (FIRST + i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
        }
    }

    __device__ __forceinline__ void scores(const char* kt) {
        constexpr int NZ = KB * 32 / ROWS;              // ROWS keys each
        Acc x[NZ];
#pragma unroll
        for (int z = 0; z < NZ; ++z)
#pragma unroll
            for (int i = 0; i < EL; ++i) x[z][i] = 0.f;
        u4 k[STEPS][NZ];
        const uint32_t lane_k = here(at.k);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
#pragma unroll
            for (int z = 0; z < NZ; ++z)
                k[j][z] = *(const u4*)(kt + (lane_k ^ (16 * HB * j)) + z * ROWS * 256);
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
#pragma unroll
            for (int z = 0; z < NZ; ++z) x[z] = F::mfma(k[j][z], q[j], x[z]);
        reads_ahead<4, 1, STEPS * NZ, STEPS * NZ>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int z = 0; z < KB; ++z)
#pragma unroll
            for (int i = 0; i < SN; ++i) s[z][i] = x[(z * SN + i) / EL][i % EL];
    }

    // bits: what the row sees of each 32 keys
    __device__ __forceinline__ void mask(const uint32_t (&bits)[KB]) {
        const uint32_t shift = here(4 * h);
#pragma unroll
        for (int z = 0; z < KB; ++z) {
            const uint32_t b = bits[z] >> shift;
#pragma unroll
            for (int i = 0; i < SN; ++i) s[z][i] = (b >> key_of(i)) & 1 ? s[z][i] : neg_inf();
        }
    }

    // Softmax weights of the scores, the maximum and the sum brought up to date.
    __device__ __forceinline__ void weights(float scale2) {
        float top = neg_inf();
#pragma unroll
        for (int z = 0; z < KB; ++z)
#pragma unroll
            for (int i = 0; i < SN; ++i) top = fmaxf(top, s[z][i]);
        if constexpr (HB == 2) {
            const LanePair o = swap32(top);
            top = fmaxf(o.a, o.b);
        } else {
            top = group4_max(top);
        }
        top = fmaxf(m, top * scale2);
        // (wave-uniform: weights stay below 2^15 while no score outgrows the maximum by more)
        if (__any(top > m + TREE_LAZY)) {
            const float alpha = fast_exp2(m - (top == neg_inf() ? 0.f : top));
            l *= alpha;
#pragma unroll
            for (int c = 0; c < PARTS; ++c) acc[c] *= alpha;
            m = top;
            pin();
        }
        pin();
        const float off = TREE_TOP - (m == neg_inf() ? 0.f : m);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};            // (four: shorter chains)
#pragma unroll
        for (int z = 0; z < KB; ++z)
#pragma unroll
            for (int i = 0; i < SN; i += 2) {
                const float w0 = fast_exp2(__builtin_fmaf(s[z][i], scale2, off));
                const float w1 = fast_exp2(__builtin_fmaf(s[z][i + 1], scale2, off));
                sum[i % 4] += w0;
                sum[i % 4 + 1] += w1;
                const h2 w = {(half_t)w0, (half_t)w1};
                p[z * (SN / 8) + i / 8][i / 2 % 4] = __builtin_bit_cast(uint32_t, w);
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // V^T of step j's keys (16 of 32 rows' products, 32 of 16 rows') and part c's channels, its
    // keys in the order of the scores.
    static constexpr int STEP_BYTES = 65536 / SN;       // 16 keys, or 32
    __device__ __forceinline__ u4 values_of(const char* vt, uint32_t lane_v, int j, int c) const {
        const char* at = vt + (lane_v ^ (256 / PARTS * c)) + j * STEP_BYTES;
        const u2 a = read_transposed(at), b = read_transposed(at + STEP_BYTES / 2);
        return (u4){a.x, a.y, b.x, b.y};
    }

    __device__ __forceinline__ void values(const char* vt) {
        u4 v[NP][PARTS];
        const uint32_t lane_v = here(at.v);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int c = 0; c < PARTS; ++c) v[j][c] = values_of(vt, lane_v, j, c);
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int c = 0; c < PARTS; ++c) acc[c] = F::mfma(v[j][c], p[j], acc[c]);
        reads_ahead<10, 2, 2 * NP * PARTS, NP * PARTS>();
        __builtin_amdgcn_sched_barrier(0);
    }

    typedef uint16_t us2 __attribute__((ext_vector_type(2)));

    // Whether V of the tile holds an infinity or a NaN: the largest magnitude of its halves, as
    // bits, is 0x7C00 or more.
    __device__ __forceinline__ bool odd(const char* vt) const {
        const uint32_t lane_v = here(at.v);
        us2 top = {0, 0};
#pragma unroll 1
        for (int j = 0; j < NP; ++j) {
            u4 v[PARTS];
#pragma unroll
            for (int c = 0; c < PARTS; ++c) v[c] = values_of(vt + j * STEP_BYTES, lane_v, 0, c);
#pragma unroll
            for (int c = 0; c < PARTS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, v[c][i] & 0x7FFF7FFFu));
        }
        return __any(top.x >= 0x7C00 || top.y >= 0x7C00);
    }

    // A V operand whose keys outside `keep` (bits of the 32 keys) are zeros; j: its step of them.
    __device__ __forceinline__ u4 keep_keys(u4 v, uint32_t keep, int j) const {
        const uint32_t b = keep >> here((SN == 16 ? 16 * j : 0) + 4 * h);
        auto pair = [&](int i) {
            return ((b >> i) & 1 ? 0xFFFFu : 0u) | ((b >> (i + 1)) & 1 ? 0xFFFF0000u : 0u);
        };
        v.x &= pair(0);
        v.y &= pair(2);
        v.z &= pair(key_of(4));
        v.w &= pair(key_of(4) + 2);
        return v;
    }

    // The second product of a tile whose V holds an infinity or a NaN, which some rows see and
    // others do not: a row at a time, of the keys that the row sees.  bits: what the lane's sees.
    __device__ __forceinline__ void values_by_row(const char* vt, const uint32_t (&bits)[KB]) {
        const int row = (int)here(__lane_id()) % ROWS;
        // (loops that stay loops: this is rare, and registers are the common path's)
#pragma unroll 1
        for (int z = 0; z < KB; ++z) {
            const u4 p0 = z ? p[NP - SN / 8] : p[0], p1 = z ? p[NP - 1] : p[SN / 8 - 1];
            const uint32_t b = z ? bits[KB - 1] : bits[0];
#pragma unroll 1
            for (int x = 0; x < ROWS; ++x) {
                const uint32_t seen = (uint32_t)__builtin_amdgcn_readlane((int)b, x);
#pragma unroll
                for (int c = 0; c < PARTS; ++c) {
                    const uint32_t lane_v = here(at.v);
                    Acc y;
#pragma unroll
                    for (int i = 0; i < EL; ++i) y[i] = 0.f;
                    y = F::mfma(keep_keys(values_of(vt + z * 8192, lane_v, 0, c), seen, 0), p0, y);
                    if constexpr (SN == 16)
                        y = F::mfma(keep_keys(values_of(vt + z * 8192, lane_v, 1, c), seen, 1), p1, y);
#pragma unroll
                    for (int i = 0; i < EL; ++i) acc[c][i] += row == x ? y[i] : 0.f;
                    pin();
                    __builtin_amdgcn_sched_barrier(0);
                    asm volatile("" ::: "memory");      // (one part's registers at a time)
                }
            }
        }
    }
};

// V rows of 32 keys that do not exist (not `live`) become zeros in LDS: what lies there may be
// anything, and a weight of 0 removes no NaN.  (Waves that share the keys all write the same
// zeros.)
__device__ __forceinline__ void clear_values(char* vt, uint32_t live, int lane_) {
    const uint32_t lane = here(lane_);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!((live >> (4 * i + (lane >> 4))) & 1)) *(u4*)(vt + i * 1024 + lane * 16) = (u4){0, 0, 0, 0};
}

// The 32 bits of what `row` sees of keys key0 .. key0 + 31 (bit: key - key0), for a tile
// that meets the tree or the end.
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
    int last;                             // dealt: the last of the unit's groups
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
        r.last = g - part + parts - 1;
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

// NW waves: WR row groups of ROWS rows by NW / WR key groups.
// SCORES: the scores are stored too (one row group).
// (Bounds of eight waves for four too: with more than 256 registers to give, the compiler
// keeps the sums in the accumulation registers and moves them for every other use.)
template <int ROWS, int NW, int WR, int KB, bool SCORES>
__global__ __launch_bounds__(WAVE * 8) __attribute__((amdgpu_waves_per_eu(2)))
void tree_kernel(const TreeParams a) {
    typedef Tile<ROWS, KB> T;
    constexpr int WK = NW / WR, KEYS = 32 * KB, STEP = KEYS * WK;
    constexpr int TILE = KEYS * 256;                       // bytes of K, and of V
    // a step's tiles: K of every key group, then V; as many steps as 128 KB hold
    constexpr int STEP_BYTES = 2 * WK * TILE, NBUF = 131072 / STEP_BYTES;
    __shared__ __attribute__((aligned(1024))) char tiles_[NBUF * STEP_BYTES];
    __shared__ float2 ml_[NW][ROWS];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int rg = wave % WR, kg = wave / WR;
    const int v = xcd_major(blockIdx.x, gridDim.x);
    const int g = __builtin_amdgcn_readfirstlane(v / a.row_tiles), rt = v - g * a.row_tiles;

    Runs run;
    Unit u = find_run(a, STEP, lane, g, run);
    int2 split = make_int2(-1, -1);
    if (u.b >= a.B) {                                      // (every wave alike, before any barrier)
        if (rt == 0 && threadIdx.x == 0) a.split[g] = split;
        return;
    }

    T t;
    t.at = lane_places<ROWS>(lane);
    t.h = lane / ROWS;
    const int R = a.N * a.NR;
    // (a row group past the last row only loads)
    const bool works = (rt * WR + rg) * ROWS < R;
    // the lane's row, worked out where it is used (in registers it would cost the loop some)
    struct Row {
        int node, rep;
        bool is;
    };
    auto row_of = [&] {
        const int row = (rt * WR + rg) * ROWS + (int)here(lane % ROWS);
        Row o;
        o.is = row < R;
        o.node = o.is ? row / a.NR : 0;
        o.rep = o.is ? row - o.node * a.NR : 0;
        return o;
    };

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

        {
            // (A lane past the last row takes the first one's: its results go nowhere.  Before the
            // blocks: a wait for these does not then wait for the tiles.)
            const Row row = row_of();
            const half_t* p = a.q + u.b * a.sq_b + row.node * a.sq_n + u.h * a.sq_h +
                              row.rep * a.sq_r + 8 * t.h;
#pragma unroll
            for (int j = 0; j < T::STEPS; ++j) t.q[j] = *(const u4*)(p + 8 * T::HB * j);
        }
        // Blocks of the pages of SPB steps' tiles, a lane a page (past the sequence's last page, it
        // again: keys there do not count), and which of them are not in the pool.
        constexpr int PPT = KEYS / PAGE, SPB = 64 / PPT;
        auto ids_of = [&](int step) {
            int i = (int)here(lane);
            i = ((step + i / PPT) * WK + kg) * PPT + i % PPT;
            return table[i < pages ? i : last_page];
        };
        int ids = ids_of(s0), ids_next = 0;
        uint64_t bad = 0;
        uint32_t bad_ring = 0;                             // 4 bits a step, the last eight
        // this wave's part of a tile: LOADS instructions of four rows, K and V each
        constexpr int LOADS = KEYS / 4 / WR;
        const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)tiles_);
        auto load = [&](int z, int step) {
            constexpr int SAME = LOADS < 4 ? LOADS : 4;    // instructions of one page
            const int at = (step - s0) % SPB * PPT;
            const uint32_t to = lds + step % NBUF * STEP_BYTES + z * WK * TILE + kg * TILE;
            const uint32_t row = here(row_in), in0 = here(z ? t.at.v_in : t.at.k_in);
#pragma unroll
            for (int i0 = 0; i0 < LOADS; i0 += SAME) {
                const int first = (rg * LOADS + i0) * 4;
                const int id = __builtin_amdgcn_readlane(ids, at + first / PAGE);
                // (a page outside the pool is not requested: what its rows hold counts as nothing)
                const bool in = (unsigned)id < (unsigned)a.num_blocks;
                const u4 from = rsrc_of(a.pool[z] + (in ? id : 0) * a.sp_b + u.h * a.sp_h,
                                        in ? POOL_BYTES : 0);
#pragma unroll
                for (int i = 0; i < SAME; ++i) {
                    const int n = LOADS < 4 ? (rg * LOADS + i) & 3 : i;       // of the page's four
                    load_to_lds(from, row + (in0 ^ (z ? v_turn<ROWS>(n) : 64 * n)), 4 * n * (uint32_t)a.sp_t,
                                to + (first + 4 * i) * 256);
                }
            }
        };
        // before a step's loads: its blocks at hand
        auto blocks = [&](int step) {
            const int n = step - s0;
            if (n % SPB == 0) {
                if (n) ids = ids_next;
                bad = __ballot((unsigned)ids >= (unsigned)a.num_blocks);
                if (step + SPB < s1) ids_next = ids_of(step + SPB);
            }
            const int sh = 4 * (step & 7);
            bad_ring = (bad_ring & ~(15u << sh)) |
                       ((uint32_t)(bad >> (n % SPB * PPT)) & ((1u << PPT) - 1)) << sh;
        };
        auto bad_of = [&](int step) { return bad_ring >> (4 * (step & 7)) & 15u; };
        // the scores of a tile (KB 1), in log2 units
        auto store_scores = [&](int64_t k0) {
            const int row = lane % ROWS;
            if (row >= R || k0 >= keys) return;
            float* to = a.scores + ((int64_t)(u.b * a.H + u.h) * R + row) * a.score_len + k0 + 4 * t.h;
#pragma unroll
            for (int i = 0; i < T::SN; i += 4) {
                const f4 x = {t.s[0][i] * a.scale2, t.s[0][i + 1] * a.scale2, t.s[0][i + 2] * a.scale2,
                              t.s[0][i + 3] * a.scale2};
                *(f4*)(to + T::key_of(i)) = x;
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
        // (k_read: what is done once K has been read)
        auto add_step = [&](int step, bool masked, char* kt, char* vt, auto&& k_read) {
            if (!works) {
                k_read();
                return true;
            }
            t.scores(kt);
            if (masked) {
                t.mask(bits);
#pragma unroll 1
                for (int z = 0; z < KB; ++z) clear_values(vt + z * 8192, z ? live[KB - 1] : live[0], lane);
                if (t.odd(vt)) return false;
            }
            k_read();
            if constexpr (SCORES) store_scores(((int64_t)step * WK + kg) * KEYS);
            t.weights(a.scale2);
            t.values(vt);
            return true;
        };
        auto add_step_by_row = [&](int step, char* kt, const char* vt, auto&& k_read) {
            t.scores(kt);
            t.mask(bits);
            k_read();
            if constexpr (SCORES) store_scores(((int64_t)step * WK + kg) * KEYS);
            t.weights(a.scale2);
            t.values_by_row(vt, bits);
        };

        // steps of the context alone, then the others
        const int plain = (ctx < keys ? ctx : keys) / STEP;
        const int sf = s1 < plain ? s1 : plain;
        t.clear();
        int step = s0;
        bool masked;
        char *kt, *vt;
        auto at_step = [&] {
            kt = tiles_ + step % NBUF * STEP_BYTES + kg * TILE;
            vt = kt + WK * TILE;
        };
        if constexpr (WR > 1) {
            // Tiles that row groups share: AHEAD steps are requested; a step's loads have come
            // and everyone is done with the step before, whose place then takes the next.
            constexpr int AHEAD = NBUF - 1;
            for (int i = s0; i < s0 + AHEAD && i < s1; ++i) {
                blocks(i);
                load(0, i);
                load(1, i);
            }
            auto turn = [&] {
                const uint32_t b = bad_of(step);
                masked = step >= sf || b != 0;
                if (masked) look(step, b);                 // (its loads come with the tile's)
                if (AHEAD > 1 && step + AHEAD <= s1)
                    wait_loads<2 * LOADS*(AHEAD - 1)>();
                else
                    wait_loads<0>();
                __syncthreads();
                at_step();
            };
            auto next = [&] {
                if (step + AHEAD < s1) {
                    blocks(step + AHEAD);
                    load(0, step + AHEAD);
                    load(1, step + AHEAD);
                }
            };
            // (A step of infinities leaves the loop for its products by row and comes back: as a
            // branch inside it, it would cost every step copies of the sums.)
            while (true) {
                while (true) {
                    turn();
                    if (!add_step(step, masked, kt, vt, next)) break;
                    if (++step >= s1) break;
                }
                if (step >= s1) break;
                add_step_by_row(step, kt, vt, next);
                if (++step >= s1) break;
            }
        } else {
            // Tiles of the wave's own: nobody to wait for, and a tile's K and V are replaced by
            // those two steps on as soon as each has been read, so that a wave waits with
            // two tiles requested.
            static_assert(NBUF == 2, "");
            auto reads_done = [&] {
                __builtin_amdgcn_s_waitcnt(0xC07F);        // lgkmcnt 0
                asm volatile("" ::: "memory");
            };
            blocks(s0);
            load(0, s0);
            load(1, s0);
            if (s0 + 1 < s1) {
                blocks(s0 + 1);
                load(0, s0 + 1);
                load(1, s0 + 1);
            }
            auto turn = [&] {
                const uint32_t b = bad_of(step);
                masked = step >= sf || b != 0;
                if (masked) look(step, b);
                // (behind the step's own: the next one's 2 LOADS, and maybe more)
                if (step + 1 < s1)
                    wait_loads<2 * LOADS>();
                else
                    wait_loads<0>();
                at_step();
            };
            auto next_k = [&] {
                reads_done();
                if (step + 2 < s1) {
                    blocks(step + 2);
                    load(0, step + 2);
                }
            };
            auto next_v = [&] {
                reads_done();
                if (step + 2 < s1) load(1, step + 2);
            };
            while (true) {
                while (true) {
                    turn();
                    if (!add_step(step, masked, kt, vt, next_k)) break;
                    next_v();
                    if (++step >= s1) break;
                }
                if (step >= s1) break;
                add_step_by_row(step, kt, vt, next_k);
                next_v();
                if (++step >= s1) break;
            }
        }

        // ---- the key groups' results made one, then the output or a record ----
        const bool whole = s0 == 0 && s1 == u.steps;
        float l, m = t.m;
        if constexpr (T::HB == 2) {
            const LanePair lp = swap32(t.l);
            l = lp.a + lp.b;
        } else {
            l = group4_sum(t.l);
        }
        constexpr int QUADS = T::QUADS / WK;               // of the row group's, this wave's
        f4 y[QUADS];
        if constexpr (WK > 1) {
            // over the tiles
            auto place = [&](int w) { return tiles_ + w * (T::QUADS * 1024); };
            __syncthreads();
            char* mine = place(wave);
            const uint32_t lane16 = here(lane * 16);
#pragma unroll
            for (int n = 0; n < T::QUADS; ++n) *(f4*)(mine + n * 1024 + lane16) = t.quad(n);
            if (t.h == 0) ml_[wave][lane] = make_float2(m, l);
            __syncthreads();
            float top = neg_inf();
#pragma unroll
            for (int k = 0; k < WK; ++k) top = fmaxf(top, ml_[k * WR + rg][lane % ROWS].x);
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < QUADS; ++n) y[n] = (f4){0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < WK; ++k) {
                const float2 o = ml_[k * WR + rg][lane % ROWS];
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
        } else {
#pragma unroll
            for (int n = 0; n < QUADS; ++n) y[n] = t.quad(n);
        }
        __syncthreads();                                   // (before the next unit's loads)
        const Row row = row_of();
        if (whole) {
            const bool seeing = row.is && row.node < nodes;
            const float inv = seeing && l != 0.f ? 1.f / l : 0.f;
            half_t* o = a.out + u.b * a.so_b + row.node * a.so_n + u.h * a.so_h + row.rep * a.so_r;
            u2 x[QUADS];
#pragma unroll
            for (int n = 0; n < QUADS; ++n) {
                h4 z;
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = seeing ? (half_t)(y[n][e] * inv) : (half_t)0.f;
                x[n] = __builtin_bit_cast(u2, z);
            }
            if constexpr (T::HB == 2) {
                // a row's two lanes hold four channels each of eight: of two such eights, each
                // lane gets one whole (16 bytes a store: a row's 32 together)
#pragma unroll
                for (int n = 0; n < QUADS; n += 2) {
                    const auto p = __builtin_amdgcn_permlane32_swap(x[n].x, x[n + 1].x, false, false);
                    const auto r = __builtin_amdgcn_permlane32_swap(x[n].y, x[n + 1].y, false, false);
                    if (row.is)
                        *(u4*)(o + T::channel_of(kg * QUADS + n + t.h)) = (u4){p[0], r[0], p[1], r[1]};
                }
            } else if (row.is) {
#pragma unroll
                for (int n = 0; n < QUADS; ++n)
                    *(u2*)(o + T::channel_of(kg * QUADS + n) + 4 * t.h) = x[n];
            }
            if (row.is) {
                if (a.lse && kg == 0 && t.h == 0)
                    a.lse[((int64_t)(u.b * a.N + row.node) * a.H + u.h) * a.NR + row.rep] =
                        seeing && m != neg_inf()
                            ? (m - TREE_TOP + __builtin_amdgcn_logf(l)) * 0.69314718055994531f
                            : neg_inf();
            }
        } else if (row.is) {
            float* rec = a.work + ((((int64_t)g * 2 + (s0 == 0)) * a.row_tiles + rt) * WR + rg) * (ROWS * 130);
#pragma unroll
            for (int n = 0; n < QUADS; ++n) *(f4*)(rec + (kg * QUADS + n) * 256 + lane * 4) = y[n];
            if (kg == 0 && t.h == 0) *(float2*)(rec + ROWS * 128 + 2 * lane) = make_float2(m, l);
        }
        if (s0 == 0) {
            const int last = run.dealt ? run.last : (u.start + u.steps - 1) / run.per;
            if (!whole) split = make_int2(u.b * a.H + u.h, last);
            if (rt == 0 && threadIdx.x == 0) a.info[u.b * a.H + u.h] = make_int2(g, last);
        }
    } while (next_unit(a, STEP, run, u));
    if (rt == 0 && threadIdx.x == 0) a.split[g] = split;
}

// Records of a unit made its output: a workgroup a (unit, ROWS rows, CQ channel quads), its
// waves take the records in turn, AHEAD at once.  Bound by the trips to memory: with a quad a
// workgroup, 128 records are one trip of 16 waves (100K keys, 198 rows: 9.7 us in eight waves'
// four trips, 7.4 us so).
//
// A decode that sums weights has a.score_parts more workgroups a unit: they bring the rows'
// statistics together themselves, rather than in a launch after this one, and add the weights
// of the unit's scores.
template <int NW>
__device__ __forceinline__ void add_scores(const TreeParams& a, int unit, int part, float (*e_s)[16]) {
    const int b = unit / a.H, h = unit - b * a.H;
    const int sum_row = a.sum_rows ? a.sum_rows[b] : b;
    if ((unsigned)sum_row >= (unsigned)a.num_sum_rows) return;
    int64_t keys = (int64_t)a.max_pages * PAGE;
    const int len = a.lens[b];
    keys = len < keys ? len : keys;
    keys = keys < a.sum_len ? keys : a.sum_len;
    constexpr int KEYS = WAVE * NW * 4;            // a round
    if ((int64_t)part * KEYS >= keys) return;
    // each row's log-sum-exp (log2 units) by 16 lanes' worth of records at a time
    const int2 gs = a.info[unit];
    const int row = threadIdx.x % 16;
    if (gs.x == gs.y) {
        if (threadIdx.x < 16)
            e_s[0][row] = row < a.NR ? a.lse[(int64_t)unit * a.NR + row] * 1.4426950408889634f : 0.f;
    } else {
        float m = neg_inf(), l = 0.f;
        for (int k = threadIdx.x / 16; k <= gs.y - gs.x; k += WAVE * NW / 16) {
            const float* rec = a.work + ((int64_t)(gs.x + k) * 2 + (k == 0)) * (16 * 130);
            const float2 o = *(const float2*)(rec + 16 * 128 + 2 * row);
            const float top = fmaxf(m, o.x), use = top == neg_inf() ? 0.f : top;
            l = l * fast_exp2(m - use) + o.y * fast_exp2(o.x - use);
            m = top;
        }
        const float most = group4_max(m);
        l = group4_sum(l * fast_exp2(m - (most == neg_inf() ? 0.f : most)));
        m = most;
        const int wave = threadIdx.x / WAVE;
        if (threadIdx.x % WAVE < 16) {
            e_s[2 * wave][row] = m;
            e_s[2 * wave + 1][row] = l;
        }
        __syncthreads();
        if (threadIdx.x < 16) {
            for (int k = 1; k < NW; ++k) {
                const float x = e_s[2 * k][row], top = fmaxf(m, x), use = top == neg_inf() ? 0.f : top;
                l = l * fast_exp2(m - use) + e_s[2 * k + 1][row] * fast_exp2(x - use);
                m = top;
            }
            e_s[0][row] = m == neg_inf() ? m : m - TREE_TOP + __builtin_amdgcn_logf(l);
        }
    }
    __syncthreads();
    float* sums = a.sums + sum_row * a.ss_row + h * a.ss_h;
    const float* scores = a.scores + (int64_t)unit * a.NR * a.score_len;
    for (int64_t t0 = (int64_t)part * KEYS + threadIdx.x * 4; t0 < keys; t0 += (int64_t)a.score_parts * KEYS) {
        const int n = keys - t0 < 4 ? (int)(keys - t0) : 4;
        f4 sum = {0.f, 0.f, 0.f, 0.f}, had = sum;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) had[i] = sums[t0 + i];
#pragma unroll 4
        for (int r = 0; r < a.NR; ++r) {
            const float e = e_s[0][r];
            const f4 s = *(const f4*)(scores + r * a.score_len + t0);
            // (-inf: it saw nothing, whatever its scores are)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += e == neg_inf() ? 0.f : fast_exp2(s[i] - e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) sums[t0 + i] = had[i] + sum[i];
    }
}

template <int ROWS, int CQ, int NW, bool SCORES>
__global__ __launch_bounds__(WAVE* NW) void tree_combine_kernel(const TreeParams a, int wr) {
    constexpr int PARTS = ROWS / 2 / CQ, AHEAD = CQ == 1 ? 8 : 2;
    __shared__ float sums[NW][CQ * 4 + 2][WAVE];
    if constexpr (SCORES) {
        __shared__ float e_s[2 * NW][16];
        if (blockIdx.y >= PARTS) {
            if (blockIdx.x < a.B * a.H) add_scores<NW>(a, blockIdx.x, blockIdx.y - PARTS, e_s);
            return;
        }
    }
    const int rb = blockIdx.y / PARTS, part = blockIdx.y % PARTS;
    // (of many units few are in several parts: they are found by the groups)
    int unit = blockIdx.x;
    int2 gs;
    if (a.B * a.H <= a.groups) {
        gs = a.info[unit];
        if (gs.x == gs.y) return;
    } else {
        if (SCORES && unit >= a.groups) return;
        gs = a.split[unit];
        if (gs.x < 0) return;
        unit = gs.x;
        gs.x = blockIdx.x;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int rt = rb / wr, rg = rb % wr, count = gs.y - gs.x + 1;
    auto record = [&](int k) {
        const int64_t slot = (int64_t)(gs.x + k) * 2 + (k == 0);
        return a.work + ((slot * a.row_tiles + rt) * wr + rg) * (ROWS * 130);
    };
    float m = neg_inf(), l = 0.f;
    f4 y[CQ];
#pragma unroll
    for (int n = 0; n < CQ; ++n) y[n] = (f4){0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave; k0 < count; k0 += NW * AHEAD) {
        float2 o[AHEAD];
        f4 x[AHEAD][CQ];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = k0 + i * NW;
            const float* rec = record(k < count ? k : k0);
            o[i] = *(const float2*)(rec + ROWS * 128 + 2 * (lane % ROWS));
#pragma unroll
            for (int n = 0; n < CQ; ++n) x[i][n] = *(const f4*)(rec + (part * CQ + n) * 256 + lane * 4);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (k0 + i * NW >= count) break;
            const float top = fmaxf(m, o[i].x), use = top == neg_inf() ? 0.f : top;
            const float keep = fast_exp2(m - use), w = fast_exp2(o[i].x - use);
            l = l * keep + o[i].y * w;
#pragma unroll
            for (int n = 0; n < CQ; ++n) y[n] = y[n] * keep + x[i][n] * w;
            m = top;
        }
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
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sums[w][CQ * 4][lane]);
    const float use = top == neg_inf() ? 0.f : top;
    f4 z = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < NW; ++w) {
        const float f = fast_exp2(sums[w][CQ * 4][lane] - use);
        total += f * sums[w][CQ * 4 + 1][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += f * sums[w][4 * wave + e][lane];
    }
    const int row = rb * ROWS + lane % ROWS, h4_ = 4 * (lane / ROWS);
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
    *(h4*)(a.out + b * a.so_b + node * a.so_n + h * a.so_h + rep * a.so_r +
           256 / ROWS * (part * CQ + wave) + h4_) = x;
    if (a.lse && part == 0 && wave == 0 && lane < ROWS)
        a.lse[((int64_t)(b * a.N + node) * a.H + h) * a.NR + rep] =
            seeing && top != neg_inf()
                ? (top - TREE_TOP + __builtin_amdgcn_logf(total)) * 0.69314718055994531f
                : neg_inf();
}

template <int ROWS, int NW, int WR, int KB, bool SCORES>
hipError_t launch(const TreeParams& a, hipStream_t stream) {
    tree_kernel<ROWS, NW, WR, KB, SCORES>
        <<<dim3(a.groups * a.row_tiles), dim3(WAVE * NW), 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // few of them: a quad a workgroup, so that the records are read by the whole chip
    // (with scores, of eight waves, so that they are too)
    constexpr int NW_FEW = SCORES ? 8 : 16;
    const int blocks = (a.N * a.NR + ROWS - 1) / ROWS, units = a.B * a.H;
    const int most = units < a.groups ? units : a.groups;  // units in several parts
    const int places = SCORES ? units : most;
    if (most * blocks * (ROWS / 8) >= 256)
        tree_combine_kernel<ROWS, 4, 8, SCORES>
            <<<dim3(places, blocks * (ROWS / 8) + a.score_parts), dim3(WAVE * 8), 0, stream>>>(a, WR);
    else
        tree_combine_kernel<ROWS, 1, NW_FEW, SCORES>
            <<<dim3(places, blocks * (ROWS / 2) + a.score_parts), dim3(WAVE * NW_FEW), 0, stream>>>(a, WR);
    return hipGetLastError();
}

}  // namespace

// Up to 16 rows, products of 16: of 32 they would be half empty (12 rows, 1 / 16 sequences of
// 16K: 14.7 / 51.2 us against 15.9 / 54.8).  Up to 32, a wave has all rows and its own keys, and
// waits for nobody (30 rows: 16.8 / 55.3 us, with tiles of two row groups 18.4 / 55.7).  Beyond,
// row groups share a tile: up to 64 rows of four waves, which start and end sooner (48 rows, 2K
// keys 12.7 us, 16 x 16K 63; of eight 16.0 and 60), up to 128 two key groups of eight (96 rows:
// 21.4 / 65 us; 24.2 / 71 with one), then one.  A run has a step at least
// (6 / 48 / 96 rows, 2K keys: 10.6 / 12.2 / 15.7 us against 11.6 / 12.8 / 16.9 of two), of more
// than 128 rows two, whose records cost more than groups give (240 rows, 4K: 20.2 against 23.1).
TreeShape tree_shape(int batch, int kv_heads, int rows, int64_t keys_bound) {
    TreeShape s;
    s.rows = rows <= 16 ? 16 : 32;
    s.wr = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
    s.nw = s.wr <= 2 ? 4 : 8;
    s.kb = s.wr >= 4 ? 2 : 1;
    s.row_tiles = (rows + s.rows * s.wr - 1) / (s.rows * s.wr);
    const int64_t step = 32 * s.kb * (s.nw / s.wr);
    const int64_t units = (int64_t)batch * kv_heads;
    const int64_t places = units * ((keys_bound + step - 1) / step + TREE_EXTRA);
    int64_t most = (TREE_CUS + s.row_tiles - 1) / s.row_tiles;
    const int64_t useful = s.wr == 8 ? (places + 1) / 2 : places;
    s.groups = (int)(most < useful ? most : useful);
    if (s.groups < 1) s.groups = 1;
    return s;
}

size_t tree_record_bytes(const TreeShape& s) {
    return (size_t)s.groups * 2 * s.row_tiles * s.wr * s.rows * 130 * sizeof(float);
}

hipError_t launch_tree_attention(const TreeParams& p, const TreeShape& s, hipStream_t stream) {
    TreeParams a = p;
    a.groups = s.groups;
    a.row_tiles = s.row_tiles;
    a.extra = TREE_EXTRA;
    if (a.scores) return launch<16, 4, 1, 1, true>(a, stream);
    switch (s.wr) {
        case 1: return s.rows == 16 ? launch<16, 4, 1, 1, false>(a, stream)
                                    : launch<32, 4, 1, 1, false>(a, stream);
        case 2: return launch<32, 4, 2, 1, false>(a, stream);
        case 4: return launch<32, 8, 4, 2, false>(a, stream);
        default: return launch<32, 8, 8, 2, false>(a, stream);
    }
}

}  // namespace ls

// Drafted trees' masks and accepted paths, the choice of the tokens that a bounded cache
// keeps, and the moves of their K and V.
#include "ls_common.h"
#include "ls_tree.h"

namespace ls {
namespace {

// ---- masks ------------------------------------------------------------------------

__global__ __launch_bounds__(TREE_MAX_NODES) void tree_masks_kernel(const int32_t* parents,
                                                                    uint64_t* masks, int32_t* depths,
                                                                    int N) {
    __shared__ int par[TREE_MAX_NODES];
    const int b = blockIdx.x, i = threadIdx.x;
    if (i < N) {
        const int p = parents[(int64_t)b * N + i];
        par[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    if (i >= N) return;
    const int words = (N + 63) / 64;
    uint64_t w[TREE_MAX_NODES / 64] = {0, 0, 0, 0};
    int depth = -1;
    for (int at = i; at >= 0; at = par[at]) {              // (downwards: it ends)
#pragma unroll
        for (int k = 0; k < TREE_MAX_NODES / 64; ++k)
            if (at / 64 == k) w[k] |= 1ull << (at & 63);
        ++depth;
    }
    for (int k = 0; k < words; ++k)
#pragma unroll
        for (int z = 0; z < TREE_MAX_NODES / 64; ++z)
            if (z == k) masks[((int64_t)b * N + i) * words + k] = w[z];
    depths[(int64_t)b * N + i] = depth;
}

// ---- moves --------------------------------------------------------------------------
//
// Kept rows of a (pool, sequence, head) move down to the front: row keep[j] to j, keep
// ascending, so keep[j] >= j.  A workgroup moves such a list in rounds, each of some rows:
// a round is stored once all its rows and those of the rounds before have arrived in
// registers, and what it stores lies before every row that a later round reads, so the
// next round's rows are requested first.

struct RowPlaces {
    const int32_t* table;
    int64_t sp_b, sp_t;
    int max_pages, num_blocks;
    // byte offset of the token at `pos` of the sequence, -1 where there is none
    __device__ __forceinline__ int64_t operator()(int64_t pos) const {
        if (pos < 0 || pos >= (int64_t)max_pages * PAGE) return -1;
        const int blk = table[pos / PAGE];
        if ((unsigned)blk >= (unsigned)num_blocks) return -1;
        return blk * sp_b + (pos % PAGE) * sp_t;
    }
};

constexpr int MOVE_THREADS = 256, MOVE_AHEAD = 8;

// Rows `at(j)` of the head to rows base + j, j < n.
template <class At>
__device__ __forceinline__ void move_rows(char* head, const RowPlaces& place, int64_t base, int n,
                                          At at) {
    constexpr int ROWS = MOVE_THREADS / 16;                // a thread: 16 bytes of each
    const int piece = 16 * (threadIdx.x % 16), first = threadIdx.x / 16;
    for (int j0 = 0; j0 < n; j0 += ROWS * MOVE_AHEAD) {
        u4 x[MOVE_AHEAD];
        int64_t to[MOVE_AHEAD];
#pragma unroll
        for (int i = 0; i < MOVE_AHEAD; ++i) {
            const int j = j0 + i * ROWS + first;
            to[i] = -1;
            if (j < n) {
                const int k = at(j);
                if (k > j) {                               // (k = j: it is there)
                    const int64_t from = place(base + k);
                    to[i] = place(base + j);
                    if (from >= 0)
                        x[i] = *(const u4*)(head + from + piece);
                    else
                        to[i] = -1;
                }
            }
        }
        // (every row of the round has arrived before one is stored)
        wait_vm_lds<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MOVE_AHEAD; ++i)
            if (to[i] >= 0) *(u4*)(head + to[i] + piece) = x[i];
    }
}

// A list is cut into slices of its rows' bytes, each a workgroup's own: LANES threads of 16
// bytes a row, AHEAD rows a thread and round.  A round's rows are requested when the one
// before has arrived, their places a round earlier, from pages that were looked up two
// rounds earlier, from entries of keep loaded three rounds earlier: nothing waits for more
// than one trip to memory a round.  Bound by memory: 2048 rows of 112 lists in 25 us (4.7 TB/s
// read and written, a large copy's 5.1; 115 us a round after the other by 256 threads a list).
constexpr int LIST_THREADS = 1024;

template <int LANES, int AHEAD>
__global__ __launch_bounds__(LIST_THREADS) void move_tokens_kernel(const MoveParams a, int pools,
                                                                   int64_t first_list) {
    constexpr int PASS = LIST_THREADS / LANES, ROUND = PASS * AHEAD, SLICES = 16 / LANES;
    static_assert(ROUND <= LIST_THREADS, "a thread looks one row's places up");
    __shared__ int64_t from_s[4][ROUND], to_s[4][ROUND];
    // the slices of a list share an XCD's cache: the lines of a row are theirs together
    const int id = blockIdx.x;
    const int64_t list = first_list + id / (8 * SLICES) * 8 + id % 8;
    if (list >= (int64_t)pools * a.H * a.B) return;
    const int pool = list % pools, h = list / pools % a.H, b = list / pools / a.H;
    int n = a.lens[b];
    n = n < a.budget ? n : a.budget;
    n = n < a.max_pages * PAGE ? n : a.max_pages * PAGE;   // (at most 2^28)
    if (n <= 0) return;
    const int t = threadIdx.x, first = t / LANES;
    const int32_t* keep =
        a.keep + (((int64_t)(a.first_layer + pool / 2) * a.B + b) * a.H + h) * a.budget;
    const int32_t* const table = a.tables + b * a.st_b;
    char* const head = a.pool[pool] + h * a.sp_h + 16 * (LANES * (id / 8 % SLICES) + t % LANES);
    const int rounds = (n + ROUND - 1) / ROUND;
    u4 x[2][AHEAD];
    int k_new = -1, k_old = -1, page_from = -1, page_to = -1;
    // what a round that is not there would move is nothing: its k is -1
    auto step = [&](int r, u4 (&mine)[AHEAD], u4 (&next)[AHEAD]) {
        if (t < ROUND) {
            const int j2 = (r + 2) * ROUND + t;
            const bool moves = (unsigned)page_from < (unsigned)a.num_blocks &&
                               (unsigned)page_to < (unsigned)a.num_blocks;
            from_s[(r + 2) & 3][t] = moves ? page_from * a.sp_b + k_old % PAGE * a.sp_t : 0;
            to_s[(r + 2) & 3][t] = moves ? page_to * a.sp_b + j2 % PAGE * a.sp_t : -1;
            const int j3 = j2 + ROUND, j4 = j3 + ROUND;
            page_from = page_to = -1;
            k_old = k_new;
            if (j3 >= 0 && k_new > j3 && k_new / PAGE < a.max_pages) {      // (k = j: it is there)
                page_from = table[k_new / PAGE];
                page_to = table[j3 / PAGE];
            }
            k_new = j4 < n ? keep[j4] : -1;
        }
        if (r >= -1) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                next[i] = *(const u4*)(head + from_s[(r + 1) & 3][i * PASS + first]);
        }
        if (r >= 0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) asm volatile("" : "+v"(mine[i])::"memory");
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (r >= 0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int64_t to = to_s[r & 3][i * PASS + first];
                if (to >= 0) *(u4*)(head + to) = mine[i];
            }
        }
    };
    for (int r = -4; r < rounds; r += 2) {
        step(r, x[0], x[1]);
        step(r + 1, x[1], x[0]);
    }
}

// One workgroup a (pool, head, sequence), each of which walks its sequence's tree itself: a
// step is a comparison of every node's parent and token, and the first that fits.
__global__ __launch_bounds__(MOVE_THREADS) void accept_tokens_kernel(const MoveParams a, int pools) {
    __shared__ int64_t tok[TREE_MAX_NODES], choice[TREE_MAX_NODES];
    __shared__ int par[TREE_MAX_NODES], path[TREE_MAX_NODES], count_s;
    const int pool = blockIdx.x, h = blockIdx.y, b = blockIdx.z, N = a.N;
    int len = a.lens[b];
    len = len > 0 ? len : 0;
    int nodes = N;
    if (a.counts) {
        const int n = a.counts[b];
        nodes = n < nodes ? (n > 0 ? n : 0) : nodes;
    }
    nodes = nodes < len ? nodes : len;
    for (int i = threadIdx.x; i < nodes; i += MOVE_THREADS) {
        tok[i] = a.tokens[(int64_t)b * N + i];
        choice[i] = a.choices[(int64_t)b * N + i];
        par[i] = a.parents[(int64_t)b * N + i];
    }
    __syncthreads();
    if (threadIdx.x < WAVE) {
        int at = 0, n = 0;
        while (at < nodes) {                               // (upwards: it ends)
            if (threadIdx.x == 0) path[n] = at;
            ++n;
            const int64_t want = choice[at];
            int next = nodes;
            for (int j0 = (at + 1) & ~(WAVE - 1); j0 < nodes; j0 += WAVE) {
                const int j = j0 + threadIdx.x;
                const uint64_t fits =
                    __ballot(j > at && j < nodes && par[j < nodes ? j : 0] == at &&
                             tok[j < nodes ? j : 0] == want);
                if (fits) {
                    next = j0 + __builtin_ctzll(fits);
                    break;
                }
            }
            at = next;
        }
        if (threadIdx.x == 0) count_s = n;
    }
    __syncthreads();
    const int n = count_s;
    if (pool == 0 && h == 0) {
        for (int i = threadIdx.x; i < N; i += MOVE_THREADS)
            a.path[(int64_t)b * N + i] = i < n ? path[i] : -1;
        if (threadIdx.x == 0) {
            a.lengths[b] = n;
            a.next[b] = n > 0 ? choice[path[n - 1]] : -1;
        }
    }
    if (pool >= pools) return;
    const RowPlaces place = {a.tables + b * a.st_b, a.sp_b, a.sp_t, a.max_pages, a.num_blocks};
    const int64_t base = len > N ? len - N : 0;
    move_rows(a.pool[pool] + h * a.sp_h, place, base, n, [&](int j) { return path[j]; });
}

// ---- selection ------------------------------------------------------------------------
//
// The kept sums of a row are found by their bits, eleven at a time from the top: how many
// have each value of the eleven among those that agree in the bits before, until the
// smallest kept value is known; then, in order, what is larger is kept, and as many equal
// ones, lowest positions first, as there is room for.  A wave has a run of the row to
// itself: it counts what it keeps, and writes it once the waves before have counted.
// Bound by its five sweeps of the row and their barriers: 56 rows of 4K 12 us, 224 of up to
// 12K 25, one of 100K 105 (a CU's work; the move behind it takes as long).

constexpr int SELECT_THREADS = 1024, SELECT_WAVES = SELECT_THREADS / WAVE;
constexpr int DIGITS = 2 * SELECT_THREADS;

// A sum's rank: larger sums have larger ranks, NaN the largest.
__device__ __forceinline__ uint32_t rank_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);      // (-0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(SELECT_THREADS) void select_tokens_kernel(const SelectParams a) {
    __shared__ int hist[DIGITS];
    __shared__ int wave_sum[SELECT_WAVES][2];
    __shared__ int found[2];
    const int row = blockIdx.x, h = row % a.H, b = row / a.H % a.B, l = row / a.H / a.B;
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const float* sums = a.sums + l * a.ss_l + b * a.ss_b + h * a.ss_h;
    int len = a.lens[b];
    len = len > 0 ? len : 0;
    if (len > a.sum_len) len = (int)a.sum_len;
    int32_t* keep = a.keep + (int64_t)row * a.budget;
    float* kept = a.kept + (int64_t)row * a.budget;
    if (len <= a.budget) {
        for (int j = threadIdx.x; j < a.budget; j += SELECT_THREADS) {
            keep[j] = j < len ? j : -1;
            kept[j] = j < len ? sums[j] : 0.f;
        }
        return;
    }
    const int tail = len - a.recent;
    // the wave's run, and what f does with WAVE of its sums at a time; some are on their way
    const int per = ((len + SELECT_WAVES - 1) / SELECT_WAVES + WAVE - 1) / WAVE * WAVE;
    const int t0 = wave * per, t1 = t0 + per < len ? t0 + per : len;
    constexpr int U = 8;
    float x[U];
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = t + i * WAVE < t1 ? sums[t + i * WAVE] : 0.f;
    };
    auto use = [&](int t, auto f) {
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (t - lane + i * WAVE < t1) f(t + i * WAVE, x[i]);
    };
    const bool held = per <= U * WAVE;                     // (rows of up to 8K: loaded once)
    load(t0 + lane);
    auto each = [&](auto f) {
        if (held) return use(t0 + lane, f);
        for (int t = t0 + lane; t - lane < t1; t += U * WAVE) {
            load(t);
            use(t, f);
        }
    };
    uint32_t prefix = 0xFFFFFFFFu;
    int want = a.budget - a.sinks - a.recent;              // of those that may go
    if (want > 0) {
        uint32_t known = 0;
        prefix = 0;
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift - 10) {
            const uint32_t digit = shift ? DIGITS - 1 : DIGITS / 2 - 1;
            for (int i = threadIdx.x; i < DIGITS; i += SELECT_THREADS) hist[i] = 0;
            __syncthreads();
            each([&](int t, float x) {
                const uint32_t r = rank_of(x);
                if (t >= a.sinks && t < tail && (r & known) == prefix)
                    atomicAdd(&hist[(r >> shift) & digit], 1);
            });
            __syncthreads();
            // from the top, two values a thread: where the last kept one is, and how many
            // are above
            const int top = DIGITS - 1 - 2 * threadIdx.x;
            const int first = hist[top], count = first + hist[top - 1];
            int upto = count;
            for (int d = 1; d < WAVE; d *= 2) {
                const int o = __shfl_up(upto, d);
                if (lane >= d) upto += o;
            }
            if (lane == WAVE - 1) wave_sum[wave][0] = upto;
            __syncthreads();
            for (int w = 0; w < wave; ++w) upto += wave_sum[w][0];
            const int above = upto - count;
            if (above < want && want <= upto) {            // (one thread's)
                const bool second = above + first < want;
                found[0] = top - second;
                found[1] = above + (second ? first : 0);
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            known |= digit << shift;
            want -= found[1];
        }
    }
    // larger ranks and what is always kept, and the first `want` of equal rank
    int over_n = 0, tie_n = 0;
    auto over = [&](int t, uint32_t r) {
        return t < t1 && (t < a.sinks || t >= tail || r > prefix);
    };
    auto tie = [&](int t, uint32_t r) {
        return t < t1 && t >= a.sinks && t < tail && r == prefix;
    };
    each([&](int t, float x) {
        const uint32_t r = rank_of(x);
        over_n += __builtin_popcountll(__ballot(over(t, r)));
        tie_n += __builtin_popcountll(__ballot(tie(t, r)));
    });
    if (lane == 0) {
        wave_sum[wave][0] = over_n;
        wave_sum[wave][1] = tie_n;
    }
    __syncthreads();
    int o = 0, e = 0;
    for (int w = 0; w < wave; ++w) {
        o += wave_sum[w][0];
        e += wave_sum[w][1];
    }
    each([&](int t, float x) {
        const uint32_t r = rank_of(x);
        const bool is_over = over(t, r), is_tie = tie(t, r);
        const uint64_t bo = __ballot(is_over), bt = __ballot(is_tie);
        const uint64_t below = (1ull << lane) - 1;
        const int before = e + __builtin_popcountll(bt & below);
        // what is kept before t: the larger ones, and of the equal ones as many as count
        const int at = o + __builtin_popcountll(bo & below) + (before < want ? before : want);
        if (is_over || (is_tie && before < want)) {
            keep[at] = t;
            kept[at] = x;
        }
        o += __builtin_popcountll(bo);
        e += __builtin_popcountll(bt);
    });
}

}  // namespace

hipError_t launch_tree_masks(const int32_t* parents, uint64_t* masks, int32_t* depths, int B, int N,
                             hipStream_t stream) {
    tree_masks_kernel<<<dim3(B), dim3(TREE_MAX_NODES), 0, stream>>>(parents, masks, depths, N);
    return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveParams& a, int pools, hipStream_t stream) {
    const int64_t lists = (int64_t)pools * a.H * a.B;
    auto go = [&](auto kernel, int slices) {
        constexpr int64_t MOST = 1 << 18;                  // lists of a launch
        for (int64_t at = 0; at < lists; at += MOST) {
            const int64_t n = lists - at < MOST ? lists - at : MOST;
            kernel<<<dim3((unsigned)((n + 7) / 8 * 8 * slices)), dim3(LIST_THREADS), 0, stream>>>(
                a, pools, at);
        }
    };
    // few lists: in narrower slices, so that more of the chip moves them (20K rows of 16 lists:
    // 86 us against 113, 2K of 112 lists 38 against 25; of 48 lists the same)
    if (lists >= 64)
        go(move_tokens_kernel<8, 4>, 2);
    else
        go(move_tokens_kernel<2, 2>, 8);
    return hipGetLastError();
}

hipError_t launch_accept_tokens(const MoveParams& a, int pools, hipStream_t stream) {
    accept_tokens_kernel<<<dim3(pools > 0 ? pools : 1, pools > 0 ? a.H : 1, a.B), dim3(MOVE_THREADS),
                           0, stream>>>(a, pools);
    return hipGetLastError();
}

hipError_t launch_select_tokens(const SelectParams& a, hipStream_t stream) {
    select_tokens_kernel<<<dim3(a.L * a.B * a.H), dim3(SELECT_THREADS), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace ls

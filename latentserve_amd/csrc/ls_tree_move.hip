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
// The kept rows of a (pool, sequence, head) move down to the front: row keep[j] to j, keep
// ascending, so keep[j] >= j.  A workgroup moves one such list in order, some rows at a
// time: all of a round's rows are in registers before one is stored, and what a round
// stores lies before every row that a later round reads.

struct RowPlaces {
    const int32_t* table;
    int64_t st_b, sp_b, sp_t;
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

__global__ __launch_bounds__(MOVE_THREADS) void move_tokens_kernel(const MoveParams a) {
    const int pool = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = a.lens[b];
    const int n = len < a.budget ? len : a.budget;
    if (n <= 0) return;
    const int32_t* keep =
        a.keep + (((int64_t)(a.first_layer + pool / 2) * a.B + b) * a.H + h) * a.budget;
    const RowPlaces place = {a.tables + b * a.st_b, a.st_b, a.sp_b, a.sp_t, a.max_pages, a.num_blocks};
    move_rows(a.pool[pool] + h * a.sp_h, place, 0, n, [&](int j) { return keep[j]; });
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
    const RowPlaces place = {a.tables + b * a.st_b, a.st_b, a.sp_b, a.sp_t, a.max_pages, a.num_blocks};
    const int64_t base = len > N ? len - N : 0;
    move_rows(a.pool[pool] + h * a.sp_h, place, base, n, [&](int j) { return path[j]; });
}

// ---- selection ------------------------------------------------------------------------
//
// The kept sums of a row are found by their bits, eight at a time from the top: how many
// have each value of the eight among those that agree in the bits before, until the
// smallest kept value is known; then one pass in order writes what is larger, and as
// many equal ones, lowest positions first, as there is room for.

constexpr int SELECT_THREADS = 1024, SELECT_WAVES = SELECT_THREADS / WAVE;

// A sum's rank: larger sums have larger ranks, NaN the largest but for those always kept.
__device__ __forceinline__ uint32_t rank_of(float x) {
    if (x != x) return 0xFFFFFFFEu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);      // (-0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(SELECT_THREADS) void select_tokens_kernel(const SelectParams a) {
    __shared__ int hist[256];
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
    auto rank = [&](int t) {
        return t < a.sinks || t >= tail ? 0xFFFFFFFFu : rank_of(sums[t]);
    };
    uint32_t prefix = 0;
    int want = a.budget;                                   // to be kept of those that agree
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += SELECT_THREADS) hist[i] = 0;
        __syncthreads();
        for (int t = threadIdx.x; t < len; t += SELECT_THREADS) {
            const uint32_t r = rank(t);
            if (shift == 24 || (r >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(r >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int above = 0, v = 255;
            while (v > 0 && above + hist[v] < want) above += hist[v--];
            found[0] = v;
            found[1] = above;
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        want -= found[1];
        __syncthreads();
    }
    // larger ranks, and the first `want` of equal rank
    int base = 0, ties = 0;
    for (int t0 = 0; t0 < len; t0 += SELECT_THREADS) {
        const int t = t0 + threadIdx.x;
        const uint32_t r = t < len ? rank(t) : 0;
        const bool over = t < len && r > prefix, tie = t < len && r == prefix;
        const uint64_t bo = __ballot(over), bt = __ballot(tie);
        const uint64_t below = (1ull << lane) - 1;
        if (lane == 0) {
            wave_sum[wave][0] = __builtin_popcountll(bo);
            wave_sum[wave][1] = __builtin_popcountll(bt);
        }
        __syncthreads();
        int o = base, e = ties, all_o = 0, all_t = 0;
        for (int w = 0; w < SELECT_WAVES; ++w) {
            if (w < wave) {
                o += wave_sum[w][0];
                e += wave_sum[w][1];
            }
            all_o += wave_sum[w][0];
            all_t += wave_sum[w][1];
        }
        o += __builtin_popcountll(bo & below);
        e += __builtin_popcountll(bt & below);
        // what is kept before t: the larger ones, and of the equal ones as many as count
        const int at = o + (e < want ? e : want);
        if (over || (tie && e < want)) {
            keep[at] = t;
            kept[at] = sums[t];
        }
        base += all_o;
        ties += all_t;
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_tree_masks(const int32_t* parents, uint64_t* masks, int32_t* depths, int B, int N,
                             hipStream_t stream) {
    tree_masks_kernel<<<dim3(B), dim3(TREE_MAX_NODES), 0, stream>>>(parents, masks, depths, N);
    return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveParams& a, int pools, hipStream_t stream) {
    move_tokens_kernel<<<dim3(pools, a.H, a.B), dim3(MOVE_THREADS), 0, stream>>>(a);
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

// Weight sums of accepted paths: what attention each cached token got from the path's rows.
//
//   sums[t] += sum over rows of exp(q k_t scale - lse of the row), t up to the row's own token
//
// No V and no softmax state, so a key's sum is one workgroup's: S = Q K^T (32x32x16 MFMA,
// rows by keys), a lane holds one key and 16 of 32 rows.  K goes to LDS as in the tree
// attention.  Up to 32 rows a wave holds them in registers and is bound by K's bytes: 16 x 16K
// keys of 2 heads, 30 rows, 26 to 29 us (4.8 TB/s; 45 with a workgroup's tiles loaded, awaited
// and multiplied once).  Of more rows, each tile reads their queries and statistics again, behind
// the request of the next tile, which it then waits for as well: bound by those loads, 40 / 128 /
// 1536 rows 52 / 90 / 921 us (2.6 TB/s of K; 190, 224 TFLOP/s).
#include "ls_common.h"
#include "ls_tree.h"
#include "ls_tree_load.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

namespace {

constexpr int WEIGH_NW = 2, WEIGH_AHEAD = 1;               // waves, tiles on their way
constexpr int WEIGH_LOADS = 9;                             // of a tile

// A wave has tiles of 32 keys to itself, every gridDim.x * WEIGH_NW-th of a head's; the next
// one and its sums are on their way to the other buffer while one is multiplied.  Four workgroups
// of two waves fill a CU's LDS (16 x 16K / 48 x up to 1.5K keys: 29.1 / 23.0 us; three tiles
// ahead, one workgroup of four waves 30.8 / 29.1, four of one wave 30.4 / 30.6).
struct WeighTile {
    char k[32 * 256];
    float sums[WAVE];
};

__global__ __launch_bounds__(WAVE* WEIGH_NW) void add_weights_kernel(const WeighParams a) {
    __shared__ __attribute__((aligned(1024))) WeighTile ring[WEIGH_NW][WEIGH_AHEAD + 1];
    __shared__ float lse_s[WEIGH_NW][32];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int half = lane >> 5, h = blockIdx.y, b = blockIdx.z;
    const int sum_row = a.sum_rows ? a.sum_rows[b] : b;
    if ((unsigned)sum_row >= (unsigned)a.num_sum_rows) return;
    int len = a.lens[b];
    len = len > 0 ? len : 0;
    int count = a.P;
    if (a.lengths) {
        const int n = a.lengths[b];
        count = n < count ? (n > 0 ? n : 0) : count;
    }
    count = count < len ? count : len;
    int64_t keys64 = (int64_t)a.max_pages * PAGE;
    keys64 = len < keys64 ? len : keys64;
    const int keys = (int)(keys64 < a.sum_len ? keys64 : a.sum_len);       // (at most 2^28)
    const int first = blockIdx.x * WEIGH_NW + wave, stride = gridDim.x * WEIGH_NW;
    const int all = (keys + 31) / 32;
    if (count == 0 || first >= all) return;
    const int tiles = (all - first + stride - 1) / stride;
    const int ctx = len - count;                           // row i sees keys up to ctx + i
    const int rows = count * a.NR;
    float* sums = a.sums + sum_row * a.ss_row + h * a.ss_h;
    const int32_t* table = a.tables + b * a.st_b;

    // pages of 32 of the wave's tiles, two a tile (-1: none), and which are there
    int ids = -1, looked = 0;
    uint64_t there = 0, there_before = 0;
    auto look_up = [&](int i0) {
        const int64_t tile = first + (int64_t)(i0 + lane / 2) * stride, k0 = 32 * tile + 16 * (lane & 1);
        ids = -1;
        if (k0 < keys) ids = table[k0 / PAGE];
        if ((unsigned)ids >= (unsigned)a.num_blocks) ids = -1;
        looked = i0;
        there_before = there;
        there = __ballot(ids >= 0);
    };
    auto request = [&](int i) {
        const int k0 = 32 * (first + i * stride);
        const uint32_t to = (uint32_t)(uintptr_t)(lds_ptr)&ring[wave][i % (WEIGH_AHEAD + 1)];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + p);
            const u4 from = rsrc_of(a.pool + (id >= 0 ? id : 0) * a.sp_b + h * a.sp_h,
                                    id >= 0 ? POOL_BYTES : 0);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const int r = 4 * z + (lane >> 4);
                load_to_lds(from, (uint32_t)(r * a.sp_t) + 16 * ((lane & 15) ^ r), 0,
                            to + 4096 * p + 1024 * z);
            }
        }
        const int n = keys - k0 < 32 ? keys - k0 : 32;
        load_words_to_lds(rsrc_of((const char*)(sums + k0), 4 * n), 4 * lane, to + 8192);
    };

    u4 q[8] = {};
    f4 lv[4] = {};
    // rows r0 and on: a lane holds row lane % 32's queries and the statistics of its 16 rows
    auto take_rows = [&](int r0) {
        const int row = r0 + (lane & 31);
        const int i = row < rows ? row / a.NR : 0, rep = row - i * a.NR;
        int node = row < rows ? (a.path ? a.path[(int64_t)b * a.P + i] : i) : -1;
        if ((unsigned)node >= (unsigned)a.N) node = -1;
        const half_t* p = a.q + b * a.sq_b + (node < 0 ? 0 : node) * a.sq_n + h * a.sq_h +
                          (node < 0 ? 0 : rep) * a.sq_r + 8 * half;
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = node < 0 ? (u4){0, 0, 0, 0} : *(const u4*)(p + 16 * j);
        // (a row that is none, or saw nothing, has no weight)
        float ls = __builtin_inff();
        if (node >= 0) {
            ls = a.lse[((int64_t)(b * a.N + node) * a.H + h) * a.NR + rep] * 1.4426950408889634f;
            if (ls == neg_inf()) ls = __builtin_inff();
        }
        __builtin_amdgcn_wave_barrier();
        lse_s[wave][lane & 31] = ls;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < 4; ++n) lv[n] = *(const f4*)(&lse_s[wave][8 * n + 4 * half]);
        __builtin_amdgcn_wave_barrier();
    };
    // what those rows give the lane's key of a tile
    auto weights = [&](const char* kt, int k0, int r0) {
        const int key = lane & 31;
        f16v s;
#pragma unroll
        for (int n = 0; n < 16; ++n) s[n] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const u4 k = *(const u4*)(kt + key * 256 + 16 * ((2 * j + half) ^ (key & 15)));
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, q[j]),
                                                       __builtin_bit_cast(h8, k), s, 0, 0, 0);
        }
        // key k0 + key is seen by path tokens from k0 + key - ctx on
        const int from = k0 + key - ctx;
        const int seen = from <= 0 ? 0 : (from < a.P ? from * a.NR : rows);
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            const int x = r0 + 8 * (n / 4) + 4 * half + n % 4;
            const float e = lv[n / 4][n % 4];
            const float p = fast_exp2(__builtin_fmaf(s[n], a.scale2, -e));
            // (a row that is none: q of 0 and a key's infinity make a NaN)
            sum += x >= seen && e != __builtin_inff() ? p : 0.f;
        }
        return sum;
    };
    const bool few = rows <= 32;
    look_up(0);
    for (int i = 0; i < WEIGH_AHEAD && i < tiles; ++i) request(i);
    if (few) take_rows(0);
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(q[j]));     // (arrived: no wait in the loop)
    for (int i = 0; i < tiles; ++i) {
        const int next = i + WEIGH_AHEAD;
        if (next < tiles) {
            if (next % 32 == 0) look_up(next);
            request(next);
        }
        if (next < tiles)
            wait_loads<WEIGH_LOADS * WEIGH_AHEAD>();
        else
            wait_loads<0>();
        const WeighTile& t = ring[wave][i % (WEIGH_AHEAD + 1)];
        const int k0 = 32 * (first + i * stride);
        float sum = 0.f;
        if (few)
            sum = weights(t.k, k0, 0);
        else
            for (int r0 = 0; r0 < rows; r0 += 32) {
                take_rows(r0);
                sum += weights(t.k, k0, r0);
            }
        const LanePair p = swap32(sum);
        const uint32_t pages = (uint32_t)((i >= looked ? there : there_before) >> (2 * (i & 31))) & 3;
        const float had = t.sums[lane & 31];
        if (half == 0 && k0 + lane < keys && (pages >> (lane >> 4)) & 1)
            sums[k0 + lane] = had + (p.a + p.b);
        __builtin_amdgcn_s_waitcnt(0xC07F);                // (reads done before the next loads)
        asm volatile("" ::: "memory");
    }
}

}  // namespace

hipError_t launch_add_weights(const WeighParams& a, int64_t keys_bound, hipStream_t stream) {
    // as many workgroups as fit at once, or one a head and sequence
    const int64_t most = (keys_bound + 32 * WEIGH_NW - 1) / (32 * WEIGH_NW);
    int64_t parts = 1024 / ((int64_t)a.H * a.B);
    parts = parts < most ? parts : most;
    if (parts < 1) parts = 1;
    add_weights_kernel<<<dim3((unsigned)parts, a.H, a.B), dim3(WAVE * WEIGH_NW), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace ls

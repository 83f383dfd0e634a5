// Weight sums of accepted paths: what attention each cached token got from the path's rows.
//
//   sums[t] += sum over rows of exp(q k_t scale - lse of the row), t up to the row's own token
//
// No V and no softmax state, so a key's sum is one workgroup's: S = Q K^T (32x32x16 MFMA,
// rows by keys), a lane holds one key and 16 of 32 rows.  K goes to LDS as in the tree
// attention.  Bound by K's bytes.
#include "ls_common.h"
#include "ls_tree.h"

namespace ls {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

namespace {

constexpr int WEIGH_NW = 4, WEIGH_TILES = 2;               // waves, 32-key tiles a wave
constexpr int WEIGH_KEYS = 32 * WEIGH_NW * WEIGH_TILES;    // keys a workgroup

__global__ __launch_bounds__(WAVE* WEIGH_NW) void add_weights_kernel(const WeighParams a) {
    __shared__ __attribute__((aligned(1024))) char kt[WEIGH_NW][WEIGH_TILES][8192];
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
    int64_t keys = (int64_t)a.max_pages * PAGE;
    keys = len < keys ? len : keys;
    keys = keys < a.sum_len ? keys : a.sum_len;
    if (count == 0) return;
    const int64_t ctx = len - count;                       // row i sees keys up to ctx + i
    const int rows = count * a.NR;
    float* sums = a.sums + sum_row * a.ss_row + h * a.ss_h;
    const int32_t* table = a.tables + b * a.st_b;

    // a launch is sized by the expected lengths; longer sequences' keys come in more rounds
    for (int64_t w0 = (int64_t)blockIdx.x * WEIGH_KEYS; w0 < keys; w0 += (int64_t)gridDim.x * WEIGH_KEYS) {
        const int64_t t0 = w0 + wave * (32 * WEIGH_TILES);
        uint32_t ok[WEIGH_TILES];                          // keys that exist, of each tile
#pragma unroll
        for (int z = 0; z < WEIGH_TILES; ++z) {
            ok[z] = 0;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int64_t k0 = t0 + 32 * z + 16 * p;
                int id = -1;
                if (k0 < keys) id = __builtin_amdgcn_readfirstlane(table[k0 / PAGE]);
                if ((unsigned)id >= (unsigned)a.num_blocks) continue;
                const int n = keys - k0 < PAGE ? (int)(keys - k0) : PAGE;
                ok[z] |= ((1u << n) - 1) << (16 * p);
                const char* from = a.pool + id * a.sp_b + h * a.sp_h;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * i + (lane >> 4), pp = lane & 15;
                    __builtin_amdgcn_global_load_lds(
                        (const void __attribute__((address_space(1)))*)(from + r * a.sp_t +
                                                                         16 * (pp ^ r)),
                        (void __attribute__((address_space(3)))*)(kt[wave][z] + 16 * 256 * p + i * 1024),
                        16, 0, 0);
                }
            }
        }
        wait_vm_lds<0>();
        float sum[WEIGH_TILES] = {};
        for (int r0 = 0; r0 < rows; r0 += 32) {
            const int row = r0 + (lane & 31);
            const int i = row < rows ? row / a.NR : 0, rep = row - i * a.NR;
            int node = row < rows ? (a.path ? a.path[(int64_t)b * a.P + i] : i) : -1;
            if ((unsigned)node >= (unsigned)a.N) node = -1;
            u4 q[8];
            {
                const half_t* p = a.q + b * a.sq_b + (node < 0 ? 0 : node) * a.sq_n + h * a.sq_h +
                                  (node < 0 ? 0 : rep) * a.sq_r + 8 * half;
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = node < 0 ? (u4){0, 0, 0, 0} : *(const u4*)(p + 16 * j);
            }
            // (a row that is none, or saw nothing, has no weight)
            float ls = __builtin_inff();
            if (node >= 0) {
                ls = a.lse[((int64_t)(b * a.N + node) * a.H + h) * a.NR + rep] * 1.4426950408889634f;
                if (ls == neg_inf()) ls = __builtin_inff();
            }
            __builtin_amdgcn_wave_barrier();
            lse_s[wave][lane & 31] = ls;
            __builtin_amdgcn_wave_barrier();
            f4 lv[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) lv[n] = *(const f4*)(&lse_s[wave][8 * n + 4 * half]);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int z = 0; z < WEIGH_TILES; ++z) {
                if (ok[z] == 0) continue;
                f16v s;
#pragma unroll
                for (int n = 0; n < 16; ++n) s[n] = 0.f;
                const int key = lane & 31;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const u4 k = *(const u4*)(kt[wave][z] + key * 256 + 16 * ((2 * j + half) ^ (key & 15)));
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, q[j]),
                                                               __builtin_bit_cast(h8, k), s, 0, 0, 0);
                }
                const int64_t k0 = t0 + 32 * z;
                if (k0 + 32 <= ctx + 1) {
                    // (a row that is none: q of 0 and a key's infinity make a NaN)
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        const float e = lv[n / 4][n % 4];
                        const float p = fast_exp2(__builtin_fmaf(s[n], a.scale2, -e));
                        sum[z] += e == __builtin_inff() ? 0.f : p;
                    }
                } else {
                    // key k0 + key is seen by path tokens from k0 + key - ctx on
                    const int64_t from = k0 + key - ctx;
                    const int first = from <= 0 ? 0 : (int)(from < a.P ? from * a.NR : (int64_t)rows);
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        const int x = r0 + 8 * (n / 4) + 4 * half + n % 4;
                        const float e = lv[n / 4][n % 4];
                        const float p = fast_exp2(__builtin_fmaf(s[n], a.scale2, -e));
                        sum[z] += x >= first && e != __builtin_inff() ? p : 0.f;
                    }
                }
            }
        }
#pragma unroll
        for (int z = 0; z < WEIGH_TILES; ++z) {
            const LanePair p = swap32(sum[z]);
            if (half == 0 && (ok[z] >> lane) & 1) sums[t0 + 32 * z + lane] += p.a + p.b;
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);                // (reads done before the next loads)
        asm volatile("" ::: "memory");
    }
}

// The decode's: its scores (log2 units) against its rows' statistics, four keys a thread.
__global__ __launch_bounds__(256) void add_scores_kernel(const TreeParams a) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int sum_row = a.sum_rows ? a.sum_rows[b] : b;
    if ((unsigned)sum_row >= (unsigned)a.num_sum_rows) return;
    int64_t keys = (int64_t)a.max_pages * PAGE;
    const int len = a.lens[b];
    keys = len < keys ? len : keys;
    keys = keys < a.sum_len ? keys : a.sum_len;
    float* sums = a.sums + sum_row * a.ss_row + h * a.ss_h;
    const int64_t unit = (int64_t)b * a.H + h;
    const float* lse = a.lse + unit * a.NR;
    const float* scores = a.scores + unit * a.NR * a.score_len;
    for (int64_t t0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; t0 < keys;
         t0 += (int64_t)gridDim.x * 1024) {
        f4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int r = 0; r < a.NR; ++r) {
            const float e = lse[r] * 1.4426950408889634f;
            if (e == neg_inf()) continue;                  // (it saw nothing)
            const f4 s = *(const f4*)(scores + r * a.score_len + t0);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += fast_exp2(s[i] - e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (t0 + i < keys) sums[t0 + i] += sum[i];
    }
}

}  // namespace

hipError_t launch_add_scores(const TreeParams& a, int64_t keys_bound, hipStream_t stream) {
    int64_t parts = (keys_bound + 1023) / 1024;
    if (parts < 1) parts = 1;
    add_scores_kernel<<<dim3((unsigned)parts, a.H, a.B), dim3(256), 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_add_weights(const WeighParams& a, int64_t keys_bound, hipStream_t stream) {
    int64_t parts = (keys_bound + WEIGH_KEYS - 1) / WEIGH_KEYS;
    if (parts < 1) parts = 1;
    if (parts > 1 << 20) parts = 1 << 20;
    add_weights_kernel<<<dim3((unsigned)parts, a.H, a.B), dim3(WAVE * WEIGH_NW), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace ls

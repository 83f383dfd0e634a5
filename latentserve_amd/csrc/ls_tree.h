// Launch descriptors of the drafted-tree attention, the weight sums and the moves of
// cached tokens (include/latentserve_amd_tree.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ls {

// ---- attention of several new tokens over the fp16 pools --------------------------
constexpr int TREE_MAX_NODES = 256;

// How a launch is cut: a workgroup's nw waves are wr row groups of `rows` rows by nw / wr key
// groups, which take a step's 32 kb keys each.
struct TreeShape {
    int rows, nw, wr, kb;
    int row_tiles;                        // workgroups that share a run of keys
    int groups;                           // runs
};

struct TreeParams {
    const _Float16* q;
    int64_t sq_b, sq_n, sq_h, sq_r;       // strides, elements
    const char* pool[2];                  // K, V
    int64_t sp_b, sp_t, sp_h;             // strides, bytes
    int num_blocks;
    const int32_t* tables;
    int64_t st_b;
    int max_pages;
    const int32_t* lens;
    const uint64_t* masks;                // [B, N, words], or null: a chain
    int words;
    const int32_t* counts;                // [B], or null: N each
    _Float16* out;
    int64_t so_b, so_n, so_h, so_r;
    float* lse;                           // [B, N, H, NR], or null
    float* work;                          // records
    int2* info;                           // [B * H]: first and last group of a unit
    int2* split;                          // [groups], of more units than groups: the unit that a group
                                          // begins and others go on with (-1: none), its last group
    float* scores;                        // [B * H, NR, score_len], or null
    int64_t score_len;
    int score_parts;                      // workgroups that add a unit's scores
    int B, H, N, NR;
    int groups, row_tiles;
    int extra;                            // steps that starting on a unit counts as
    float scale2;                         // softmax scale x log2 e
    // weight sums (with scores)
    float* sums;
    int64_t ss_row, ss_h;
    int64_t sum_len;
    const int32_t* sum_rows;
    int num_sum_rows;
};

constexpr int TREE_EXTRA = 1;
constexpr int TREE_CUS = 256;             // groups of a launch at most

TreeShape tree_shape(int batch, int kv_heads, int rows, int64_t keys_bound);
size_t tree_record_bytes(const TreeShape& s);
// With scores (up to 16 rows, one node): they are kept, and added to the sums as weights.
hipError_t launch_tree_attention(const TreeParams& a, const TreeShape& s, hipStream_t stream);

// ---- weight sums of accepted paths ---------------------------------------------------
struct WeighParams {
    const _Float16* q;
    int64_t sq_b, sq_n, sq_h, sq_r;
    const float* lse;                     // [B, N, H, NR]
    const char* pool;
    int64_t sp_b, sp_t, sp_h;             // bytes
    int num_blocks;
    const int32_t* tables;
    int64_t st_b;
    int max_pages;
    const int32_t* lens;
    float* sums;
    int64_t ss_row, ss_h;
    int64_t sum_len;
    const int32_t* sum_rows;
    int num_sum_rows;
    const int32_t* path;                  // [B, P], or null
    const int32_t* lengths;               // [B], or null
    int B, H, N, P, NR;
    float scale2;
};
hipError_t launch_add_weights(const WeighParams& a, int64_t keys_bound, hipStream_t stream);

// ---- moves of cached tokens -----------------------------------------------------------
constexpr int MOVE_POOLS = 64;            // K and V pools of one launch, in its arguments

struct MoveParams {
    char* pool[MOVE_POOLS];               // K and V of each layer in turn
    int64_t sp_b, sp_t, sp_h;             // bytes
    int num_blocks;
    const int32_t* tables;
    int64_t st_b;
    int max_pages;
    const int32_t* lens;
    int B, H;
    int first_layer;                      // of the launch's pools
    // eviction: keep [layers, B, H, budget]
    const int32_t* keep;
    int budget;
    // acceptance
    const int64_t* tokens;
    const int32_t* parents;
    const int64_t* choices;
    const int32_t* counts;
    int32_t* path;
    int32_t* lengths;
    int64_t* next;
    int N;
};
hipError_t launch_move_tokens(const MoveParams& a, int pools, hipStream_t stream);
hipError_t launch_accept_tokens(const MoveParams& a, int pools, hipStream_t stream);
hipError_t launch_tree_masks(const int32_t* parents, uint64_t* masks, int32_t* depths, int B, int N,
                             hipStream_t stream);

struct SelectParams {
    const float* sums;
    int64_t ss_l, ss_b, ss_h;
    int64_t sum_len;
    const int32_t* lens;
    int32_t* keep;
    float* kept;
    int L, B, H, budget, sinks, recent;
};
hipError_t launch_select_tokens(const SelectParams& a, hipStream_t stream);

}  // namespace ls

// The kernels of gqa_tree_decode: arguments and launchers.
#pragma once

#include "tree_common.cuh"

namespace gqa {

constexpr int kTreeTileKeys = 128;  // keys of a place in the cut of tree_cut.cuh

struct TreeArgs {
    TreeCache cache;
    const void* q;
    const void* k_cache;
    const void* v_cache;
    void* out;
    const uint32_t* mask;  // [batch][tokens][words] or null: a causal run
    float* workspace;      // partial records
    int4* cut_units;       // [ctas][2], behind the records: the unit a CTA starts and does not finish
    int64_t q_stride;      // elements between tokens of q
    int32_t batch;
    int32_t num_q_heads;
    int32_t num_kv_heads;
    int32_t group;
    float scale_log2;      // log2(e) / sqrt(head_dim)
    // Filled by the launchers:
    int32_t tile_tokens;   // tokens whose heads fill a query tile
    int32_t tile_rows;     // rows of a query tile in a record
    int32_t ctas;          // the keys of all units are cut over this many CTAs
    // BF16:
    int32_t box_keys;      // rows per bulk copy of K and V
    int32_t box_tokens;    // tokens per bulk copy of q
    int32_t head_first;    // order of the middle coordinates of the cache maps
};

// Whether node t sees node j (both below the sequence's n).
__device__ __forceinline__ bool tree_sees(const uint32_t* mask, int64_t row, int words, int t, int j) {
    if (mask == nullptr) return j <= t;
    return (__ldg(mask + row * words + (j >> 5)) >> (j & 31)) & 1u;
}

size_t tree_attention_workspace(int32_t tokens, int32_t group, int32_t ctas);  // BF16
int launch_tree_attention(TreeArgs a, const gqa_kv_layout& layout, int32_t sm_count, cudaStream_t stream);
size_t tree_rows_workspace(int32_t tokens, int32_t group, int32_t ctas);  // FP32
int launch_tree_rows(TreeArgs a, int32_t sm_count, cudaStream_t stream);

}  // namespace gqa

// What the operators of tree-drafted decoding share: a sequence's place in the cache, checks of the
// cache description, tensor maps.
#pragma once

#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/gqa_b200.h"
#include "decode_kernels.cuh"
#include "work_map.cuh"

namespace gqa {

constexpr int kTreeMaxTokens = GQA_TREE_MAX_TOKENS;

// Cache addressing and lengths as the kernels of a tree step see them (strides in elements).
struct TreeCache {
    const int32_t* seq_lens;     // [batch], history + nodes
    const int32_t* tree_sizes;   // [batch] nodes, or null: `tokens` everywhere
    const int32_t* block_table;  // null: every sequence reads block `fixed_block`
    int32_t* status;
    int64_t stride_block;
    int64_t stride_token;
    int64_t stride_head;
    int32_t tokens;
    int32_t blocks_per_seq;
    int32_t block_tokens;
    int32_t fixed_block;
    int32_t num_blocks;
    int32_t capacity;  // positions a sequence can hold
};

// Sequence b: n nodes in slots [base, base + n). Not ok: out of range, to be skipped.
struct TreeSpan {
    int32_t base;
    int32_t n;
    bool ok;
};

__device__ __forceinline__ void raise_bad_input(int32_t* status) {
    if (status != nullptr) atomicExch(status, kStatusBadInput);
}

__device__ __forceinline__ TreeSpan tree_span(const TreeCache& c, int b) {
    const int32_t len = __ldg(c.seq_lens + b);
    TreeSpan s;
    s.n = c.tree_sizes != nullptr ? __ldg(c.tree_sizes + b) : c.tokens;
    s.ok = s.n >= 0 && s.n <= c.tokens && len >= s.n && len <= c.capacity;
    s.base = len - s.n;
    if (!s.ok) s.n = 0;
    return s;
}

// Element offset of head 0 of `slot` of sequence b; false when the block table names no block.
__device__ __forceinline__ bool tree_row(const TreeCache& c, int b, int32_t slot, int64_t* offset) {
    int32_t blk = c.fixed_block;
    if (c.block_table != nullptr) {
        const int32_t lb = slot / c.block_tokens;
        slot -= lb * c.block_tokens;
        blk = __ldg(c.block_table + (int64_t)b * c.blocks_per_seq + lb);
    }
    *offset = (int64_t)blk * c.stride_block + (int64_t)slot * c.stride_token;
    return (uint32_t)blk < (uint32_t)c.num_blocks;
}

// Checks of the cache description common to the tree operators (host); fills *out.
struct TreeCacheDesc {
    int32_t dtype;
    int32_t batch;
    int32_t tokens;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t blocks_per_seq;
    int32_t fixed_block;
    const gqa_kv_layout* layout;
    const void* k_cache;
    const void* v_cache;
    const int32_t* seq_lens_dev;
    const int32_t* tree_sizes_dev;
    const int32_t* block_table_dev;
    int32_t* status_dev;
};
int tree_cache_args(const TreeCacheDesc& d, TreeCache* out);

// Whether n rows of `bytes` bytes, a_step apart from a on, share a byte with those b_step apart from b on (steps of
// `bytes` at least; host). Two comparisons unless the spans meet.
inline bool rows_overlap(const void* a, int64_t a_step, const void* b, int64_t b_step, int64_t n, int64_t bytes) {
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    if (a0 + (n - 1) * a_step + bytes <= b0 || b0 + (n - 1) * b_step + bytes <= a0) return false;
    for (int64_t i = 0, j = 0; i < n && j < n;) {
        const uintptr_t row_a = a0 + i * a_step, row_b = b0 + j * b_step;
        if (row_a + bytes <= row_b) {
            ++i;
        } else if (row_b + bytes <= row_a) {
            ++j;
        } else {
            return true;
        }
    }
    return false;
}

// Tensor maps of the tree attention kernel, encoded anew for every call. The cache as (channel,
// token / head by ascending stride, block) with boxes of box_keys rows x 64 channels of one head; the
// queries as (channel, head, row of tokens) with boxes of 64 channels x group heads x box_tokens.
int tree_cache_map(const void* base, const gqa_kv_layout& l, int32_t num_kv_heads, int32_t box_keys,
                   bool* head_before_token, CUtensorMap* map);
int tree_query_map(const void* base, int64_t rows, int64_t token_stride, int32_t num_q_heads,
                   int32_t group, int32_t box_tokens, CUtensorMap* map);
int current_sm_count(int32_t* out);

}  // namespace gqa

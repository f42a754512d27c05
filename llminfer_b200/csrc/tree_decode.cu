// Attention of a tree of drafted tokens over the cache (gqa_tree_decode): the C entry. The kernels are in
// tree_attention.cu (BF16) and tree_rows.cu (FP32).
#include <cmath>
#include <cstring>

#include "ptx.cuh"
#include "tree_attention.cuh"

namespace gqa {
namespace {

constexpr int kMaxGroup = 8;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool shape_ok(int32_t dtype, int32_t batch, int32_t tokens, int32_t num_q_heads, int32_t num_kv_heads) {
    return (dtype == GQA_DTYPE_F32 || dtype == GQA_DTYPE_BF16) && batch > 0 && batch <= kMaxRaggedBatch &&
           tokens > 0 && tokens <= kTreeMaxTokens && num_q_heads > 0 && num_kv_heads > 0 &&
           num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads <= kMaxGroup;
}

}  // namespace
}  // namespace gqa

extern "C" {

size_t gqa_tree_workspace_bytes(int32_t dtype, int32_t batch, int32_t tokens, int32_t num_q_heads,
                                int32_t num_kv_heads, int32_t sm_count) {
    if (!gqa::shape_ok(dtype, batch, tokens, num_q_heads, num_kv_heads)) return 0;
    if (sm_count <= 0 && gqa::current_sm_count(&sm_count) != GQA_OK) return 0;
    const int32_t group = num_q_heads / num_kv_heads;
    return dtype == GQA_DTYPE_F32 ? gqa::tree_rows_workspace(tokens, group, sm_count)
                                  : gqa::tree_attention_workspace(tokens, group, sm_count);
}

int gqa_tree_decode(const gqa_tree_decode_params* p) {
    using namespace gqa;
    if (p == nullptr) return GQA_ERR_NULL;
    TreeArgs a;
    std::memset(&a, 0, sizeof(a));
    const TreeCacheDesc d = {p->dtype, p->batch, p->tokens, p->num_kv_heads, p->head_dim,
                             p->blocks_per_seq, p->fixed_block, &p->layout, p->k_cache, p->v_cache,
                             p->seq_lens_dev, p->tree_sizes_dev, p->block_table_dev, p->status_dev};
    const int rc = tree_cache_args(d, &a.cache);
    if (rc != GQA_OK) return rc;
    if (p->num_q_heads <= 0 || p->num_q_heads % p->num_kv_heads != 0) return GQA_ERR_SHAPE;
    if (!shape_ok(p->dtype, p->batch, p->tokens, p->num_q_heads, p->num_kv_heads)) {
        return GQA_ERR_UNSUPPORTED;
    }
    // Keys are counted up to the end of a tile in 32 bits.
    if (a.cache.capacity > INT32_MAX - kTreeTileKeys) return GQA_ERR_SHAPE;
    if (p->q == nullptr || p->out == nullptr || p->workspace == nullptr) return GQA_ERR_NULL;
    const int64_t eb = p->dtype == GQA_DTYPE_F32 ? 4 : 2;
    const int64_t q_row = (int64_t)p->num_q_heads * kHeadDim;
    a.q_stride = p->q_token_stride != 0 ? p->q_token_stride : q_row;
    if (a.q_stride < q_row) return GQA_ERR_SHAPE;
    if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->workspace) || a.q_stride * eb % 16) {
        return GQA_ERR_ALIGN;
    }
    // Rows of one head are written while others are still to be read.
    if (rows_overlap(p->q, a.q_stride * eb, p->out, q_row * eb, (int64_t)p->batch * p->tokens, q_row * eb)) {
        return GQA_ERR_UNSUPPORTED;
    }
    int32_t sms = 0;
    if (current_sm_count(&sms) != GQA_OK) return GQA_ERR_CUDA;
    if (p->workspace_bytes < gqa_tree_workspace_bytes(p->dtype, p->batch, p->tokens, p->num_q_heads,
                                                      p->num_kv_heads, sms)) {
        return GQA_ERR_WORKSPACE;
    }
    a.q = p->q;
    a.k_cache = p->k_cache;
    a.v_cache = p->v_cache;
    a.out = p->out;
    a.mask = p->mask_dev;
    a.num_q_heads = p->num_q_heads;
    a.num_kv_heads = p->num_kv_heads;
    a.group = p->num_q_heads / p->num_kv_heads;
    a.scale_log2 = (1.0f / std::sqrt((float)kHeadDim)) * 1.44269504088896340736f;
    a.batch = p->batch;
    a.workspace = static_cast<float*>(p->workspace);
    if (p->num_kv_heads > 65535) return GQA_ERR_SHAPE;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(p->stream);
    return p->dtype == GQA_DTYPE_BF16 ? launch_tree_attention(a, p->layout, sms, stream)
                                      : launch_tree_rows(a, sms, stream);
}

}  // extern "C"

// Attention of a tree of drafted tokens over the cache (gqa_tree_decode): C entry and the FP32 kernel on
// CUDA cores (the BF16 kernel is in tree_attention.cu).
//
// Node t of sequence b sees the history (positions < base) and the nodes its mask row names; keys a row
// does not see are never used, so their rows may hold anything. tree_rows_kernel: one CTA per (sequence,
// node, KV head), kWarps warps that take chunks of 32 keys in turn; a lane scores one key against the
// group's queries (kept in shared memory), then the warp adds p v with four channels per lane.
// Running maximum and sum are FP32 in the exp2 domain; the warps are merged at the end.
#include <cuda_bf16.h>

#include <cmath>
#include <cstring>

#include "ptx.cuh"
#include "tree_attention.cuh"

namespace gqa {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxGroup = 8;

__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

__global__ void __launch_bounds__(kWarps * 32) tree_rows_kernel(const TreeArgs a) {
    __shared__ float s_q[kMaxGroup][kHeadDim];
    __shared__ float s_o[kWarps][kMaxGroup][kHeadDim];
    __shared__ float s_m[kWarps][kMaxGroup], s_l[kWarps][kMaxGroup];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    pdl_launch_dependents();
    pdl_wait();
    const TreeSpan span = tree_span(a.cache, b);
    if (!span.ok && t == 0 && hk == 0 && threadIdx.x == 0) raise_bad_input(a.cache.status);
    if (t >= span.n) return;
    const int group = a.group;
    const int words = (a.cache.tokens + 31) / 32;
    const int64_t row = (int64_t)b * a.cache.tokens + t;
    for (int i = threadIdx.x; i < group * kHeadDim / 4; i += kWarps * 32) {
        float x[4];
        load4(static_cast<const float*>(a.q) + row * a.q_stride + (int64_t)hk * group * kHeadDim + i * 4, x);
#pragma unroll
        for (int c = 0; c < 4; ++c) (&s_q[0][0])[i * 4 + c] = x[c] * a.scale_log2;
    }
    __syncthreads();

    float m[kMaxGroup], l[kMaxGroup], o[kMaxGroup][4];
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
        o[g][0] = o[g][1] = o[g][2] = o[g][3] = 0.0f;
    }
    const int len = span.base + span.n;
    for (int k0 = warp * 32; k0 < len; k0 += kWarps * 32) {
        const int key = k0 + lane;
        bool sees = key < len && (key < span.base || tree_sees(a.mask, row, words, t, key - span.base));
        int64_t off = 0;
        if (sees && !tree_row(a.cache, b, key, &off)) {
            raise_bad_input(a.cache.status);
            sees = false;
        }
        off += (int64_t)hk * a.cache.stride_head;
        float s[kMaxGroup];
#pragma unroll
        for (int g = 0; g < kMaxGroup; ++g) s[g] = 0.0f;
        if (sees) {
            const float* kp = static_cast<const float*>(a.k_cache) + off;
#pragma unroll 4
            for (int d = 0; d < kHeadDim; d += 4) {
                float x[4];
                load4(kp + d, x);
#pragma unroll
                for (int g = 0; g < kMaxGroup; ++g) {
                    if (g < group) {
                        const float4 qv = *reinterpret_cast<const float4*>(&s_q[g][d]);
                        s[g] += x[0] * qv.x + x[1] * qv.y + x[2] * qv.z + x[3] * qv.w;
                    }
                }
            }
        }
        float p[kMaxGroup];
#pragma unroll
        for (int g = 0; g < kMaxGroup; ++g) {
            p[g] = 0.0f;
            if (g >= group) continue;
            float top = sees ? s[g] : -INFINITY;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float next = fmaxf(m[g], top);
            const float ref = safe_max(next);
            const float alpha = exp2f(m[g] - ref);
            m[g] = next;
            p[g] = sees ? exp2f(s[g] - ref) : 0.0f;
            l[g] = l[g] * alpha + p[g];
#pragma unroll
            for (int c = 0; c < 4; ++c) o[g][c] *= alpha;
        }
        uint32_t todo = __ballot_sync(0xffffffffu, sees);
        while (todo != 0) {
            const int j = __ffs(todo) - 1;
            todo &= todo - 1;
            const int64_t at = __shfl_sync(0xffffffffu, off, j);
            float x[4];
            load4(static_cast<const float*>(a.v_cache) + at + lane * 4, x);
#pragma unroll
            for (int g = 0; g < kMaxGroup; ++g) {
                if (g < group) {
                    const float pj = __shfl_sync(0xffffffffu, p[g], j);
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[g][c] += pj * x[c];
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
        if (g >= group) continue;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], d);
        if (lane == 0) {
            s_m[warp][g] = m[g];
            s_l[warp][g] = l[g];
        }
        *reinterpret_cast<float4*>(&s_o[warp][g][lane * 4]) = make_float4(o[g][0], o[g][1], o[g][2], o[g][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < group * kHeadDim / 4; i += kWarps * 32) {
        const int g = i / (kHeadDim / 4);
        const int d = (i - g * (kHeadDim / 4)) * 4;
        float top = -INFINITY;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][g]);
        const float ref = safe_max(top);
        float sum = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(s_m[w][g] - ref);
            sum += s_l[w][g] * f;
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] += s_o[w][g][d + c] * f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = sum == 0.0f ? 0.0f : y[c] / sum;
        store4(static_cast<float*>(a.out) + (row * a.num_q_heads + (int64_t)hk * group + g) * kHeadDim + d, y);
    }
}

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
    if (dtype == GQA_DTYPE_F32) return 16;
    if (sm_count <= 0 && gqa::current_sm_count(&sm_count) != GQA_OK) return 0;
    return gqa::tree_attention_workspace(tokens, num_q_heads / num_kv_heads, sm_count);
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
    if (p->q == nullptr || p->out == nullptr || p->workspace == nullptr) return GQA_ERR_NULL;
    const int64_t eb = p->dtype == GQA_DTYPE_F32 ? 4 : 2;
    const int64_t q_row = (int64_t)p->num_q_heads * kHeadDim;
    a.q_stride = p->q_token_stride != 0 ? p->q_token_stride : q_row;
    if (a.q_stride < q_row) return GQA_ERR_SHAPE;
    if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->workspace) || a.q_stride * eb % 16) {
        return GQA_ERR_ALIGN;
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
    if (p->dtype == GQA_DTYPE_BF16) return launch_tree_attention(a, p->layout, sms, stream);
    const dim3 grid((unsigned)p->tokens, (unsigned)p->num_kv_heads, (unsigned)p->batch);
    const cudaError_t e = launch_pdl(tree_rows_kernel, grid, dim3(kWarps * 32), 0, stream, a);
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"

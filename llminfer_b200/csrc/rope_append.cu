// Rotary positions with the KV append of a tree's nodes (gqa_rope_append): optional per-head RMS norm,
// rotation of the first rotary_dim channels in either pairing, queries to q_out, keys and values to
// their cache slots. Cache slot (history + node) and rotary position (history + depth) are apart.
//
// Mathematics. theta = position * freq_i is a product of up to 2^17 and 1, of which only the part
// inside one turn matters: in FP32 the product alone is off by 2^-24 * theta (0.008 rad at position
// 131072). Here turns = position * (freq_i / 2 pi) is FP64, its nearest integer is taken off, and the
// rest (|r| <= 1/2, exact to 2^-36 turns at that position) goes to sincospif(2 r) in FP32. Norm and rotation are
// FP32, the only rounding to the row type is the store.
//
// A warp takes one token and walks over some of its heads: lane l holds channels 4 l .. 4 l + 3, so
// that a head is one coalesced row (256 bytes in BF16) and the lane's angles serve every head. In the half pairing
// the partner of channel i is i + rotary_dim / 2, i.e. the lane rotary_dim / 8 further on: one
// shuffle per channel; interleaved pairs lie inside the lane. The kernel is bound by bytes (rows
// in, rows out); heads are loaded kBatch at a time so that enough of them are in flight.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kWarps = 8;
constexpr int kBatch = 4;  // heads in flight per warp

struct RopeArgs {
    TreeCache cache;
    const void* q;
    void* q_out;
    const void* k_new;
    const void* v_new;
    const void* weight;  // [2][128] or null
    const double* freq;
    const int32_t* depth;  // [batch][tokens] or null
    void* k_cache;
    void* v_cache;
    int64_t q_stride;
    int64_t q_out_stride;
    int64_t k_stride;
    int64_t v_stride;
    int32_t num_q_heads;
    int32_t num_kv_heads;
    int32_t rotary_dim;
    int32_t heads_per_warp;
    float eps;
    float attn_factor;
};

__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    x[0] = bf16_lo_to_f32(u.x);
    x[1] = bf16_hi_to_f32(u.x);
    x[2] = bf16_lo_to_f32(u.y);
    x[3] = bf16_hi_to_f32(u.y);
}
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

// grid.x: groups of kWarps warps over the heads of a token (queries, keys, values in this order);
// grid.y * grid.z: tokens.
template <typename T, bool HALF, bool NORM>
__global__ void __launch_bounds__(kWarps * 32) rope_append_kernel(const RopeArgs a, int32_t nodes) {
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    const int heads = a.num_q_heads + 2 * a.num_kv_heads;
    const int first = (blockIdx.x * kWarps + warp) * a.heads_per_warp;
    const int bt = blockIdx.z * gridDim.y + blockIdx.y;
    const int rot_lanes = a.rotary_dim >> 2;   // lanes that hold rotated channels
    const int half_lanes = a.rotary_dim >> 3;  // distance of the partner lane (half pairing)
    // Turns per position of this lane's pairs; the frequencies are the caller's constants, but a
    // kernel ahead in the stream may still be writing them.
    pdl_wait();
    if (bt >= nodes || first >= heads) return;
    const int b = bt / a.cache.tokens;
    const int t = bt - b * a.cache.tokens;
    const TreeSpan span = tree_span(a.cache, b);
    if (!span.ok && t == 0 && first == 0 && lane == 0) raise_bad_input(a.cache.status);
    if (t >= span.n) return;
    int64_t row = 0;
    const bool placed = tree_row(a.cache, b, span.base + t, &row);
    if (!placed && first == 0 && lane == 0) raise_bad_input(a.cache.status);

    constexpr int kAngles = HALF ? 4 : 2;
    float cs[kAngles], sn[kAngles];
    if (lane < rot_lanes) {
        const int pos = span.base + (a.depth != nullptr ? __ldg(a.depth + bt) : t);
        const int pair = HALF ? (lane < half_lanes ? lane : lane - half_lanes) * 4 : lane * 2;
#pragma unroll
        for (int i = 0; i < kAngles; ++i) {
            const double turns = (double)pos * (__ldg(a.freq + pair + i) * 0.15915494309189533577);
            const float r = (float)(turns - rint(turns));
            sincospif(2.0f * r, &sn[i], &cs[i]);
            sn[i] *= a.attn_factor;
            cs[i] *= a.attn_factor;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kAngles; ++i) { cs[i] = 1.0f; sn[i] = 0.0f; }
    }
    const bool upper = lane >= half_lanes;
    const int partner = lane < rot_lanes ? (upper ? lane - half_lanes : lane + half_lanes) : lane;

    const int end = min(heads, first + a.heads_per_warp);
#pragma unroll 1
    for (int h0 = first; h0 < end; h0 += kBatch) {
        float x[kBatch][4];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + i;
            if (h >= end) continue;
            const T* src;
            if (h < a.num_q_heads) {
                src = static_cast<const T*>(a.q) + bt * a.q_stride + h * kHeadDim;
            } else if (h < a.num_q_heads + a.num_kv_heads) {
                src = static_cast<const T*>(a.k_new) + bt * a.k_stride + (h - a.num_q_heads) * kHeadDim;
            } else {
                src = static_cast<const T*>(a.v_new) + bt * a.v_stride +
                      (h - a.num_q_heads - a.num_kv_heads) * kHeadDim;
            }
            load4(src + lane * 4, x[i]);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + i;
            if (h >= end) continue;
            const bool is_q = h < a.num_q_heads;
            const int hk = is_q ? 0 : (h - a.num_q_heads) % a.num_kv_heads;
            if (h < a.num_q_heads + a.num_kv_heads) {
                if (NORM) {
                    float sum = 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) sum += x[i][c] * x[i][c];
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    const float scale = rsqrtf(sum * (1.0f / kHeadDim) + a.eps);
                    float w[4];
                    load4(static_cast<const T*>(a.weight) + (is_q ? 0 : kHeadDim) + lane * 4, w);
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[i][c] = x[i][c] * scale * w[c];
                }
                float y[4];
                if (HALF) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float other = __shfl_sync(0xffffffffu, x[i][c], partner);
                        // lower half: x cos - other sin; upper half: other sin + x cos
                        y[c] = x[i][c] * cs[c % kAngles] + (upper ? other : -other) * sn[c % kAngles];
                        if (lane >= rot_lanes) y[c] = x[i][c];
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        y[2 * c] = x[i][2 * c] * cs[c] - x[i][2 * c + 1] * sn[c];
                        y[2 * c + 1] = x[i][2 * c] * sn[c] + x[i][2 * c + 1] * cs[c];
                        if (lane >= rot_lanes) { y[2 * c] = x[i][2 * c]; y[2 * c + 1] = x[i][2 * c + 1]; }
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) x[i][c] = y[c];
            }
            if (is_q) {
                store4(static_cast<T*>(a.q_out) + bt * a.q_out_stride + h * kHeadDim + lane * 4, x[i]);
            } else if (placed) {
                void* cache = h < a.num_q_heads + a.num_kv_heads ? a.k_cache : a.v_cache;
                store4(static_cast<T*>(cache) + row + hk * a.cache.stride_head + lane * 4, x[i]);
            }
        }
    }
}

template <typename T>
cudaError_t launch(const RopeArgs& a, int32_t nodes, bool half, dim3 grid, cudaStream_t stream) {
    auto kernel = half ? (a.weight != nullptr ? rope_append_kernel<T, true, true>
                                              : rope_append_kernel<T, true, false>)
                       : (a.weight != nullptr ? rope_append_kernel<T, false, true>
                                              : rope_append_kernel<T, false, false>);
    return launch_pdl(kernel, grid, dim3(kWarps * 32), 0, stream, a, nodes);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace gqa

extern "C" int gqa_rope_append(const gqa_rope_params* p) {
    using namespace gqa;
    if (p == nullptr) return GQA_ERR_NULL;
    if (p->num_q_heads <= 0) return GQA_ERR_SHAPE;
    RopeArgs a;
    std::memset(&a, 0, sizeof(a));
    const TreeCacheDesc d = {p->dtype, p->batch, p->tokens, p->num_kv_heads, p->head_dim,
                             p->blocks_per_seq, p->fixed_block, &p->layout, p->k_cache, p->v_cache,
                             p->seq_lens_dev, p->tree_sizes_dev, p->block_table_dev, p->status_dev};
    const int rc = tree_cache_args(d, &a.cache);
    if (rc != GQA_OK) return rc;
    if (p->q == nullptr || p->q_out == nullptr || p->k_new == nullptr || p->v_new == nullptr ||
        p->freq_dev == nullptr) {
        return GQA_ERR_NULL;
    }
    if (p->rotary_dim < 8 || p->rotary_dim > kHeadDim || p->rotary_dim % 8 != 0) return GQA_ERR_SHAPE;
    if (p->style != GQA_ROPE_HALF && p->style != GQA_ROPE_INTERLEAVED) return GQA_ERR_UNSUPPORTED;
    const int64_t eb = p->dtype == GQA_DTYPE_F32 ? 4 : 2;
    const int64_t q_row = (int64_t)p->num_q_heads * kHeadDim, kv_row = (int64_t)p->num_kv_heads * kHeadDim;
    a.q_stride = p->q_token_stride != 0 ? p->q_token_stride : q_row;
    a.q_out_stride = p->q_out_token_stride != 0 ? p->q_out_token_stride : q_row;
    a.k_stride = p->k_token_stride != 0 ? p->k_token_stride : kv_row;
    a.v_stride = p->v_token_stride != 0 ? p->v_token_stride : kv_row;
    if (a.q_stride < q_row || a.q_out_stride < q_row || a.k_stride < kv_row || a.v_stride < kv_row) {
        return GQA_ERR_SHAPE;
    }
    if (a.q_stride * eb % 16 || a.q_out_stride * eb % 16 || a.k_stride * eb % 16 || a.v_stride * eb % 16 ||
        !aligned16(p->q) || !aligned16(p->q_out) || !aligned16(p->k_new) || !aligned16(p->v_new) ||
        !aligned16(p->qk_weight) || (reinterpret_cast<uintptr_t>(p->freq_dev) & 7u) != 0) {
        return GQA_ERR_ALIGN;
    }
    // In place means row on row: with another stride a warp would overwrite rows not yet read.
    if (p->q == p->q_out && a.q_stride != a.q_out_stride) return GQA_ERR_SHAPE;
    a.q = p->q;
    a.q_out = p->q_out;
    a.k_new = p->k_new;
    a.v_new = p->v_new;
    a.weight = p->qk_weight;
    a.freq = p->freq_dev;
    a.depth = p->depth_dev;
    a.k_cache = p->k_cache;
    a.v_cache = p->v_cache;
    a.num_q_heads = p->num_q_heads;
    a.num_kv_heads = p->num_kv_heads;
    a.rotary_dim = p->rotary_dim;
    a.eps = p->eps;
    a.attn_factor = p->attn_factor;
    int32_t sms = 0;
    if (current_sm_count(&sms) != GQA_OK) return GQA_ERR_CUDA;
    const int64_t nodes = (int64_t)p->batch * p->tokens;
    const int32_t heads = p->num_q_heads + 2 * p->num_kv_heads;
    // One head per warp while that does not fill the GPU's 64 warps per SM; then more, so that the angles of
    // a token are computed once for several heads.
    const int64_t per = nodes * heads / ((int64_t)sms * 64);
    a.heads_per_warp = per >= 2 * kBatch ? 2 * kBatch : (per >= kBatch ? kBatch : (per >= 2 ? 2 : 1));
    const int64_t cols = (heads + kWarps * a.heads_per_warp - 1) / (kWarps * a.heads_per_warp);
    const int64_t gy = nodes < 32768 ? nodes : 32768, gz = (nodes + gy - 1) / gy;
    if (gz > 65535) return GQA_ERR_SHAPE;
    const dim3 grid((unsigned)cols, (unsigned)gy, (unsigned)gz);
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(p->stream);
    const bool half = p->style == GQA_ROPE_HALF;
    const cudaError_t e = p->dtype == GQA_DTYPE_F32
                              ? launch<float>(a, (int32_t)nodes, half, grid, stream)
                              : launch<__nv_bfloat16>(a, (int32_t)nodes, half, grid, stream);
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

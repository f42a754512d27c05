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
// A block takes a token and some or all of its heads. Its threads compute the token's angles once, one pair each,
// into shared memory; a warp then walks over its heads two at a time, 16 lanes per head. A lane holds two
// groups of four channels: in the half pairing i .. i + 3 and their partners i + rotary_dim / 2 .., so that a rotation
// stays inside the lane, else eight neighbours. (With one head per warp, partners fetched by
// shuffles, the kernel was bound by instruction issue at 44 us for 3072 tokens of 80 heads, 0.43 of the measured copy
// bandwidth.) The rows' addresses need neither lengths nor angles, so a warp asks for its kBatch
// pairs of heads before it looks at either.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kBatch = 4;      // pairs of heads of a warp, all in flight
constexpr int kMaxWarps = 16;  // of a block

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
    int32_t heads_per_block;
    float eps;
    float attn_factor;
};

// Four channels as they lie in memory.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> { using type = uint2; };
template <> struct Raw<float> { using type = float4; };

__device__ __forceinline__ void unpack(uint2 u, float (&x)[4]) {
    x[0] = bf16_lo_to_f32(u.x);
    x[1] = bf16_hi_to_f32(u.x);
    x[2] = bf16_lo_to_f32(u.y);
    x[3] = bf16_hi_to_f32(u.y);
}
__device__ __forceinline__ void unpack(float4 u, float (&x)[4]) {
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
}
__device__ __forceinline__ void pack(const float (&x)[4], uint2* u) {
    *u = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}
__device__ __forceinline__ void pack(const float (&x)[4], float4* u) {
    *u = make_float4(x[0], x[1], x[2], x[3]);
}

// grid.x: parts of a token's heads (queries, keys, values in this order); grid.y * grid.z: tokens.
template <typename T, bool HALF, bool NORM>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) rope_append_kernel(const RopeArgs a, int32_t nodes) {
    using R = typename Raw<T>::type;
    __shared__ float s_cos[kHeadDim / 2], s_sin[kHeadDim / 2];
    __shared__ float s_weight[NORM ? 2 * kHeadDim : 1];
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int warps = blockDim.x >> 5;
    const int heads = a.num_q_heads + 2 * a.num_kv_heads;
    const int keys_at = a.num_q_heads, values_at = a.num_q_heads + a.num_kv_heads;
    const int bt = blockIdx.z * gridDim.y + blockIdx.y;
    pdl_launch_dependents();
    if (bt >= nodes) return;
    const int end = min(heads, (int)(blockIdx.x + 1) * a.heads_per_block);
    const int mine = blockIdx.x * a.heads_per_block + 2 * warp + (lane >> 4);  // this half warp's first head
    // The lane's channels: g0 .. g0 + 3 and g1 .. g1 + 3.
    const int l = lane & 15;
    const bool rotated = l < (a.rotary_dim >> 3);
    const int g0 = HALF && rotated ? 4 * l : 8 * l;
    const int g1 = HALF && rotated ? g0 + (a.rotary_dim >> 1) : g0 + 4;
    pdl_wait();

    R x[kBatch][2];
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + 2 * i * warps;
            if (h >= end) continue;
            const T* src = h < keys_at ? static_cast<const T*>(a.q) + bt * a.q_stride + h * kHeadDim
                           : h < values_at
                               ? static_cast<const T*>(a.k_new) + bt * a.k_stride + (h - keys_at) * kHeadDim
                               : static_cast<const T*>(a.v_new) + bt * a.v_stride + (h - values_at) * kHeadDim;
            x[i][0] = *reinterpret_cast<const R*>(src + g0);
            x[i][1] = *reinterpret_cast<const R*>(src + g1);
        }
    };
    load(mine);
    const int b = bt / a.cache.tokens;
    const int t = bt - b * a.cache.tokens;
    const int pairs = a.rotary_dim >> 1;
    double freq = 0.0;
    if ((int)threadIdx.x < pairs) freq = __ldg(a.freq + threadIdx.x);
    const int ahead = a.depth != nullptr ? __ldg(a.depth + bt) : t;
    if (NORM) {
        for (int i = threadIdx.x; i < 2 * kHeadDim / 4; i += blockDim.x) {
            float w[4];
            unpack(*reinterpret_cast<const R*>(static_cast<const T*>(a.weight) + 4 * i), w);
            *reinterpret_cast<float4*>(s_weight + 4 * i) = make_float4(w[0], w[1], w[2], w[3]);
        }
    }
    const TreeSpan span = tree_span(a.cache, b);
    if (!span.ok && t == 0 && blockIdx.x == 0 && threadIdx.x == 0) raise_bad_input(a.cache.status);
    if (t >= span.n) return;
    int64_t row = 0;
    const bool placed = tree_row(a.cache, b, span.base + t, &row);
    if (!placed && blockIdx.x == 0 && threadIdx.x == 0) raise_bad_input(a.cache.status);
    if ((int)threadIdx.x < pairs) {
        const double turns = (double)(span.base + ahead) * (freq * 0.15915494309189533577);
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        s_cos[threadIdx.x] = cs * a.attn_factor;
        s_sin[threadIdx.x] = sn * a.attn_factor;
    }
    __syncthreads();
    // The four pairs of the lane (channels that are not rotated turn by nothing).
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = rotated ? s_cos[4 * l + i] : 1.0f;
        sn[i] = rotated ? s_sin[4 * l + i] : 0.0f;
    }

#pragma unroll 1
    for (int h0 = mine; h0 - (lane >> 4) < end; h0 += 2 * kBatch * warps) {
        if (h0 != mine) load(h0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + 2 * i * warps;
            const bool is_q = h < keys_at;
            float scale = 1.0f;
            float v[2][4];
            unpack(x[i][0], v[0]);
            unpack(x[i][1], v[1]);
            if (NORM) {
                // Both halves of the warp take part, whatever their heads are.
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) sum += v[0][c] * v[0][c] + v[1][c] * v[1][c];
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                scale = rsqrtf(sum * (1.0f / kHeadDim) + a.eps);
            }
            if (h >= end) continue;
            if (h < values_at) {
                if (NORM) {
                    const float* w = s_weight + (is_q ? 0 : kHeadDim);
                    const float4 w0 = *reinterpret_cast<const float4*>(w + g0);
                    const float4 w1 = *reinterpret_cast<const float4*>(w + g1);
                    v[0][0] *= scale * w0.x; v[0][1] *= scale * w0.y; v[0][2] *= scale * w0.z; v[0][3] *= scale * w0.w;
                    v[1][0] *= scale * w1.x; v[1][1] *= scale * w1.y; v[1][2] *= scale * w1.z; v[1][3] *= scale * w1.w;
                }
                float y[2][4];
                if (HALF) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        y[0][c] = v[0][c] * cs[c] - v[1][c] * sn[c];
                        y[1][c] = v[0][c] * sn[c] + v[1][c] * cs[c];
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int g = c >> 1, at = 2 * (c & 1);
                        y[g][at] = v[g][at] * cs[c] - v[g][at + 1] * sn[c];
                        y[g][at + 1] = v[g][at] * sn[c] + v[g][at + 1] * cs[c];
                    }
                }
                pack(y[0], &x[i][0]);
                pack(y[1], &x[i][1]);
            }
            T* dst;
            if (is_q) {
                dst = static_cast<T*>(a.q_out) + bt * a.q_out_stride + h * kHeadDim;
            } else if (placed) {
                dst = row + (h < values_at ? static_cast<T*>(a.k_cache) + (h - keys_at) * a.cache.stride_head
                                           : static_cast<T*>(a.v_cache) + (h - values_at) * a.cache.stride_head);
            } else {
                continue;
            }
            *reinterpret_cast<R*>(dst + g0) = x[i][0];
            *reinterpret_cast<R*>(dst + g1) = x[i][1];
        }
    }
}

template <typename T>
cudaError_t launch(const RopeArgs& a, int32_t nodes, bool half, dim3 grid, int threads, cudaStream_t stream) {
    auto kernel = half ? (a.weight != nullptr ? rope_append_kernel<T, true, true>
                                              : rope_append_kernel<T, true, false>)
                       : (a.weight != nullptr ? rope_append_kernel<T, false, true>
                                              : rope_append_kernel<T, false, false>);
    return launch_pdl(kernel, grid, dim3((unsigned)threads), 0, stream, a, nodes);
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
    // Up to kBatch pairs of heads per warp and 16 warps per block, i.e. a block per token for up to 128 heads;
    // where the tokens alone do not fill the GPU (32 warps per SM) they are cut by heads, down to a pair
    // per warp, in blocks of four warps that spread over the SMs.
    const int64_t pairs = (heads + 1) / 2;
    int64_t per_warp = nodes * pairs / ((int64_t)sms * 32);
    per_warp = per_warp < 1 ? 1 : (per_warp > kBatch ? kBatch : per_warp);
    int64_t warps = (pairs + per_warp - 1) / per_warp;
    int64_t cols = per_warp < kBatch ? (warps + 3) / 4 : (warps + kMaxWarps - 1) / kMaxWarps;
    if (cols * kMaxWarps < warps) cols = (warps + kMaxWarps - 1) / kMaxWarps;
    warps = (warps + cols - 1) / cols;
    a.heads_per_block = (int32_t)(2 * ((pairs + cols - 1) / cols));
    cols = (heads + a.heads_per_block - 1) / a.heads_per_block;
    warps = warps < 2 ? 2 : warps;  // the angles take 64 threads
    const int64_t gy = nodes < 32768 ? nodes : 32768, gz = (nodes + gy - 1) / gy;
    if (gz > 65535) return GQA_ERR_SHAPE;
    const dim3 grid((unsigned)cols, (unsigned)gy, (unsigned)gz);
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(p->stream);
    const bool half = p->style == GQA_ROPE_HALF;
    const cudaError_t e = p->dtype == GQA_DTYPE_F32
                              ? launch<float>(a, (int32_t)nodes, half, grid, (int)warps * 32, stream)
                              : launch<__nv_bfloat16>(a, (int32_t)nodes, half, grid, (int)warps * 32, stream);
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

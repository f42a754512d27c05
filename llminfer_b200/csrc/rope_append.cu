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
// stays inside the lane, else eight neighbours. The rows' addresses need neither lengths nor angles, so
// a warp asks for all its heads before it looks at either.
//
// Measured: 64 sequences of up to 64 nodes (48 on average), 64 / 8 heads, BF16, norm: 32 us, 3.9 TB/s of rows read and
// written (0.59 of a copy); bound by the life of a block (load, angles, norm, store) at the 25 warps per SM that 80
// registers leave. Fewer heads per warp: 34 us with 8, 36 with 2; 8 nodes of 32 / 8 heads: 2.5 - 2.9 us, a launch.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kMaxWarps = 8;  // of a block
// Pairs of heads of a warp, all in flight: 128 bytes a lane.
template <typename T> constexpr int kPairs = 32 / (int)sizeof(T) / 2;

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
    int32_t batch;
    int32_t num_q_heads;
    int32_t num_kv_heads;
    int32_t rotary_dim;
    int32_t pairs_per_warp;  // pairs of heads, kPairs at most
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

// grid.x: parts of a token's heads (queries, keys, values in this order); grid.y: tokens; grid.z: sequences.
template <typename T, bool HALF, bool NORM>
__global__ void __launch_bounds__(kMaxWarps * 32, 3) rope_append_kernel(const RopeArgs a) {
    using R = typename Raw<T>::type;
    constexpr int kBatch = kPairs<T>;
    __shared__ float s_cos[kHeadDim / 2], s_sin[kHeadDim / 2];
    __shared__ float s_weight[NORM ? 2 * kHeadDim : 1];
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int heads = a.num_q_heads + 2 * a.num_kv_heads;
    const int keys_at = a.num_q_heads, values_at = a.num_q_heads + a.num_kv_heads;
    const int b = blockIdx.z, t = blockIdx.y;
    const int bt = b * a.cache.tokens + t;
    pdl_launch_dependents();
    const int end = min(heads, (int)(blockIdx.x + 1) * a.heads_per_block);
    // This half warp's heads: mine, mine + 2, ... (pairs_per_warp of them, the warps side by side).
    const int mine = blockIdx.x * a.heads_per_block + 2 * a.pairs_per_warp * warp + (lane >> 4);
    // The lane's channels: g0 .. g0 + 3 and g1 .. g1 + 3.
    const int l = lane & 15;
    const bool rotated = l < (a.rotary_dim >> 3);
    const int g0 = HALF && rotated ? 4 * l : 8 * l;
    const int g1 = HALF && rotated ? g0 + (a.rotary_dim >> 1) : g0 + 4;
    // Head h of the token lies at the base of its kind + 128 h.
    const T* q_in = static_cast<const T*>(a.q) + bt * a.q_stride;
    const T* k_in = static_cast<const T*>(a.k_new) + bt * a.k_stride - keys_at * kHeadDim;
    const T* v_in = static_cast<const T*>(a.v_new) + bt * a.v_stride - values_at * kHeadDim;
    pdl_wait();

    R x[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const int h = mine + 2 * i;
        if (h >= end || i >= a.pairs_per_warp) continue;
        const T* src = (h < keys_at ? q_in : h < values_at ? k_in : v_in) + h * kHeadDim;
        x[i][0] = *reinterpret_cast<const R*>(src + g0);
        x[i][1] = *reinterpret_cast<const R*>(src + g1);
    }
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
    if ((int)threadIdx.x < pairs) {
        const double turns = (double)(span.base + ahead) * (freq * 0.15915494309189533577);
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        s_cos[threadIdx.x] = cs * a.attn_factor;
        s_sin[threadIdx.x] = sn * a.attn_factor;
    }
    // Queries go to q_out; keys and values to the token's cache row, if it has a block.
    T* k_out = nullptr;
    T* v_out = nullptr;
    const int last = mine - (lane >> 4) + 2 * a.pairs_per_warp - 1;  // of the warp
    if (last >= keys_at) {
        int64_t row = 0;
        if (tree_row(a.cache, b, span.base + t, &row)) {
            k_out = static_cast<T*>(a.k_cache) + row;
            v_out = static_cast<T*>(a.v_cache) + row;
        } else if (lane == 0) {
            raise_bad_input(a.cache.status);
        }
    }
    T* q_out = static_cast<T*>(a.q_out) + bt * a.q_out_stride;
    __syncthreads();
    if (mine - (lane >> 4) >= end) return;

    // Coefficients of the lane's four pairs with the norm's weights in them, for queries or keys:
    // y_a = v_a ca + v_c sc, y_c = v_a sa + v_c cc. Channels that are not rotated turn by nothing. Two pairs at once:
    // packed arithmetic, since a large launch is bound by the instructions it issues.
    Two ca[2], sa[2], sc[2], cc[2];
    auto coefficients = [&](bool for_q) {
        float wa[4] = {1.0f, 1.0f, 1.0f, 1.0f}, wc[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (NORM) {
            const float* w = s_weight + (for_q ? 0 : kHeadDim);
            const float4 w0 = *reinterpret_cast<const float4*>(w + g0);
            const float4 w1 = *reinterpret_cast<const float4*>(w + g1);
            if (HALF) {
                wa[0] = w0.x; wa[1] = w0.y; wa[2] = w0.z; wa[3] = w0.w;
                wc[0] = w1.x; wc[1] = w1.y; wc[2] = w1.z; wc[3] = w1.w;
            } else {
                wa[0] = w0.x; wa[1] = w0.z; wa[2] = w1.x; wa[3] = w1.z;
                wc[0] = w0.y; wc[1] = w0.w; wc[2] = w1.y; wc[3] = w1.w;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float c0 = rotated ? s_cos[4 * l + i] : 1.0f, s0 = rotated ? s_sin[4 * l + i] : 0.0f;
            const float c1 = rotated ? s_cos[4 * l + i + 1] : 1.0f, s1 = rotated ? s_sin[4 * l + i + 1] : 0.0f;
            ca[i / 2] = two_of(c0 * wa[i], c1 * wa[i + 1]);
            sa[i / 2] = two_of(s0 * wa[i], s1 * wa[i + 1]);
            sc[i / 2] = two_of(-s0 * wc[i], -s1 * wc[i + 1]);
            cc[i / 2] = two_of(c0 * wc[i], c1 * wc[i + 1]);
        }
    };
    bool for_q = mine < keys_at;
    coefficients(for_q);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        if (i >= a.pairs_per_warp) break;
        const int h = mine + 2 * i;
        if (h - (lane >> 4) < values_at) {  // the same for the warp: its lower head is rotated
            float v[2][4];
            unpack(x[i][0], v[0]);
            unpack(x[i][1], v[1]);
            // The pairs' members: channels g0 + c and g1 + c, or neighbours.
            Two va[2], vc[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                va[k] = HALF ? two_of(v[0][2 * k], v[0][2 * k + 1]) : two_of(v[k][0], v[k][2]);
                vc[k] = HALF ? two_of(v[1][2 * k], v[1][2 * k + 1]) : two_of(v[k][1], v[k][3]);
            }
            float scale = 1.0f;
            if (NORM) {
                // Both halves of the warp take part, whatever their heads are.
                const Two squares = fma2(va[0], va[0], fma2(va[1], va[1], fma2(vc[0], vc[0], mul2(vc[1], vc[1]))));
                float lo, hi;
                split(squares, &lo, &hi);
                float sum = lo + hi;
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                scale = rsqrtf(sum * (1.0f / kHeadDim) + a.eps);
                if (for_q != (h < keys_at)) {  // the first key behind queries
                    for_q = false;
                    coefficients(false);
                }
            }
            if (h < values_at && h < end && (NORM || rotated)) {  // else as it came, infinities too
                const Two both = two_of(scale, scale);
                float y[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    Two ya = fma2(va[k], ca[k], mul2(vc[k], sc[k]));
                    Two yc = fma2(va[k], sa[k], mul2(vc[k], cc[k]));
                    if (NORM) {
                        ya = mul2(ya, both);
                        yc = mul2(yc, both);
                    }
                    if (HALF) {
                        split(ya, &y[0][2 * k], &y[0][2 * k + 1]);
                        split(yc, &y[1][2 * k], &y[1][2 * k + 1]);
                    } else {
                        split(ya, &y[k][0], &y[k][2]);
                        split(yc, &y[k][1], &y[k][3]);
                    }
                }
                pack(y[0], &x[i][0]);
                pack(y[1], &x[i][1]);
            }
        }
        if (h >= end) continue;
        T* dst;
        if (h < keys_at) {
            dst = q_out + h * kHeadDim;
        } else {
            const bool key = h < values_at;
            dst = (key ? k_out : v_out) + (h - (key ? keys_at : values_at)) * a.cache.stride_head;
            if (k_out == nullptr) continue;
        }
        *reinterpret_cast<R*>(dst + g0) = x[i][0];
        *reinterpret_cast<R*>(dst + g1) = x[i][1];
    }
}

template <typename T>
cudaError_t launch(RopeArgs a, bool half, int32_t heads, int32_t sms, cudaStream_t stream) {
    // kPairs pairs of heads per warp, so that angles and coefficients serve several, and a block per token
    // where that is 8 warps at most; where the tokens alone do not fill the GPU (32 warps per SM) fewer
    // pairs per warp, in blocks of two warps (the angles take 64 threads) that spread over the SMs.
    const int64_t pairs = (heads + 1) / 2;
    const int64_t share = (int64_t)a.batch * a.cache.tokens * pairs / ((int64_t)sms * 32);
    a.pairs_per_warp = share < 1 ? 1 : (share > kPairs<T> ? kPairs<T> : (int32_t)share);
    const int per_warp = 2 * a.pairs_per_warp;
    int warps = (heads + per_warp - 1) / per_warp;
    const int cols = a.pairs_per_warp == kPairs<T> ? (warps + kMaxWarps - 1) / kMaxWarps : (warps + 1) / 2;
    warps = (warps + cols - 1) / cols;
    warps = warps < 2 ? 2 : warps;
    a.heads_per_block = warps * per_warp;
    const dim3 grid((unsigned)((heads + a.heads_per_block - 1) / a.heads_per_block), (unsigned)a.cache.tokens,
                    (unsigned)a.batch);
    auto kernel = half ? (a.weight != nullptr ? rope_append_kernel<T, true, true>
                                              : rope_append_kernel<T, true, false>)
                       : (a.weight != nullptr ? rope_append_kernel<T, false, true>
                                              : rope_append_kernel<T, false, false>);
    return launch_pdl(kernel, grid, dim3((unsigned)warps * 32), 0, stream, a);
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
    if (p->q != p->q_out && rows_overlap(p->q, a.q_stride * eb, p->q_out, a.q_out_stride * eb,
                                         (int64_t)p->batch * p->tokens, q_row * eb)) {
        return GQA_ERR_UNSUPPORTED;
    }
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
    if (p->batch > 65535) return GQA_ERR_SHAPE;
    a.batch = p->batch;
    const int32_t heads = p->num_q_heads + 2 * p->num_kv_heads;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(p->stream);
    const bool half = p->style == GQA_ROPE_HALF;
    const cudaError_t e = p->dtype == GQA_DTYPE_F32 ? launch<float>(a, half, heads, sms, stream)
                                                    : launch<__nv_bfloat16>(a, half, heads, sms, stream);
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

// Tree attention in FP32 on CUDA cores (gqa_tree_decode, FP32).
//
// Mathematics. As in the BF16 kernel: tiles of query rows (a unit's tokens times the group, 16, 32 or 64 rows, whichever
// holds them) against tiles of 64 keys, S = Q K^T, P = 2^(S - m) with a running maximum m and sum l per row,
// O = O 2^(m' - m) + P V; all of it FP32, the scale and log2(e) multiplied into Q.
//
// Layout. 8 warps; a warp owns RT rows, a lane of them the scores of the keys `lane` and lane + 32 and the output channels
// 4 lane .. + 3. 512 bytes of K or V take four cycles to load from shared memory, the same 16 bytes of Q or P for
// all lanes one or two, so a warp spans keys and channels and holds several rows: 167 us in a graph for 8 nodes of 32 / 8 heads
// over 32768 keys, 949 for 64. (Half warps of 16 keys with rows of their own took 197 and 910: slower for few rows, faster
// for many; one layout was kept, the one of the small trees.)
// Maximum and P stay inside the warp. Products are packed pairs of FP32 (over channels in S, over output
// channels in O). K and V tiles come by cp.async, two tiles deep; rows are padded to 132 floats, which
// spreads 8 of them over all banks. Bound by shared memory and its latency at two warps per scheduler: 64 nodes
// over 32768 keys run at 36 TFLOP/s, half of what the FP32 units could do; 8 nodes at a quarter of the memory's rate.
//
// Work. The flat sequence of key tiles of all units, cut evenly over one CTA per SM, as for BF16.
//
// Masks. Only tiles that reach the nodes look at the mask; a key that a row does not see gets the weight -1,
// which the second product skips: K and V may hold anything there.
#include <cmath>
#include <mutex>

#include "ptx.cuh"
#include "tree_attention.cuh"
#include "tree_cut.cuh"

namespace gqa {
namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;                 // of a tile; a place of the cut is kTile keys
constexpr int kPitch = kHeadDim + 4;      // floats between rows in shared memory
constexpr int kStages = 2;

template <int RT>
struct Shape {
    static constexpr int kRows = 8 * RT;
    static constexpr int kQ = kRows * kPitch;
    static constexpr int kStage = 2 * kKeys * kPitch;  // K, then V
    static constexpr int kWeights = kKeys * kRows;  // [warp][key][row of the warp]
    static constexpr size_t kBytes = (size_t)(kQ + kStages * kStage + kWeights) * sizeof(float);
};

// 16 bytes to shared memory, zeros when `some` is false (the source is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool some) {
    const uint32_t bytes = some ? 16u : 0u;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_all_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

struct Four {
    Two a, b;
};
__device__ __forceinline__ Four load_four(const float* p) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p);
    return Four{Two{u.x}, Two{u.y}};
}

// N neighbouring floats.
__device__ __forceinline__ void load_rows(const float* p, float (&x)[2]) {
    const float2 u = *reinterpret_cast<const float2*>(p);
    x[0] = u.x; x[1] = u.y;
}
template <int N>
__device__ __forceinline__ void load_rows(const float* p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 u = *reinterpret_cast<const float4*>(p + i);
        x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w;
    }
}
__device__ __forceinline__ void store_rows(float* p, const float (&x)[2]) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
}
template <int N>
__device__ __forceinline__ void store_rows(float* p, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
}

// O += P V over the keys of a tile; MASKED: weights below zero are keys the row does not see.
template <int RT, bool MASKED>
__device__ __forceinline__ void add_values(const float* weights, const float* values, Two (&o)[RT][2]) {
#pragma unroll 8
    for (int key = 0; key < kKeys; ++key) {
        const Four v = load_four(values + key * kPitch);
        float w[RT];
        load_rows(weights + key * RT, w);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (MASKED && w[i] < 0.0f) continue;
            const Two ww = two_of(w[i], w[i]);
            o[i][0] = fma2(ww, v.a, o[i][0]);
            o[i][1] = fma2(ww, v.b, o[i][1]);
        }
    }
}

template <int RT>
__global__ void __launch_bounds__(kThreads, 1) tree_rows_kernel(const TreeArgs a) {
    using S = Shape<RT>;
    extern __shared__ __align__(16) float smem[];
    float* s_q = smem;
    float* s_kv = s_q + S::kQ;
    float* s_w = s_kv + kStages * S::kStage;
    const Tables tables = tables_at(reinterpret_cast<int32_t*>(s_w + S::kWeights), a.batch);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    build_tables<1>(a, tables);
    float* weights = s_w + warp * kKeys * RT;
    const Cut cut = cut_of(a, tables, 1);
    int pos = cut.begin(blockIdx.x);
    const int pos_end = cut.begin(blockIdx.x + 1);
    const int words = (a.cache.tokens + 31) / 32;
    int last_cta = -1;  // of the unit this CTA starts and others finish
    Piece p;
    while (next_piece<1>(a, tables, &pos, pos_end, &p)) {
        if (tid == 0 && !p.whole && p.tile == 0) {
            last_cta = cut.owner(p.u.place + kUnitPad + p.u.tiles - 1);
            a.cut_units[2 * blockIdx.x] = make_int4(last_cta, p.u.b, p.u.hk, p.u.token0);
            a.cut_units[2 * blockIdx.x + 1] = make_int4(p.u.tokens, 0, 0, 0);
        }
        const int base = p.u.len - p.u.n;
        const int key_first = p.tile * kTile;
        const int key_end = min(p.u.len, (p.tile + p.tiles) * kTile);
        const int steps = ceil_div(key_end - key_first, kKeys);
        const int64_t row0 = (int64_t)p.u.b * a.cache.tokens + p.u.token0;  // the unit's first token
        auto load = [&](int j) {
            // The warp's 8 keys: lane i finds the row of key 8 i + warp, then a row goes by in 32 copies.
            int64_t off = -1;
            if (lane < kKeys / 8) {
                const int key = key_first + j * kKeys + 8 * lane + warp;
                if (key < key_end && !tree_row(a.cache, p.u.b, key, &off)) {
                    raise_bad_input(a.cache.status);
                    off = -1;
                }
            }
            float* stage = s_kv + (j % kStages) * S::kStage;
#pragma unroll
            for (int i = 0; i < kKeys / 8; ++i) {
                const int64_t from = __shfl_sync(0xffffffffu, off, i);
                const int64_t at = (from < 0 ? 0 : from + p.u.hk * a.cache.stride_head) + lane * 4;
                const uint32_t to = smem_u32(stage + (8 * i + warp) * kPitch + lane * 4);
                copy16(to, static_cast<const float*>(a.k_cache) + at, from >= 0);
                copy16(to + kKeys * kPitch * 4, static_cast<const float*>(a.v_cache) + at, from >= 0);
            }
        };
        __syncthreads();  // the last piece's tiles have been read
        load(0);
        copies_end_group();
        for (int i = tid; i < S::kRows * (kHeadDim / 4); i += kThreads) {
            const int row = i / (kHeadDim / 4), d = i % (kHeadDim / 4) * 4;
            const int t = row / a.group, g = row - t * a.group;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (t < p.u.tokens) {
                x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (row0 + t) * a.q_stride +
                                                     (int64_t)(p.u.hk * a.group + g) * kHeadDim + d);
            }
            x.x *= a.scale_log2; x.y *= a.scale_log2; x.z *= a.scale_log2; x.w *= a.scale_log2;
            *reinterpret_cast<float4*>(s_q + row * kPitch + d) = x;
        }
        float m[RT], l[RT];
        Two o[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) o[i][k] = two_of(0.0f, 0.0f);
        }
        for (int j = 0; j < steps; ++j) {
            if (j + 1 < steps) load(j + 1);
            copies_end_group();
            copies_wait_all_but_one();
            __syncthreads();
            const float* keys = s_kv + (j % kStages) * S::kStage;
            const float* values = keys + kKeys * kPitch + 4 * lane;
            const int key0 = key_first + j * kKeys;
            const bool tail = key0 + kKeys > base;

            Two s2[RT][2];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int k = 0; k < 2; ++k) s2[i][k] = two_of(0.0f, 0.0f);
            }
#pragma unroll 4
            for (int d = 0; d < kHeadDim; d += 4) {
                Four q[RT], k[2];
#pragma unroll
                for (int i = 0; i < RT; ++i) q[i] = load_four(s_q + (warp * RT + i) * kPitch + d);
#pragma unroll
                for (int i = 0; i < 2; ++i) k[i] = load_four(keys + (lane + 32 * i) * kPitch + d);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) s2[i][n] = fma2(q[i].b, k[n].b, fma2(q[i].a, k[n].a, s2[i][n]));
                }
            }
            float w[2][RT];  // scores, then weights
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float lo, hi;
                    split(s2[i][n], &lo, &hi);
                    w[n][i] = lo + hi;
                }
            }
            uint32_t unseen = 0;  // bit 2 i + n
            if (tail) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const int t = (warp * RT + i) / a.group;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int key = key0 + lane + 32 * n;
                        const bool sees = t < p.u.tokens && key < p.u.len &&
                                          (key < base || tree_sees(a.mask, row0 + t, words, p.u.token0 + t, key - base));
                        if (!sees) {
                            unseen |= 1u << (2 * i + n);
                            w[n][i] = -INFINITY;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                float top = fmaxf(w[0][i], w[1][i]);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                if (top > m[i]) {
                    const float alpha = exp2f(m[i] - safe_max(top));
                    m[i] = top;
                    l[i] *= alpha;
                    const Two f = two_of(alpha, alpha), zero = two_of(0.0f, 0.0f);
#pragma unroll
                    for (int k = 0; k < 2; ++k) o[i][k] = fma2(o[i][k], f, zero);
                }
                const float ref = safe_max(m[i]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    w[n][i] = exp2f(w[n][i] - ref);
                    l[i] += w[n][i];
                    if (unseen >> (2 * i + n) & 1u) w[n][i] = -1.0f;
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) store_rows(weights + (lane + 32 * n) * RT, w[n]);
            __syncwarp();
            if (tail) {
                add_values<RT, true>(weights, values, o);
            } else {
                add_values<RT, false>(weights, values, o);
            }
            __syncthreads();
        }
        // ---- the end of the piece --------------------------------------------------------------------
        float* rec = a.workspace + (int64_t)(2 * blockIdx.x + (p.tile == 0 ? 1 : 0)) * a.tile_rows * kRecordCols;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = warp * RT + i;
            const int t = row / a.group, g = row - t * a.group;
            float sum = l[i];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (t >= p.u.tokens) continue;
            float4 x;
            split(o[i][0], &x.x, &x.y);
            split(o[i][1], &x.z, &x.w);
            if (p.whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                *reinterpret_cast<float4*>(static_cast<float*>(a.out) +
                                           ((row0 + t) * a.num_q_heads + p.u.hk * a.group + g) * kHeadDim + 4 * lane) =
                    make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            } else {
                *reinterpret_cast<float4*>(rec + (lane * a.tile_rows + row) * 4) = x;
                if (lane == 0) {
                    rec[kHeadDim * a.tile_rows + row] = m[i];
                    rec[(kHeadDim + 1) * a.tile_rows + row] = sum;
                }
            }
        }
    }
    if (tid == 0 && last_cta < 0) a.cut_units[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
}

// The smallest of 16, 32 and 64 rows that holds all rows, else 64.
int tile_rows_of(int32_t tokens, int32_t group) {
    const int rows = tokens * group;
    return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

template <int RT>
int launch(const TreeArgs& a, cudaStream_t stream) {
    const size_t smem = Shape<RT>::kBytes + table_bytes(a.batch);
    auto kernel = tree_rows_kernel<RT>;
    {
        static std::mutex mu;
        static size_t configured[64] = {};
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GQA_ERR_CUDA;
        std::lock_guard<std::mutex> lock(mu);
        if (configured[dev] < smem) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
                return GQA_ERR_CUDA;
            }
            configured[dev] = smem;
        }
    }
    if (launch_pdl(kernel, dim3(a.ctas), dim3(kThreads), smem, stream, a) != cudaSuccess) return GQA_ERR_CUDA;
    return launch_merge<1, float>(a, stream) == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

size_t record_bytes(int32_t tokens, int32_t group, int32_t ctas) {
    return (size_t)2 * ctas * tile_rows_of(tokens, group) * kRecordCols * sizeof(float);
}

}  // namespace

size_t tree_rows_workspace(int32_t tokens, int32_t group, int32_t ctas) {
    return record_bytes(tokens, group, ctas) + 2 * (size_t)ctas * sizeof(int4);
}

int launch_tree_rows(TreeArgs a, int32_t sm_count, cudaStream_t stream) {
    a.ctas = sm_count;
    a.cut_units = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(a.workspace) +
                                          record_bytes(a.cache.tokens, a.group, sm_count));
    a.tile_rows = tile_rows_of(a.cache.tokens, a.group);
    a.tile_tokens = a.tile_rows / a.group;
    // Places are 32-bit numbers.
    const int64_t per_seq = (int64_t)(ceil_div(a.cache.capacity, kTile) + kUnitPad) * a.num_kv_heads *
                            ceil_div(a.cache.tokens, a.tile_tokens);
    if (per_seq * a.batch > (1 << 30)) return GQA_ERR_SHAPE;
    return a.tile_rows == 16 ? launch<2>(a, stream) : a.tile_rows == 32 ? launch<4>(a, stream) : launch<8>(a, stream);
}

}  // namespace gqa

// Verification of a drafted tree against the target's probabilities (gqa_tree_verify).
//
// Mathematics. Rejecting child after child of one node takes the residual of a residual:
// r_0 = p, r_{k+1} = max(r_k - q, 0) / s_{k+1}. Multiplied out, r_k S_k = max(p - c_k q, 0) with S_0 = 1,
// c_0 = 0, c_{k+1} = c_k + S_k and S_k the sum of max(p - c_k q, 0) over the vocabulary: one scalar replaces the
// chain, and a rejection costs one pass over the rows p and q of that node. Accepted nodes cost no row
// at all, only p and q at the child's token, which are fetched for every node of the tree before
// the walk starts. Tests and sums are FP64: p, q and u are FP32 or BF16 values, so u q is exact and the
// outcome does not depend on how the sum was cut.
//
// One thread-block cluster per sequence; the CTAs take equal slices of the vocabulary, the warps of
// a CTA contiguous segments of its slice. Every CTA walks the tree itself (same inputs, same sums,
// same steps); after a pass the CTAs read one another's partial sums through distributed shared
// memory. To place the sample, the partial sums name the segment in which the cumulative sum
// passes u S, and one warp walks that segment again.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kWords = kTreeMaxTokens / 32;

struct VerifyArgs {
    const void* target;
    const void* draft;
    const int32_t* words;    // the nodes' tokens
    const int32_t* parents;
    const float* u_accept;
    const float* u_sample;
    const int32_t* tree_sizes;
    int32_t* path;
    int32_t* kept;
    int32_t* next_token;
    int32_t* status;
    int64_t target_seq, target_node, draft_seq, draft_node;
    int32_t batch;
    int32_t tokens;
    int32_t vocab;
    int32_t cluster;
};

__device__ __forceinline__ float value(const float* p) { return __ldg(p); }
__device__ __forceinline__ float value(const __nv_bfloat16* p) {
    return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
}
// 16 bytes of a row.
__device__ __forceinline__ void vector_of(const float* p, float (&x)[4]) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
}
__device__ __forceinline__ void vector_of(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo_to_f32(w[i]);
        x[2 * i + 1] = bf16_hi_to_f32(w[i]);
    }
}

// max(p - c q, 0); NaN and negative entries count as 0, and q counts as 0 where it is no number.
__device__ __forceinline__ double rest_of(float p, float q, double c) {
    return fmax(fma(-c, (double)fmaxf(q, 0.0f), (double)fmaxf(p, 0.0f)), 0.0);
}

// Where the walk stands.
struct Walk {
    int node;       // current node
    int tried;      // its last tried child (or the node itself)
    int count;      // nodes on the path
    int rejected;   // children of `node` rejected so far
    int pass;       // 1: the sum of the residual is needed, 0: the walk has ended
    int last;       // no child is left: the sum is for the sample
    double c;
    double sum;
};

// What a CTA tells its cluster after a pass. The steps must agree: if inputs change under the
// kernel, CTAs that walked apart see it here, all at once, and leave together instead of waiting
// for one another at the next barrier.
struct Said {
    double sum;
    uint64_t step;
};
__device__ __forceinline__ Said ld_cluster_said(uint32_t addr) {
    Said v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v.sum) : "r"(addr) : "memory");
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v.step) : "r"(addr + 8) : "memory");
    return v;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kThreads) tree_verify_kernel(const VerifyArgs a) {
    constexpr int VE = 16 / (int)sizeof(T);
    __shared__ uint32_t s_child[kTreeMaxTokens][kWords];
    __shared__ float s_p[kTreeMaxTokens], s_q[kTreeMaxTokens], s_u[kTreeMaxTokens];
    __shared__ int32_t s_word[kTreeMaxTokens];
    __shared__ int32_t s_path[kTreeMaxTokens];
    __shared__ int32_t s_gone[kTreeMaxTokens];  // rejected tokens (draft without probabilities)
    __shared__ double s_warp[kWarps];
    __shared__ Said s_said[2];  // this CTA's sum and step, buffers in turn: read by the whole cluster
    __shared__ Walk w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % a.cluster;
    const int b = blockIdx.x / a.cluster;
    pdl_launch_dependents();
    pdl_wait();
    int n = a.tree_sizes != nullptr ? __ldg(a.tree_sizes + b) : a.tokens;
    bool bad = n < 0 || n > a.tokens;
    if (bad) n = 0;
    const T* target = static_cast<const T*>(a.target) + b * a.target_seq;
    const T* draft = DRAFT ? static_cast<const T*>(a.draft) + b * a.draft_seq : nullptr;

    // ---- children and the values at the drafted tokens ----------------------------------------
    for (int i = tid; i < kTreeMaxTokens * kWords; i += kThreads) (&s_child[0][0])[i] = 0;
    __syncthreads();
    if (tid > 0 && tid < n) {
        const int par = __ldg(a.parents + (int64_t)b * a.tokens + tid);
        const int word = __ldg(a.words + (int64_t)b * a.tokens + tid);
        s_word[tid] = word;
        s_u[tid] = __ldg(a.u_accept + (int64_t)b * a.tokens + tid);
        if (par >= 0 && par < tid && word >= 0 && word < a.vocab) {
            s_p[tid] = fmaxf(value(target + par * a.target_node + word), 0.0f);
            s_q[tid] = DRAFT ? fmaxf(value(draft + par * a.draft_node + word), 0.0f) : 1.0f;
            atomicOr(&s_child[par][tid >> 5], 1u << (tid & 31));
        } else {
            bad = true;
        }
    }
    if (tid == 0) w = Walk{0, 0, 1, 0, 0, 0, 0.0, 1.0};
    if (tid < kTreeMaxTokens) s_path[tid] = -1;
    bad = __syncthreads_or(bad);
    if (bad && rank == 0 && tid == 0) raise_bad_input(a.status);

    const T* p_row = target;
    const T* q_row = draft;
    int turn = 0;
    double total = 0.0;      // sum of the residual after the last pass
    double before = 0.0;     // of the CTAs before this one
    double own = 0.0;
    bool later = false;      // a CTA after this one has something in its slice
    // This CTA's and warp's vectors of 16 bytes. A vector is cut at the row's ends, where single
    // elements are read; rows p and q that are not equally aligned are read element by element.
    int vec_lo = 0, vec_hi = 0, shift = 0;
    bool wide = false;

    auto set_rows = [&](int node) {
        p_row = target + node * a.target_node;
        if (DRAFT) q_row = draft + node * a.draft_node;
        shift = (int)((reinterpret_cast<uintptr_t>(p_row) & 15u) / sizeof(T));
        wide = !DRAFT || ((reinterpret_cast<uintptr_t>(p_row) ^ reinterpret_cast<uintptr_t>(q_row)) & 15u) == 0;
        const int64_t vecs = (a.vocab + shift + VE - 1) / VE;
        const int64_t lo = vecs * rank / a.cluster, hi = vecs * (rank + 1) / a.cluster;
        vec_lo = (int)(lo + (hi - lo) * warp / kWarps);
        vec_hi = (int)(lo + (hi - lo) * (warp + 1) / kWarps);
    };
    // The residual at the elements of vector `vec`; elements outside the row are 0.
    auto residual = [&](int vec, double c, int rejected, double (&r)[VE]) {
        const int e0 = vec * VE - shift;
        float p[VE], q[VE];
        if (wide && e0 >= 0 && e0 + VE <= a.vocab) {
            vector_of(p_row + e0, p);
            if (DRAFT && c > 0.0) vector_of(q_row + e0, q);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const bool in = e0 + i >= 0 && e0 + i < a.vocab;
                p[i] = in ? value(p_row + e0 + i) : 0.0f;
                if (DRAFT && c > 0.0) q[i] = in ? value(q_row + e0 + i) : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            r[i] = DRAFT && c > 0.0 ? rest_of(p[i], q[i], c) : (double)fmaxf(p[i], 0.0f);
        }
        if (!DRAFT) {
            for (int k = 0; k < rejected; ++k) {
                const int at = s_gone[k] - e0;
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    if (at == i) r[i] = 0.0;
                }
            }
        }
    };
    // The sum of the residual over the vocabulary, the same value in every thread of the cluster.
    // False: the CTAs do not agree where the walk stands.
    auto pass = [&](double c, int rejected) -> bool {
        uint64_t lead = 0;
        double sum = 0.0;
        for (int vec = vec_lo + lane; vec < vec_hi; vec += 32) {
            double r[VE];
            residual(vec, c, rejected, r);
#pragma unroll
            for (int i = 0; i < VE; ++i) sum += r[i];
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) s_warp[warp] = sum;
        __syncthreads();
        own = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) own += s_warp[i];
        // Every CTA reads the sums in the same order: the running sums are the same in all of them.
        const uint64_t step = (uint64_t)n | (uint64_t)w.node << 8 | (uint64_t)rejected << 16 |
                              (uint64_t)w.last << 24 | (uint64_t)(uint32_t)turn << 32;
        if (tid == 0) s_said[turn & 1] = Said{own, step};
        cluster_sync_all();
        total = before = 0.0;
        later = false;
        bool agreed = true;
        for (int k = 0; k < a.cluster; ++k) {
            const Said said = ld_cluster_said(cluster_map(smem_u32(&s_said[turn & 1]), (uint32_t)k));
            if (k == 0) lead = said.step;
            agreed = agreed && said.step == lead;
            if (k < rank) before += said.sum;
            later = later || (k > rank && said.sum > 0.0);
            total += said.sum;
        }
        ++turn;
        return agreed;
    };

    // ---- the walk ---------------------------------------------------------------------------------
    for (;;) {
        if (tid == 0 && n == 0) w.last = 1;  // nothing to walk: one pass over nothing
        if (tid == 0 && n > 0) {
            for (;;) {
                int child = -1;
                for (int k = w.tried >> 5; k < kWords && child < 0; ++k) {
                    uint32_t bits = s_child[w.node][k];
                    if (k == (w.tried >> 5)) bits &= ~((2u << (w.tried & 31)) - 1u);
                    if (bits != 0) child = k * 32 + __ffs(bits) - 1;
                }
                if (child < 0) {
                    w.last = 1;
                    w.pass = 1;
                    break;
                }
                w.tried = child;
                double room = rest_of(s_p[child], DRAFT && w.c > 0.0 ? s_q[child] : 0.0f, w.c);
                if (!DRAFT) {
                    for (int k = 0; k < w.rejected; ++k) {
                        if (s_gone[k] == s_word[child]) room = 0.0;
                    }
                }
                if ((double)s_u[child] * (double)s_q[child] * w.sum < room) {
                    w.node = child;
                    w.c = 0.0;
                    w.sum = 1.0;
                    w.rejected = 0;
                    s_path[w.count++] = child;
                } else {
                    w.c += w.sum;
                    s_gone[w.rejected++] = s_word[child];
                    // Is another child left? If not, the pass for this rejection is the sample's too.
                    bool more = false;
                    for (int k = w.tried >> 5; k < kWords; ++k) {
                        uint32_t bits = s_child[w.node][k];
                        if (k == (w.tried >> 5)) bits &= ~((2u << (w.tried & 31)) - 1u);
                        more = more || bits != 0;
                    }
                    w.last = more ? 0 : 1;
                    w.pass = 1;
                    break;
                }
            }
        }
        __syncthreads();
        const double c = w.c;
        const int rejected = w.rejected;
        const bool last = w.last != 0;
        if (n > 0) set_rows(w.node);
        bool agreed = pass(c, rejected);
        __syncthreads();
        if (agreed && !last) {
            if (tid == 0) w.sum = total;
            continue;
        }
        double cc = c;
        int gone = rejected;
        if (agreed && !(total > 0.0) && rejected > 0) {  // nothing is left of p: p itself
            cc = 0.0;
            gone = 0;
            agreed = pass(cc, gone);
            __syncthreads();
        }
        if (!agreed || n == 0) {
            if (rank == 0) {
                if (!agreed && tid == 0) raise_bad_input(a.status);
                if (tid < a.tokens) a.path[(int64_t)b * a.tokens + tid] = -1;
                if (tid == 0) {
                    a.kept[b] = 0;
                    a.next_token[b] = -1;
                }
            }
            break;
        }
        // ---- the sample -----------------------------------------------------------------------
        // The first CTA whose running sum passes the threshold (or the last one with anything in it)
        // holds the sample; in it, likewise, the warp, the round of 32 vectors, the lane.
        const double threshold = (double)__ldg(a.u_sample + b) * total;
        // The running sums are the same numbers in every CTA, so exactly one of them passes it.
        const bool mine = total > threshold ? !(before > threshold) && before + own > threshold
                                            : own > 0.0 && !later;
        if (mine && warp == 0) {
            double run = before;
            int seg = -1, fallback = 0;
            double seg_run = run;
            for (int i = 0; i < kWarps; ++i) {
                if (s_warp[i] > 0.0) {
                    fallback = i;
                    seg_run = run;
                    if (run + s_warp[i] > threshold) {
                        seg = i;
                        break;
                    }
                }
                run += s_warp[i];
            }
            if (seg < 0) seg = fallback;
            run = seg_run;
            const int64_t vecs = (a.vocab + shift + VE - 1) / VE;
            const int64_t lo = vecs * rank / a.cluster, hi = vecs * (rank + 1) / a.cluster;
            const int first = (int)(lo + (hi - lo) * seg / kWarps);
            const int end = (int)(lo + (hi - lo) * (seg + 1) / kWarps);
            int found = -1, latest = -1;  // latest: last element with anything in it
            for (int v0 = first; v0 < end && found < 0; v0 += 32) {
                double r[VE];
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < VE; ++i) r[i] = 0.0;
                if (v0 + lane < end) residual(v0 + lane, cc, gone, r);
                int here = -1;
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    sum += r[i];
                    if (r[i] > 0.0) here = (v0 + lane) * VE - shift + i;
                }
                double incl = sum;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += up;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, run + incl > threshold && sum > 0.0);
                const uint32_t some = __ballot_sync(0xffffffffu, here >= 0);
                if (over != 0) {
                    const int who = __ffs(over) - 1;
                    double at = run + (incl - sum);
                    int pick = here;
#pragma unroll
                    for (int i = VE - 1; i >= 0; --i) {
                        double upto = at;
#pragma unroll
                        for (int j = 0; j <= i; ++j) upto += r[j];
                        if (r[i] > 0.0 && upto > threshold) pick = (v0 + lane) * VE - shift + i;
                    }
                    found = __shfl_sync(0xffffffffu, pick, who);
                } else if (some != 0) {
                    latest = __shfl_sync(0xffffffffu, here, 31 - __clz(some));
                }
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) a.next_token[b] = found >= 0 ? found : latest;
        }
        if (rank == 0) {
            if (tid < a.tokens) {
                a.path[(int64_t)b * a.tokens + tid] = tid == 0 ? 0 : (tid < w.count ? s_path[tid] : -1);
            }
            if (tid == 0) {
                a.kept[b] = w.count;
                if (!(total > 0.0)) {
                    a.next_token[b] = -1;
                    raise_bad_input(a.status);
                }
            }
        }
        break;
    }
    // No CTA may leave while another still reads its sums.
    cluster_sync_all();
}

template <typename T, bool DRAFT>
cudaError_t launch(const VerifyArgs& a, cudaStream_t stream) {
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)a.cluster;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.batch * a.cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, tree_verify_kernel<T, DRAFT>, a);
}

}  // namespace
}  // namespace gqa

extern "C" int gqa_tree_verify(const gqa_tree_verify_params* p) {
    using namespace gqa;
    if (p == nullptr) return GQA_ERR_NULL;
    if (p->dtype != GQA_DTYPE_F32 && p->dtype != GQA_DTYPE_BF16) return GQA_ERR_DTYPE;
    if (p->batch <= 0 || p->tokens <= 0 || p->tokens > kTreeMaxTokens || p->vocab <= 0) return GQA_ERR_SHAPE;
    if (p->batch > (1 << 24)) return GQA_ERR_SHAPE;
    if (p->vocab > (1 << 30)) return GQA_ERR_SHAPE;
    if (p->target == nullptr || p->tokens_dev == nullptr || p->parents_dev == nullptr ||
        p->u_accept == nullptr || p->u_sample == nullptr || p->path == nullptr || p->kept == nullptr ||
        p->next_token == nullptr) {
        return GQA_ERR_NULL;
    }
    const uintptr_t eb = p->dtype == GQA_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(p->target) % eb || reinterpret_cast<uintptr_t>(p->draft) % eb) {
        return GQA_ERR_ALIGN;
    }
    VerifyArgs a;
    std::memset(&a, 0, sizeof(a));
    a.target = p->target;
    a.draft = p->draft;
    a.words = p->tokens_dev;
    a.parents = p->parents_dev;
    a.u_accept = p->u_accept;
    a.u_sample = p->u_sample;
    a.tree_sizes = p->tree_sizes_dev;
    a.path = p->path;
    a.kept = p->kept;
    a.next_token = p->next_token;
    a.status = p->status_dev;
    a.batch = p->batch;
    a.tokens = p->tokens;
    a.vocab = p->vocab;
    a.target_node = p->target_node_stride != 0 ? p->target_node_stride : p->vocab;
    a.draft_node = p->draft_node_stride != 0 ? p->draft_node_stride : p->vocab;
    a.target_seq = p->target_seq_stride != 0 ? p->target_seq_stride : a.target_node * p->tokens;
    a.draft_seq = p->draft_seq_stride != 0 ? p->draft_seq_stride : a.draft_node * p->tokens;
    if (a.target_node < 0 || a.draft_node < 0 || a.target_seq < 0 || a.draft_seq < 0) return GQA_ERR_SHAPE;
    a.cluster = kMaxCluster;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(p->stream);
    cudaError_t e;
    if (p->dtype == GQA_DTYPE_F32) {
        e = p->draft != nullptr ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
    } else {
        e = p->draft != nullptr ? launch<__nv_bfloat16, true>(a, stream)
                                : launch<__nv_bfloat16, false>(a, stream);
    }
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

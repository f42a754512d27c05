// Verification of a drafted tree against the target's probabilities (gqa_tree_verify).
//
// Mathematics. Rejecting child after child of one node takes the residual of a residual:
// r_0 = p, r_{k+1} = max(r_k - q, 0) / s_{k+1}. Multiplied out, r_k S_k = max(p - c_k q, 0) with S_0 = 1,
// c_0 = 0, c_{k+1} = c_k + S_k and S_k the sum of max(p - c_k q, 0) over the vocabulary: one scalar replaces the
// chain, and a rejection costs one pass over the rows p and q of that node. Accepted nodes cost no row
// at all, only p and q at the child's token, which are fetched for every node of the tree before
// the walk starts. Tests and sums are FP64: p, q and u are FP32 or BF16 values, so u q is exact. S, c and the running
// sums round in FP64 in an order that follows the cluster's size (so the batch, the vocabulary and the SM count): a test or a
// threshold within about 2^-50 of equality may fall either way with another size.
//
// Without draft probabilities the residual is p without the rejected tokens. One pass per node then
// serves all its children: R = the sum of p without any child's token; after j rejections the
// sum is R plus p at the tokens still to be tried (only positive terms: nothing cancels).
//
// One thread-block cluster per sequence; the CTAs take equal slices of the vocabulary, the warps of
// a CTA contiguous segments of its slice. Every CTA walks the tree itself (same inputs, same sums,
// same steps); after a pass the CTAs read one another's partial sums through distributed shared
// memory. To place the sample, the partial sums name the segment in which the cumulative sum
// passes u S, the kept sums of its rounds the round of 32 vectors, and one warp looks through that. A pass is bound by the latency of its loads: a lane
// has eight vectors of each row in flight (two: 4.4 us a pass over 16000 elements per CTA). Measured: 16 sequences of 32
// nodes over 128000 words 21 us (up to four passes that depend on one another, about 3 us each, with 2 us of exchange and
// walk), 64 sequences over 151643 words without draft probabilities 20 us, one of 8 nodes over 32000 words 7 us.
#include <cuda_bf16.h>

#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxRounds = 64;  // rounds of 32 vectors of a warp's segment whose sums are kept
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
    int32_t cluster;  // a power of two
    int32_t cluster_log2;
};

__device__ __forceinline__ float value(const float* p) { return __ldg(p); }
__device__ __forceinline__ float value(const __nv_bfloat16* p) {
    return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
}
// 16 bytes of a row as its elements.
__device__ __forceinline__ void elements(uint4 u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void elements(uint4 u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo_to_f32(w[i]);
        x[2 * i + 1] = bf16_hi_to_f32(w[i]);
    }
}

// max(p - c q, 0); NaN and negative entries count as 0. The two conversions (8 cycles per warp each, as
// measured, where the bit operations that could replace one take 14) bound a pass.
__device__ __forceinline__ double rest_of(float p, float q, double c) {
    const double r = fma(-c, (double)fmaxf(q, 0.0f), (double)p);
    return r > 0.0 ? r : 0.0;
}
__device__ __forceinline__ double rest_of(float p) { return (double)fmaxf(p, 0.0f); }

// The sums over the warp of eight values per lane: lane 4 k of a warp gets that of value k. Halves of the values
// change places with each step: 9 exchanges instead of 40.
__device__ __forceinline__ double reduce8(const double (&v)[8], int lane) {
    double a[4], b[2], c;
    const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = (h16 ? v[i + 4] : v[i]) + __shfl_xor_sync(0xffffffffu, h16 ? v[i] : v[i + 4], 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        b[i] = (h8 ? a[i + 2] : a[i]) + __shfl_xor_sync(0xffffffffu, h8 ? a[i] : a[i + 2], 8);
    }
    c = (h4 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, h4 ? b[0] : b[1], 4);
    c += __shfl_xor_sync(0xffffffffu, c, 2);
    return c + __shfl_xor_sync(0xffffffffu, c, 1);
}

// In pairs: an FP64 sum is a chain of long latencies otherwise.
template <int N>
__device__ __forceinline__ double sum_of(const double (&r)[N]) {
    double s[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) s[i] = r[2 * i] + r[2 * i + 1];
#pragma unroll
    for (int n = N / 2; n > 1; n /= 2) {
#pragma unroll
        for (int i = 0; i < n / 2; ++i) s[i] = s[2 * i] + s[2 * i + 1];
    }
    return s[0];
}

// Where the walk stands.
enum Action : int {
    kSum,     // a pass over the current node's rows, then on with the walk
    kSample,  // a pass, then the sample
    kPlace,   // the sample from the sums of the last pass
};
struct Walk {
    int node;      // current node
    int tried;     // its last tried child (or the node itself)
    int count;     // nodes on the path
    int rejected;  // children of `node` rejected so far
    int action;
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
__global__ void __launch_bounds__(kThreads, 1) tree_verify_kernel(const VerifyArgs a) {
    constexpr int VE = 16 / (int)sizeof(T);
    constexpr int kUnroll = 8;  // vectors of a row a lane has in flight
    __shared__ uint32_t s_child[kTreeMaxTokens][kWords];
    __shared__ float s_p[kTreeMaxTokens], s_q[kTreeMaxTokens], s_u[kTreeMaxTokens];
    __shared__ int32_t s_word[kTreeMaxTokens];
    __shared__ int32_t s_path[kTreeMaxTokens];
    __shared__ uint8_t s_first[kTreeMaxTokens];        // passes the test that holds before a rejection
    __shared__ uint8_t s_again[kTreeMaxTokens];        // an earlier sibling has the same token
    __shared__ double s_ahead[kTreeMaxTokens];         // p at the tokens of later siblings
    __shared__ int32_t s_gone[kTreeMaxTokens];         // tokens left out of the sum (no draft)
    __shared__ uint8_t s_hit[kWarps][kTreeMaxTokens];  // those inside a warp's segment
    __shared__ int s_gone_count;
    __shared__ double s_warp[kWarps];
    __shared__ double s_round[kWarps][kMaxRounds];  // sums of the rounds of the last pass
    __shared__ Said s_said[2];  // this CTA's sum and step, buffers in turn: read by the whole cluster
    __shared__ Walk w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % a.cluster;
    const int b = blockIdx.x / a.cluster;
    pdl_launch_dependents();
    for (int i = tid; i < kTreeMaxTokens * kWords; i += kThreads) (&s_child[0][0])[i] = 0;
    if (tid == 0) {
        w = Walk{0, 0, 1, 0, kSum, 0.0, 1.0};
        s_gone_count = 0;
    }
    pdl_wait();
    const T* target = static_cast<const T*>(a.target) + b * a.target_seq;
    const T* draft = DRAFT ? static_cast<const T*>(a.draft) + b * a.draft_seq : nullptr;

    // ---- children and the values at the drafted tokens ----------------------------------------
    int par = -1, word = -1;
    float u = 0.0f;
    if (tid > 0 && tid < a.tokens) {
        par = __ldg(a.parents + (int64_t)b * a.tokens + tid);
        word = __ldg(a.words + (int64_t)b * a.tokens + tid);
        u = __ldg(a.u_accept + (int64_t)b * a.tokens + tid);
    }
    const float u_sample = __ldg(a.u_sample + b);
    int n = a.tree_sizes != nullptr ? __ldg(a.tree_sizes + b) : a.tokens;
    bool bad = n < 0 || n > a.tokens;
    if (bad) n = 0;
    const bool node = tid > 0 && tid < n;
    const bool fine = node && par >= 0 && par < tid && word >= 0 && word < a.vocab;
    bad = bad || (node && !fine);
    __syncthreads();
    if (fine) {
        const float p = value(target + par * a.target_node + word);
        const float q = DRAFT ? value(draft + par * a.draft_node + word) : 1.0f;
        atomicOr(&s_child[par][tid >> 5], 1u << (tid & 31));
        s_word[tid] = word;
        s_u[tid] = u;
        s_p[tid] = p;
        s_q[tid] = q;
        s_first[tid] = (double)u * (double)fmaxf(q, 0.0f) < rest_of(p);
    }
    bad = __syncthreads_or(bad);
    if (bad && rank == 0 && tid == 0) raise_bad_input(a.status);
    if (!DRAFT) {
        if (fine) {
            bool again = false;
            for (int k = 0; k < kWords; ++k) {
                uint32_t bits = s_child[par][k];
                if (k == (tid >> 5)) bits &= (1u << (tid & 31)) - 1u;
                if (k > (tid >> 5)) bits = 0;
                for (; bits != 0; bits &= bits - 1) again = again || s_word[k * 32 + __ffs(bits) - 1] == word;
            }
            s_again[tid] = again;
        }
        __syncthreads();
    }

    const T* p_row = target;
    const T* q_row = draft;
    int turn = 0;
    double total = 0.0;      // sum of the residual after the last pass
    double before = 0.0;     // of the CTAs before this one
    double own = 0.0;
    double parts = 0.0, upto = 0.0;  // lane k: CTA k's sum, and the sum up to it
    double run_to = 0.0;     // lane i: sum of this CTA's segments 0 .. i
    // The row in vectors of 16 bytes. A vector is cut at the row's ends, where single elements are
    // read; rows p and q that are not equally aligned are read element by element.
    int vecs = 0, shift = 0;
    bool wide = false;

    auto set_rows = [&](int at) {
        p_row = target + at * a.target_node;
        if (DRAFT) q_row = draft + at * a.draft_node;
        shift = (int)((reinterpret_cast<uintptr_t>(p_row) & 15u) / sizeof(T));
        wide = !DRAFT || ((reinterpret_cast<uintptr_t>(p_row) ^ reinterpret_cast<uintptr_t>(q_row)) & 15u) == 0;
        vecs = (a.vocab + shift + VE - 1) / VE;
    };
    // First vector of segment `seg` of this CTA's slice (slices and segments of equal length but the last:
    // shifts, where an exact cut would take four 64-bit divisions, 0.9 us ahead of the first load).
    auto segment = [&](int seg) -> int {
        const int slice = (vecs + a.cluster - 1) >> a.cluster_log2;
        const int part = (slice + kWarps - 1) / kWarps;
        const int lo = min(vecs, rank * slice), hi = min(vecs, lo + slice);
        return min(hi, lo + seg * part);
    };
    // The tokens left out that lie in vectors [first, end), into this warp's list.
    auto collect = [&](int first, int end, int gone) -> int {
        int hits = 0;
        for (int k0 = 0; k0 < gone; k0 += 32) {
            const int k = k0 + lane;
            const int vec = k < gone ? (s_gone[k] + shift) / VE : -1;
            const bool in = vec >= first && vec < end;
            const uint32_t some = __ballot_sync(0xffffffffu, in);
            if (in) s_hit[warp][hits + __popc(some & ((1u << lane) - 1u))] = (uint8_t)k;
            hits += __popc(some);
        }
        __syncwarp();
        return hits;
    };
    auto whole = [&](int vec) { return vec * VE >= shift && vec * VE - shift + VE <= a.vocab; };
    // The residual of a vector from its elements; `hits` tokens are left out.
    auto rest = [&](int vec, const float (&p)[VE], const float (&q)[VE], double c, int hits, double (&r)[VE]) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            r[i] = DRAFT && c > 0.0 ? rest_of(p[i], q[i], c) : rest_of(p[i]);
        }
        if (!DRAFT) {
            for (int k = 0; k < hits; ++k) {
                const int at = s_gone[s_hit[warp][k]] + shift - vec * VE;
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    if (at == i) r[i] = 0.0;
                }
            }
        }
    };
    // The residual at any vector; elements outside the row are 0.
    auto residual = [&](int vec, double c, int hits, double (&r)[VE]) {
        const int e0 = vec * VE - shift;
        float p[VE], q[VE];
        if (wide && whole(vec)) {
            elements(__ldg(reinterpret_cast<const uint4*>(p_row + e0)), p);
            if (DRAFT && c > 0.0) elements(__ldg(reinterpret_cast<const uint4*>(q_row + e0)), q);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const bool in = e0 + i >= 0 && e0 + i < a.vocab;
                p[i] = in ? value(p_row + e0 + i) : 0.0f;
                if (DRAFT && c > 0.0) q[i] = in ? value(q_row + e0 + i) : 0.0f;
            }
        }
        rest(vec, p, q, c, hits, r);
    };
    // The sums of the cluster's CTAs, the same values in every thread. False: the CTAs do not agree
    // where the walk stands.
    auto exchange = [&]() -> bool {
        const uint64_t step = (uint64_t)n | (uint64_t)w.node << 8 | (uint64_t)w.rejected << 16 |
                              (uint64_t)w.action << 24 | (uint64_t)(uint32_t)turn << 32;
        if (tid == 0) s_said[turn & 1] = Said{own, step};
        cluster_sync_all();
        // Lane k reads CTA k; running sums by a scan, the same operations on the same numbers in every CTA.
        const bool one = lane < a.cluster;
        Said said = {0.0, 0};
        if (one) said = ld_cluster_said(cluster_map(smem_u32(&s_said[turn & 1]), (uint32_t)lane));
        parts = said.sum;
        upto = said.sum;
#pragma unroll
        for (int d = 1; d < kMaxCluster; d <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += up;
        }
        total = __shfl_sync(0xffffffffu, upto, a.cluster - 1);
        before = rank > 0 ? __shfl_sync(0xffffffffu, upto, rank - 1) : 0.0;
        const bool agreed = __all_sync(0xffffffffu, !one || said.step == step);
        ++turn;
        return agreed;
    };
    auto pass = [&](double c, int gone) -> bool {
        const int lo = segment(warp), hi = segment(warp + 1);
        const int hits = DRAFT ? 0 : collect(lo, hi, gone);
        double sum = 0.0;
        for (int v0 = lo; v0 < hi; v0 += 32 * kUnroll) {
            uint4 up[kUnroll], uq[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const int vec = v0 + 32 * k + lane;
                if (vec < hi && wide && whole(vec)) {
                    up[k] = __ldg(reinterpret_cast<const uint4*>(p_row + (vec * VE - shift)));
                    if (DRAFT && c > 0.0) uq[k] = __ldg(reinterpret_cast<const uint4*>(q_row + (vec * VE - shift)));
                }
            }
            double round[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                round[k] = 0.0;
                const int vec = v0 + 32 * k + lane;
                if (vec >= hi) continue;
                double r[VE];
                if (wide && whole(vec)) {
                    float p[VE], q[VE];
                    elements(up[k], p);
                    if (DRAFT && c > 0.0) elements(uq[k], q);
                    rest(vec, p, q, c, hits, r);
                } else {
                    residual(vec, c, hits, r);
                }
                round[k] = sum_of(r);
            }
            __syncwarp();
            const double of = reduce8(round, lane);  // lane 4 k: round k
            const int at = (v0 - lo) / 32 + (lane >> 2);
            if ((lane & 3) == 0 && at < kMaxRounds) s_round[warp][at] = of;
            sum += sum_of(round);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) s_warp[warp] = sum;
        __syncthreads();
        // The running sums of the segments, in lanes 0 .. kWarps - 1 of every warp.
        run_to = lane < kWarps ? s_warp[lane] : 0.0;
#pragma unroll
        for (int d = 1; d < kWarps; d <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run_to, d);
            if (lane >= d) run_to += up;
        }
        own = __shfl_sync(0xffffffffu, run_to, kWarps - 1);
        const bool agreed = exchange();
        __syncthreads();
        return agreed;
    };
    // One warp: the element of vectors [first, end) at which the running sum (`run` before them) passes the
    // threshold, else the last one with anything in it, else -1.
    auto place = [&](int first, int end, double run, double threshold, double c, int hits) -> int {
        int found = -1, latest = -1;  // latest: last element with anything in it
        for (int v0 = first; v0 < end && found < 0; v0 += 32) {
            double r[VE];
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < VE; ++i) r[i] = 0.0;
            if (v0 + lane < end) residual(v0 + lane, c, hits, r);
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
                double at = run + (incl - sum);
                int pick = -1;
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    at += r[i];
                    if (pick < 0 && r[i] > 0.0 && at > threshold) pick = (v0 + lane) * VE - shift + i;
                }
                found = __shfl_sync(0xffffffffu, pick >= 0 ? pick : here, __ffs(over) - 1);
            } else if (some != 0) {
                latest = __shfl_sync(0xffffffffu, here, 31 - __clz(some));
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        return found >= 0 ? found : latest;
    };
    // The child of w.node after w.tried, -1: none.
    auto next_child = [&]() -> int {
        for (int k = w.tried >> 5; k < kWords; ++k) {
            uint32_t bits = s_child[w.node][k];
            if (k == (w.tried >> 5)) bits &= ~((2u << (w.tried & 31)) - 1u);
            if (bits != 0) return k * 32 + __ffs(bits) - 1;
        }
        return -1;
    };

    // ---- the walk ---------------------------------------------------------------------------------
    bool agreed = true;
    int gone = 0;
    for (;;) {
        if (tid == 0 && n == 0) w.action = kPlace;  // nothing to walk
        if (tid == 0 && n > 0) {
            for (;;) {
                const int child = next_child();
                if (child < 0) {
                    w.action = !DRAFT && w.rejected > 0 ? kPlace : kSample;
                    break;
                }
                w.tried = child;
                bool taken;
                if (w.rejected == 0) {
                    taken = s_first[child];
                } else {
                    const double room = DRAFT ? rest_of(s_p[child], s_q[child], w.c)
                                              : s_again[child] ? 0.0 : rest_of(s_p[child]);
                    taken = (double)s_u[child] * (double)fmaxf(s_q[child], 0.0f) * w.sum < room;
                }
                if (taken) {
                    w.node = child;
                    w.c = 0.0;
                    w.sum = 1.0;
                    w.rejected = 0;
                    s_gone_count = 0;
                    s_path[w.count++] = child;
                    continue;
                }
                ++w.rejected;
                if (DRAFT) {
                    w.c += w.sum;
                    w.action = next_child() < 0 ? kSample : kSum;
                    break;
                }
                if (w.rejected > 1) {
                    w.sum = total + s_ahead[child];
                    continue;
                }
                // The first rejection here: all children's tokens leave the sum.
                int count = 0;
                double ahead = 0.0;
                for (int k = kWords - 1; k >= 0; --k) {
                    for (uint32_t bits = s_child[w.node][k]; bits != 0;) {
                        const int at = k * 32 + 31 - __clz(bits);
                        bits &= ~(1u << (at & 31));
                        s_ahead[at] = ahead;
                        if (!s_again[at]) {
                            s_gone[count++] = s_word[at];
                            ahead += rest_of(s_p[at]);
                        }
                    }
                }
                s_gone_count = count;
                w.action = kSum;
                break;
            }
        }
        __syncthreads();
        const int action = w.action;
        const double c = w.c;
        if (action == kPlace) {
            agreed = exchange();
            __syncthreads();
        } else {
            gone = s_gone_count;
            set_rows(w.node);
            agreed = pass(c, gone);
        }
        if (!agreed || n == 0) break;
        if (action == kSum) {
            if (tid == 0) w.sum = DRAFT ? total : total + s_ahead[w.tried];
            continue;
        }
        double cc = c;
        if (!(total > 0.0) && w.rejected > 0) {  // nothing is left of p: p itself
            cc = 0.0;
            gone = 0;
            agreed = pass(cc, gone);
            if (!agreed) break;
        }
        // ---- the sample -----------------------------------------------------------------------
        // The first CTA whose running sum passes the threshold (or the last one with anything in it)
        // holds the sample; in it, likewise, the warp, the round of 32 vectors, the lane.
        const double threshold = (double)u_sample * total;
        const uint32_t passed = __ballot_sync(0xffffffffu, lane < a.cluster && parts > 0.0 && upto > threshold);
        const uint32_t filled = __ballot_sync(0xffffffffu, lane < a.cluster && parts > 0.0);
        const bool mine = filled != 0 && (passed != 0 ? __ffs(passed) - 1 : 31 - __clz(filled)) == rank;
        if (mine && warp == 0) {
            const double segs = lane < kWarps ? s_warp[lane] : 0.0;
            const uint32_t over_at = __ballot_sync(0xffffffffu, segs > 0.0 && before + run_to > threshold);
            const uint32_t some_at = __ballot_sync(0xffffffffu, segs > 0.0);
            const int seg = over_at != 0 ? __ffs(over_at) - 1 : 31 - __clz(some_at);
            double run = before + (seg > 0 ? __shfl_sync(0xffffffffu, run_to, seg - 1) : 0.0);
            const int first = segment(seg), end = segment(seg + 1);
            const int hits = DRAFT ? 0 : collect(first, end, gone);
            int token = -1;
            // First which round of the pass, then which element. Rounds beyond those kept are looked over.
            const int rounds = (end - first + 31) / 32;
            if (rounds > 1) {
                double at = run;
                int pick = -1, last = -1;
                double pick_run = run, last_run = run;
                for (int r0 = 0; r0 < min(rounds, kMaxRounds) && pick < 0; r0 += 32) {
                    const int i = r0 + lane;
                    const double sum = i < min(rounds, kMaxRounds) ? s_round[seg][i] : 0.0;
                    double incl = sum;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, incl, d);
                        if (lane >= d) incl += up;
                    }
                    const double ahead = at + (incl - sum);
                    const uint32_t over = __ballot_sync(0xffffffffu, sum > 0.0 && at + incl > threshold);
                    const uint32_t some = __ballot_sync(0xffffffffu, sum > 0.0);
                    if (over != 0) {
                        pick = r0 + __ffs(over) - 1;
                        pick_run = __shfl_sync(0xffffffffu, ahead, __ffs(over) - 1);
                    } else if (some != 0) {
                        last = r0 + 31 - __clz(some);
                        last_run = __shfl_sync(0xffffffffu, ahead, 31 - __clz(some));
                    }
                    at += __shfl_sync(0xffffffffu, incl, 31);
                }
                if (pick < 0 && rounds > kMaxRounds) {
                    token = place(first + 32 * kMaxRounds, end, at, threshold, cc, hits);
                }
                if (token < 0) {
                    const int at_round = first + 32 * (pick >= 0 ? pick : max(last, 0));
                    token = place(at_round, min(end, at_round + 32), pick >= 0 ? pick_run : last_run, threshold, cc, hits);
                }
            } else {
                token = place(first, end, run, threshold, cc, hits);
            }
            if (lane == 0) a.next_token[b] = token;
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
    if ((!agreed || n == 0) && rank == 0) {
        if (!agreed && tid == 0) raise_bad_input(a.status);
        if (tid < a.tokens) a.path[(int64_t)b * a.tokens + tid] = -1;
        if (tid == 0) {
            a.kept[b] = 0;
            a.next_token[b] = -1;
        }
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
    // As many CTAs per sequence as leave a lane more than one vector of a row and run all at once (one per
    // SM), at most 8 (portable clusters).
    int32_t sms = 0;
    if (current_sm_count(&sms) != GQA_OK) return GQA_ERR_CUDA;
    const int64_t vectors = (int64_t)p->vocab * (int64_t)eb / 16;
    a.cluster = 1;
    a.cluster_log2 = 0;
    while (a.cluster < kMaxCluster && vectors > (int64_t)2 * a.cluster * kThreads &&
           (int64_t)2 * a.cluster * a.batch <= sms) {
        a.cluster *= 2;
        ++a.cluster_log2;
    }
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

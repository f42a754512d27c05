// Keeps the accepted path of a draft tree (gqa_tree_commit): in every layer the K and V rows of its
// nodes move, in place, to the first of the draft's cache slots; the lengths follow.
//
// The path ascends, path[i] >= i, so row i never lands on the source of a later row: a thread that
// owns one 16-byte column of the rows walks the path upwards and needs no second buffer. It reads kBatch rows
// before it writes them (destinations i .. i + kBatch - 1, later sources >= i + kBatch), so that
// their loads are in flight together. Bound by bytes: every moved row is read and written once (32 sequences
// of 64 nodes in 36 layers of 8 heads: 17 us, 4.4 TB/s of scattered 256-byte rows; one sequence of 8 nodes: 2.5 us).
#include <cstring>

#include "ptx.cuh"
#include "tree_common.cuh"

namespace gqa {
namespace {

constexpr int kThreads = 128;
constexpr int kBatch = 8;

struct CommitArgs {
    TreeCache cache;
    void* k_cache;
    void* v_cache;
    const int32_t* path;
    const int32_t* kept;
    int32_t* lens_out;
    int64_t layer_bytes;
    int32_t elem_bytes;
    int32_t cols;          // 16-byte columns of a row of all heads
    int32_t cols_per_head;
    int32_t keep_history;  // what a skipped sequence leaves in lens_out: its history, else its length
};

// grid.x: blocks of kThreads columns, K and V side by side; grid.y: layers; grid.z: sequences.
__global__ void __launch_bounds__(kThreads) tree_commit_kernel(const CommitArgs a) {
    __shared__ int32_t s_path[kTreeMaxTokens];
    __shared__ int64_t s_src[kTreeMaxTokens];  // byte offset of the source row, -1: stays
    __shared__ int64_t s_dst[kTreeMaxTokens];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.z;
    const TreeSpan span = tree_span(a.cache, b);
    const int kept = __ldg(a.kept + b);
    bool ok = span.ok && kept >= 0 && kept <= span.n;
    const int tid = threadIdx.x;
    if (ok && tid < kept) s_path[tid] = __ldg(a.path + (int64_t)b * a.cache.tokens + tid);
    __syncthreads();
    if (ok && tid < kept) {
        const int32_t from = s_path[tid];
        ok = from < span.n && from > (tid > 0 ? s_path[tid - 1] : -1);
        int64_t src = 0, dst = 0;
        // Rows that stay are looked up too: without a block nothing can have been written there.
        if (ok) ok = tree_row(a.cache, b, span.base + from, &src) && tree_row(a.cache, b, span.base + tid, &dst);
        s_src[tid] = from != tid ? src * a.elem_bytes : -1;
        s_dst[tid] = dst * a.elem_bytes;
    }
    ok = __syncthreads_and(ok);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
        int32_t len = span.base + kept;
        if (!ok) {
            raise_bad_input(a.cache.status);
            len = __ldg(a.cache.seq_lens + b);
            const int32_t n = a.cache.tree_sizes != nullptr ? __ldg(a.cache.tree_sizes + b) : a.cache.tokens;
            if (a.keep_history && n >= 0 && n <= a.cache.tokens && len >= n) len -= n;
        }
        a.lens_out[b] = len;
    }
    if (!ok) return;
    const int col = blockIdx.x * kThreads + tid;
    if (col >= 2 * a.cols) return;
    const bool is_v = col >= a.cols;
    const int c = is_v ? col - a.cols : col;
    const int head = c / a.cols_per_head;
    char* base = static_cast<char*>(is_v ? a.v_cache : a.k_cache) + blockIdx.y * a.layer_bytes +
                 (int64_t)head * a.cache.stride_head * a.elem_bytes + (c - head * a.cols_per_head) * 16;
#pragma unroll 1
    for (int i0 = 0; i0 < kept; i0 += kBatch) {
        uint4 row[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + i < kept && s_src[i0 + i] >= 0) {
                row[i] = *reinterpret_cast<const uint4*>(base + s_src[i0 + i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + i < kept && s_src[i0 + i] >= 0) {
                *reinterpret_cast<uint4*>(base + s_dst[i0 + i]) = row[i];
            }
        }
    }
}

int commit(const gqa_tree_commit_params* p, bool keep_history) {
    if (p == nullptr) return GQA_ERR_NULL;
    CommitArgs a;
    std::memset(&a, 0, sizeof(a));
    const TreeCacheDesc d = {p->dtype, p->batch, p->tokens, p->num_kv_heads, p->head_dim,
                             p->blocks_per_seq, p->fixed_block, &p->layout, p->k_cache, p->v_cache,
                             p->seq_lens_dev, p->tree_sizes_dev, p->block_table_dev, p->status_dev};
    const int rc = tree_cache_args(d, &a.cache);
    if (rc != GQA_OK) return rc;
    if (p->path == nullptr || p->kept == nullptr || p->seq_lens_out == nullptr) return GQA_ERR_NULL;
    if (p->num_layers <= 0 || p->num_layers > 65535 || p->batch > 65535) return GQA_ERR_SHAPE;
    if (p->num_layers > 1 && p->layer_stride <= 0) return GQA_ERR_SHAPE;
    // One block of a sequence writes its length while the others still read these.
    const int64_t lens_bytes = (int64_t)p->batch * sizeof(int32_t);
    for (const int32_t* in : {p->seq_lens_dev, p->kept, p->tree_sizes_dev}) {
        if (in != nullptr && rows_overlap(p->seq_lens_out, 0, in, 0, 1, lens_bytes)) return GQA_ERR_UNSUPPORTED;
    }
    const uintptr_t out = reinterpret_cast<uintptr_t>(p->seq_lens_out), path = reinterpret_cast<uintptr_t>(p->path);
    if (out + lens_bytes > path && out < path + lens_bytes * p->tokens) return GQA_ERR_UNSUPPORTED;
    a.elem_bytes = p->dtype == GQA_DTYPE_F32 ? 4 : 2;
    a.layer_bytes = p->num_layers > 1 ? p->layer_stride * a.elem_bytes : 0;
    if (a.layer_bytes % 16 != 0) return GQA_ERR_ALIGN;
    a.k_cache = p->k_cache;
    a.v_cache = p->v_cache;
    a.path = p->path;
    a.kept = p->kept;
    a.lens_out = p->seq_lens_out;
    a.keep_history = keep_history ? 1 : 0;
    a.cols_per_head = kHeadDim * a.elem_bytes / 16;
    a.cols = p->num_kv_heads * a.cols_per_head;
    const dim3 grid((unsigned)((2 * a.cols + kThreads - 1) / kThreads), (unsigned)p->num_layers,
                    (unsigned)p->batch);
    const cudaError_t e = launch_pdl(tree_commit_kernel, grid, dim3(kThreads), 0,
                                     reinterpret_cast<cudaStream_t>(p->stream), a);
    return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // namespace
}  // namespace gqa

extern "C" {

int gqa_tree_commit(const gqa_tree_commit_params* p) { return gqa::commit(p, false); }

int gqa_tree_commit_history(const gqa_tree_commit_params* p) { return gqa::commit(p, true); }

}  // extern "C"

// How the kernels of gqa_tree_decode share the work: the key tiles of all units in one flat sequence, cut evenly
// over the CTAs, and the merge of the units that were cut.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"
#include "tree_attention.cuh"

namespace gqa {
namespace {

constexpr int kTile = kTreeTileKeys;
constexpr int kUnitPad = 1;   // places a unit counts on top of its tiles
constexpr int kRecordCols = kHeadDim + 2;
constexpr int kLongList = 30;  // records of a unit that a merge shares among its threads
constexpr int kFewGroups = 8;  // groups of 8 rows up to which the merge has a block for every CTA

// x / d for 0 <= x < 2^30, d > 0 and quotients below 2^21: every role divides a few times before its first
// instruction of use, alone in its warp, where the general division is a chain of a hundred cycles.
__device__ __forceinline__ int fast_div(int x, int d) {
    int q = __float2int_rz(__fdividef((float)x, (float)d));  // off by at most one
    const int r = x - q * d;
    q += r >= d ? 1 : 0;
    return r < 0 ? q - 1 : q;
}

// ---- the flat sequence of key tiles -------------------------------------------------------------
struct Tables {
    int32_t* len;   // [batch] keys (0: nothing to do)
    int32_t* n;     // [batch] nodes
    int32_t* base;  // [batch + 1] places before the sequence
};
__device__ __forceinline__ Tables tables_at(int32_t* smem, int batch) {
    return Tables{smem, smem + batch, smem + 2 * batch};
}
size_t table_bytes(int batch) { return (3 * (size_t)batch + 1) * sizeof(int32_t); }

// Runs of tokens (units per KV head) of a tree of n > 0 nodes; QT: query tiles per unit.
template <int QT>
__device__ __forceinline__ int runs_of(const TreeArgs& a, int n) {
    const int run = a.tile_tokens * QT;
    return n <= run ? 1 : fast_div(n + run - 1, run);
}
template <int QT>
__device__ __forceinline__ int units_of(const TreeArgs& a, int n) {
    return a.num_kv_heads * runs_of<QT>(a, n);
}
__device__ __forceinline__ int places_of(int len) { return ceil_div(len, kTile) + kUnitPad; }

// All threads of the block.
template <int QT>
__device__ void build_tables(const TreeArgs& a, const Tables& t) {
    for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
        const TreeSpan s = tree_span(a.cache, b);
        if (!s.ok && blockIdx.x == 0) raise_bad_input(a.cache.status);
        t.n[b] = s.n;
        t.len[b] = s.n > 0 ? s.base + s.n : 0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int per = ceil_div(a.batch, 32);
        const int lo = min(a.batch, (int)threadIdx.x * per), hi = min(a.batch, lo + per);
        int sum = 0;
        for (int b = lo; b < hi; ++b) sum += t.n[b] > 0 ? places_of(t.len[b]) * units_of<QT>(a, t.n[b]) : 0;
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, d);
            if ((int)threadIdx.x >= d) incl += up;
        }
        int run = incl - sum;
        for (int b = lo; b < hi; ++b) {
            t.base[b] = run;
            run += t.n[b] > 0 ? places_of(t.len[b]) * units_of<QT>(a, t.n[b]) : 0;
        }
        if (threadIdx.x == 31) t.base[a.batch] = incl;
    }
    __syncthreads();
}

// The places cut over the CTAs: the first `extra` take per + 1 places, the others per; no more CTAs take
// part than get `fewest` places each. 32-bit arithmetic: every role does this before its first instruction of use.
struct Cut {
    int total;
    int ctas;
    int per;
    int extra;
    __device__ int begin(int c) const { return c >= ctas ? total : c * per + min(c, extra); }
    __device__ int owner(int place) const {
        const int wide = extra * (per + 1);
        return place < wide ? fast_div(place, per + 1) : extra + fast_div(place - wide, per);
    }
};
__device__ __forceinline__ Cut cut_of(const TreeArgs& a, const Tables& t, int fewest) {
    Cut c;
    c.total = t.base[a.batch];
    c.ctas = min(a.ctas, ceil_div(c.total, fewest));
    c.per = c.ctas > 0 ? c.total / c.ctas : 0;
    c.extra = c.total - c.per * c.ctas;
    return c;
}

struct Unit {
    int b;
    int hk;
    int token0;  // first node
    int tokens;  // nodes
    int len;     // keys, the tree's nodes among them
    int n;       // the tree's nodes
    int place;   // first place of the unit
    int tiles;   // key tiles, at places place + kUnitPad ..
};
template <int QT>
__device__ __forceinline__ Unit unit_at(const TreeArgs& a, const Tables& t, int place) {
    int lo = 0, hi = a.batch;  // the last sequence that starts at or before the place
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.base[mid] <= place) lo = mid; else hi = mid;
    }
    Unit u;
    u.b = lo;
    u.len = t.len[lo];
    u.n = t.n[lo];
    const int per = places_of(u.len);
    const int i = fast_div(place - t.base[lo], per);
    const int runs = runs_of<QT>(a, u.n);
    u.hk = runs == 1 ? i : fast_div(i, runs);
    u.token0 = (i - u.hk * runs) * a.tile_tokens * QT;
    u.tokens = min(u.n - u.token0, a.tile_tokens * QT);
    u.place = t.base[lo] + i * per;
    u.tiles = per - kUnitPad;
    return u;
}

// A CTA's next piece at or after `pos` (moved behind it); false at the end of its range.
struct Piece {
    Unit u;
    int tile;    // first key tile
    int tiles;
    bool whole;
};
template <int QT>
__device__ __forceinline__ bool next_piece(const TreeArgs& a, const Tables& t, int* pos, int end, Piece* p) {
    while (*pos < end) {
        p->u = unit_at<QT>(a, t, *pos);
        const int from = max(*pos - p->u.place - kUnitPad, 0);
        const int to = min(end - p->u.place, p->u.tiles + kUnitPad) - kUnitPad;
        *pos = min(end, p->u.place + p->u.tiles + kUnitPad);
        if (to <= from) continue;  // nothing but padding
        p->tile = from;
        p->tiles = to - from;
        p->whole = p->tiles == p->u.tiles;
        return true;
    }
    return false;
}

// Merges the records of the units that were cut: out = sum_i O_i 2^(m_i - m) / sum_i l_i 2^(m_i - m), in a fixed
// order. grid.y: groups of 8 rows. grid.x: the CTAs of the launch before, each of which starts at most one unit that
// others finish and has left its description; or, when there are fewer units than CTAs and many groups of rows, the
// cut units, for which a block looks through all descriptions: blocks with nothing to do then took longer to
// start than the others to merge (64 nodes of 64 / 8 heads over 32768 keys, 4736 blocks or 512: 91 or 86 us; with 64
// rows the search costs more: 11.3 or 12.1 us for 8 nodes over 1024 keys). Thread: row tid % 8 of the group,
// channels 4 (tid / 8 % 32) .. + 3, and of the unit's records those of its part of 256 threads: each record is a round
// trip to L2, six at once, so that long lists (few units cut over all SMs) are shared by PARTS parts of a block.
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }

template <int QT, typename T, int PARTS>
__global__ void __launch_bounds__(256 * PARTS, 4 / PARTS) tree_merge_kernel(const TreeArgs a) {
    __shared__ float4 s_o[PARTS > 1 ? PARTS - 1 : 1][256];
    __shared__ float2 s_ml[PARTS > 1 ? PARTS - 1 : 1][256];
    __shared__ int4 s_head;
    __shared__ int s_count[8 * PARTS], s_tokens, s_c0;
    const int part = threadIdx.x >> 8, tid = threadIdx.x & 255;
    const int r = blockIdx.y * 8 + (tid & 7);  // row of the unit
    const int tile_rows = a.tile_tokens * a.group;
    const int tile = r >= tile_rows ? 1 : 0, row = r - tile * tile_rows;
    const int chunk = tid >> 3;
    const int token = r / a.group;  // of the unit
    const int64_t record = (int64_t)QT * a.tile_rows * kRecordCols;
    const float* rec = a.workspace + (int64_t)tile * a.tile_rows * kRecordCols;
    T* out = static_cast<T*>(a.out) + (r - token * a.group) * kHeadDim + chunk * 4;
    if (threadIdx.x == 0) s_c0 = -1;
    pdl_launch_dependents();
    pdl_wait();
    int c0 = blockIdx.x;
    int4 head;  // last CTA, sequence, KV head, first token
    int tokens;
    if (PARTS == 1 && gridDim.x == (unsigned)a.ctas) {
        head = __ldcg(a.cut_units + 2 * c0);
        if (head.x < 0) return;
        tokens = __ldcg(a.cut_units + 2 * c0 + 1).x;
    } else {
        int passed = 0;
        for (int from = 0; from < a.ctas; from += 256 * PARTS) {
            const int c = from + threadIdx.x, warp = threadIdx.x >> 5;
            int4 one = make_int4(-1, 0, 0, 0);
            int its_tokens = 0;
            if (c < a.ctas) {
                one = __ldcg(a.cut_units + 2 * c);
                its_tokens = __ldcg(a.cut_units + 2 * c + 1).x;
            }
            const uint32_t cut = __ballot_sync(0xffffffffu, one.x >= 0);
            if ((threadIdx.x & 31) == 0) s_count[warp] = __popc(cut);
            __syncthreads();
            int before = passed + __popc(cut & ((1u << (threadIdx.x & 31)) - 1u));
            for (int w = 0; w < 8 * PARTS; ++w) {
                before += w < warp ? s_count[w] : 0;
                passed += s_count[w];
            }
            if (one.x >= 0 && before == (int)blockIdx.x) {
                s_head = one;
                s_tokens = its_tokens;
                s_c0 = c;
            }
            __syncthreads();
        }
        c0 = s_c0;
        if (c0 < 0) return;
        head = s_head;
        tokens = s_tokens;
    }
    const bool live = token < tokens;
    if (PARTS == 1 && !live) return;
    // The part's records: CTAs first .. last.
    const int count = head.x - c0 + 1, share = ceil_div(count, PARTS);
    const int first = c0 + part * share, last = live ? min(head.x, first + share - 1) : -1;
    auto at = [&](int c) { return rec + (int64_t)(2 * c + (c == c0 ? 1 : 0)) * record; };
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kBatch = 6;
    for (int c = first; c <= last; c += kBatch) {
        float mi[kBatch], li[kBatch];
        float4 oi[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            mi[i] = -INFINITY;
            if (c + i > last) continue;
            const float* p = at(c + i);
            mi[i] = __ldcg(p + kHeadDim * a.tile_rows + row);
            li[i] = __ldcg(p + (kHeadDim + 1) * a.tile_rows + row);
            oi[i] = __ldcg(reinterpret_cast<const float4*>(p + ((int64_t)chunk * a.tile_rows + row) * 4));
        }
        float next = m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) next = fmaxf(next, mi[i]);
        const float ref = safe_max(next);
        const float f = ex2_approx(m - ref);
        l *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (c + i > last) continue;
            const float w = ex2_approx(mi[i] - ref);
            l += li[i] * w;
            o.x += oi[i].x * w; o.y += oi[i].y * w; o.z += oi[i].z * w; o.w += oi[i].w * w;
        }
        m = next;
    }
    if (PARTS > 1) {
        if (part > 0) {
            s_o[part - 1][tid] = o;
            s_ml[part - 1][tid] = make_float2(m, l);
        }
        __syncthreads();
        if (part > 0 || !live) return;
        float top = m;
#pragma unroll
        for (int i = 0; i < PARTS - 1; ++i) top = fmaxf(top, s_ml[i][tid].x);
        const float ref = safe_max(top);
        const float f = ex2_approx(m - ref);
        l *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int i = 0; i < PARTS - 1; ++i) {
            const float2 ml = s_ml[i][tid];
            const float4 x = s_o[i][tid];
            const float w = ex2_approx(ml.x - ref);
            l += ml.y * w;
            o.x += x.x * w; o.y += x.y * w; o.z += x.z * w; o.w += x.w * w;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    out += (((int64_t)head.y * a.cache.tokens + head.w + token) * a.num_q_heads + head.z * a.group) * kHeadDim;
    store4(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// Units are at most batch * heads * runs; where the SMs are kLongList or more times as many, a unit has that many records
// (one unit of 252 rows over 16486 keys: 27 us with four parts, 42 with one).
template <int QT, typename T>
cudaError_t launch_merge(const TreeArgs& a, cudaStream_t stream) {
    const int unit = a.tile_tokens * QT;
    const int unit_tokens = a.cache.tokens < unit ? a.cache.tokens : unit;
    const int64_t units = (int64_t)a.batch * a.num_kv_heads * ceil_div(a.cache.tokens, unit);
    const int groups = ceil_div(unit_tokens * a.group, 8);
    const bool search = groups > kFewGroups && units < a.ctas;
    const dim3 grid((unsigned)(search ? units : a.ctas), (unsigned)groups);
    return search && units * kLongList <= a.ctas
               ? launch_pdl(tree_merge_kernel<QT, T, 4>, grid, dim3(1024), 0, stream, a)
               : launch_pdl(tree_merge_kernel<QT, T, 1>, grid, dim3(256), 0, stream, a);
}

}  // namespace
}  // namespace gqa

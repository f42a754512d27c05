// How the kernels of gqa_tree_decode share the work: the key tiles of all units in one flat sequence, cut evenly
// over the CTAs, and the merge of the units that were cut.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"
#include "tree_attention.cuh"

namespace gqa {
namespace {

constexpr int kTile = 128;    // keys per place
constexpr int kUnitPad = 1;   // places a unit counts on top of its tiles
constexpr int kRecordCols = kHeadDim + 2;

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

// Merges the records of the units that were cut: out = sum_i O_i 2^(m_i - m) / sum_i l_i 2^(m_i - m), pieces in
// ascending order. grid.x: CTAs of the launch before, each of which starts at most one unit that others
// finish and has left its description; grid.y: groups of 8 rows. Thread: row tid % 8 of the group, channels
// 4 (tid / 8) .. + 3.
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }

template <int QT, typename T>
__global__ void __launch_bounds__(256, 4) tree_merge_kernel(const TreeArgs a) {
    const int r = blockIdx.y * 8 + (threadIdx.x & 7);  // row of the unit
    const int tile_rows = a.tile_tokens * a.group;
    const int tile = r >= tile_rows ? 1 : 0, row = r - tile * tile_rows;
    const int chunk = threadIdx.x >> 3;
    const int token = r / a.group;  // of the unit
    const int64_t record = (int64_t)QT * a.tile_rows * kRecordCols;
    const float* rec = a.workspace + (int64_t)tile * a.tile_rows * kRecordCols;
    const int c0 = blockIdx.x;
    T* out = static_cast<T*>(a.out) + (r - token * a.group) * kHeadDim + chunk * 4;
    pdl_launch_dependents();
    pdl_wait();
    const int4 head = __ldcg(a.cut_units + 2 * c0);  // last CTA, sequence, KV head, first token
    const int c1 = head.x;
    if (c1 < 0 || token >= __ldcg(a.cut_units + 2 * c0 + 1).x) return;
    auto at = [&](int c) { return rec + (int64_t)(2 * c + (c == c0 ? 1 : 0)) * record; };
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kBatch = 6;
    for (int c = c0; c <= c1; c += kBatch) {
        float mi[kBatch], li[kBatch];
        float4 oi[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            mi[i] = -INFINITY;
            if (c + i > c1) continue;
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
            if (c + i > c1) continue;
            const float w = ex2_approx(mi[i] - ref);
            l += li[i] * w;
            o.x += oi[i].x * w; o.y += oi[i].y * w; o.z += oi[i].z * w; o.w += oi[i].w * w;
        }
        m = next;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    out += (((int64_t)head.y * a.cache.tokens + head.w + token) * a.num_q_heads + head.z * a.group) * kHeadDim;
    store4(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

}  // namespace
}  // namespace gqa

// Tree attention on the 5th-generation tensor cores (gqa_tree_decode, BF16).
//
// Mathematics. For a KV head the queries of up to 16 .. 128 nodes times the group form tiles of 128 rows;
// a tile of keys is 128 positions of the cache. S = Q K^T and O += P V run as 128 x 128 x 128 products with
// FP32 accumulators in tensor memory, P = 2^(c (S - m)) with the running maximum m and sum l in FP32
// registers, one thread per row. P is rounded to BF16 for the second product (V is BF16 and both operands
// have one type); the sum takes the unrounded weights: the rounded ones would cost two instructions more per pair
// (89 us instead of 86 for the wide tree below). m is only moved when a tile's maximum exceeds it by 2^8 (a published idea): the weights then stay
// below 2^8, and O (in tensor memory) is rescaled a few times per sequence instead of once per tile. A weight is off by at most
// half a step (2^-8 of it at its binade's start), so the output is off by that part of the weighted mean of |v| before its own
// rounding. Where one key has nearly all the weight that is a common factor, up to 2^-8 away from 1 unless the
// weight is a power of two: gqa_decode, which sums the rounded weights, returns such a value row unchanged.
// Relative to FP64, all outputs of a measured case together: 0.0022 - 0.0024 (FP32 weights: 0.0017, the output's rounding).
//
// A CTA has two streams of softmax, a warpgroup each. With one query tile (rows <= 128) the streams
// take the key tiles in turn, each with its own O, m and l, merged at the end; with two query tiles they
// share every key tile. While one stream computes weights, the tensor cores work for the other:
//   S(j) .. weights(j) .. O += P(j) V, then S(j + 2) of the same stream, whose S and P share columns.
// Warps 0-7: softmax, warp 8: bulk copies of Q, K and V into 128-byte swizzled rows (a ring of 32 KiB
// tiles), warp 9: its lane 0 issues the products.
//
// Work. All units (sequence, KV head, run of tokens) put their key tiles in one flat sequence that is cut evenly
// over one CTA per SM, whatever the lengths are: few rows over a long history fill the GPU as well as
// a ragged batch does. A piece that is a whole unit writes the output; other pieces leave (O, m, l) as
// a record, at most two per CTA, merged by tree_merge_kernel.
//
// Masks. Keys before the nodes are seen by every row; only tiles that reach the nodes look at the mask (a
// 128-bit window per row). Scores of unseen keys are replaced, not added to, so that K may hold anything there. V
// rows past the end are zeroed in shared memory (0 * NaN). A node's V row that holds an infinity or
// NaN is zeroed too, and added by hand to the rows that see it, in the epilogue.
//
// Measured in a graph, the merge included (32 / 8 heads unless stated): 16 sequences of 256 - 8192 keys, 16 nodes: 66 us, 4.2 TB/s of
// keys and values; 64 nodes of 64 / 8 heads over 32768 keys: 86 us, 800 TFLOP/s (call after call from a host program: 101 us, 680); tensor
// pipe, exponentials and issue each a quarter busy at 8192 keys: two softmax warps per scheduler wait for tensor memory and
// barriers; 8 nodes over 1024 keys: 11.4 us; 4 x 131072 keys, 64 / 8 heads, 8 nodes: 313 - 335 us in a short burst, 390 us at the
// clock of a long one.
#include <cuda_bf16.h>

#include <cstring>
#include <mutex>

#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tree_attention.cuh"
#include "tree_cut.cuh"

namespace gqa {
namespace {

// kTile: also the rows per query tile.
constexpr int kTileBytes = kTile * kHeadDim * 2;
constexpr int kHalfBytes = kTileBytes / 2;      // 64 channels
constexpr int kSlots = 6;                       // query tiles and ring together
constexpr int kSoftmaxThreads = 256;
constexpr int kThreads = kSoftmaxThreads + 64;
constexpr float kLazyMax = 8.0f;                // log2 of how far a score may exceed m
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint32_t kColS = 0, kColO = 256;      // tensor memory: S0, S1, O0, O1 of 128 columns
constexpr uint32_t kColumns = 512;

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Waits with a time limit; also gives up when another role has (its arrivals will not come).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* dead) {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t start = 0;
    for (uint32_t tries = 1;; ++tries) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((tries & 255u) == 0) {
            const uint64_t t = now_ns();
            if (start == 0) start = t;
            if (*dead || t - start > kWaitNs) {
                *dead = 1;
                return false;
            }
        }
    }
}

// wait_bar by a whole warp: one answer, and the lanes together again.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* dead) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, dead));
}

// Barrier 1 of the softmax warps: true when all of them say so.
__device__ __forceinline__ bool meet(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)ok), "n"(kSoftmaxThreads)
        : "memory");
    return all != 0;
}

// ---- order of a piece's tiles in the ring ----------------------------------------------------------
// The first `lead` K tiles, then V(t), K(t + lead) in turn: as the products ask for them.
struct Order {
    int n;
    int lead;
    __device__ int k(int t) const { return t < lead ? t : lead + 2 * (t - lead) + 1; }
    __device__ int v(int t) const { return min(lead, n) + t + min(t, max(n - lead, 0)); }
};

template <int QT>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const TreeArgs a) {
    constexpr int kRing = kSlots - QT;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_kv_full[kRing], s_kv_empty[kRing], s_q_full[2], s_q_empty[2];
    __shared__ uint64_t s_s_full[2], s_p_ready[2], s_o_full[2], s_o_free[2], s_drain;
    __shared__ float s_ml[2][2][kTile];       // m (scaled, log2) and l of the streams' rows
    __shared__ uint32_t s_bad[2][4];          // nodes with a non-finite V row, by turns of the pieces
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    // Rows of a query tile that no token fills are zeros: a long launch runs at the clock that the power limit
    // leaves (1.3 of 1.965 GHz at 128K keys), and products of zeros draw less (391 -> 381 us there).
    const uint32_t q_tiles = smem_u32(smem);
    constexpr uint32_t q_half = kTileBytes / 2;
    constexpr uint32_t q_slots = QT;
    uint8_t* ring_ptr = smem + QT * kTileBytes;
    const uint32_t ring = smem_u32(ring_ptr);
    const Tables tables = tables_at(reinterpret_cast<int32_t*>(smem + kSlots * kTileBytes), a.batch);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* dead = &s_dead;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(smem_u32(&s_kv_full[i]), 1);
            mbar_init(smem_u32(&s_kv_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_q_full[i]), 1);
            mbar_init(smem_u32(&s_q_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_s_full[i]), 1);
            mbar_init(smem_u32(&s_p_ready[i]), 4);
            mbar_init(smem_u32(&s_o_full[i]), 1);
            mbar_init(smem_u32(&s_o_free[i]), 8);
        }
        mbar_init(smem_u32(&s_drain), 1);
        mbar_init_fence();
        s_dead = 0;
        for (int i = 0; i < 8; ++i) (&s_bad[0][0])[i] = 0;
    }
    if (warp == 8 && lane == 0) {
        prefetch_tensormap(&map_q);
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    if (warp == 9) tmem_alloc(smem_u32(&s_tmem), kColumns);
    for (int i = threadIdx.x; i < QT * kTileBytes / 16; i += kThreads) {
        reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
    const int row_token = (threadIdx.x & 127) / a.group;  // of a softmax thread's row, inside its tile
    const int row_head = (threadIdx.x & 127) - row_token * a.group;
    pdl_wait();
    pdl_launch_dependents();
    build_tables<QT>(a, tables);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    const Cut cut = cut_of(a, tables, 2);  // a tile for each stream: fewer records to merge
    int pos = cut.begin(blockIdx.x);
    const int pos_end = cut.begin(blockIdx.x + 1);
    // One query tile: the streams take key tiles in turn; two: both take every key tile.
    auto two_tiles = [&](const Unit& u) { return QT == 2 && u.tokens > a.tile_tokens; };

    if (warp == 8) {
        // ---- bulk copies ---------------------------------------------------------------------------
        const uint64_t policy = l2_policy_evict_first();
        const int boxes = kTile / a.box_keys;
        const uint32_t q_bytes = 2u * a.box_tokens * a.group * 128u;
        uint32_t fills = 0, q_fills = 0;
        Piece p;
        bool ok = true;
        while (ok && next_piece<QT>(a, tables, &pos, pos_end, &p)) {
            const bool two = two_tiles(p.u);
            auto load_q = [&]() {
                for (int st = 0; st < (two ? 2 : 1) && ok; ++st) {
                    const uint32_t slot = q_fills % q_slots, round = q_fills / q_slots;
                    if (round > 0 && !wait_warp(smem_u32(&s_q_empty[slot]), (round - 1) & 1u, dead)) ok = false;
                    if (!ok) return;
                    ++q_fills;
                    if (lane < 2) {
                        const uint32_t bar = smem_u32(&s_q_full[slot]);
                        const int row = p.u.b * a.cache.tokens + p.u.token0 + st * a.tile_tokens;
                        if (lane == 0) mbar_arrive_expect_tx(bar, q_bytes);
                        __syncwarp(3u);
                        asm volatile(
                            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                            " [%0], [%1, {%3, %4, %5}], [%2];"
                            ::"r"(q_tiles + (2 * slot + lane) * q_half), "l"(reinterpret_cast<uint64_t>(&map_q)),
                            "r"(bar), "r"(lane * 64), "r"(p.u.hk * a.group), "r"(row)
                            : "memory");
                    }
                    __syncwarp();
                }
            };
            auto load = [&](const CUtensorMap* map, int t) {
                const uint32_t slot = fills % kRing, round = fills / kRing;
                if (round > 0 && !wait_warp(smem_u32(&s_kv_empty[slot]), (round - 1) & 1u, dead)) ok = false;
                if (!ok) return;
                ++fills;
                const uint32_t bar = smem_u32(&s_kv_full[slot]);
                if (lane == 0) mbar_arrive_expect_tx(bar, kTileBytes);
                __syncwarp();
                // Lane 2 i + h copies half h of the tile's i-th box.
                if (lane < 2 * boxes) {
                    const int box = lane >> 1, h = lane & 1;
                    const int key = (p.tile + t) * kTile + box * a.box_keys;
                    int blk = a.cache.num_blocks, tok = 0;  // a block past the cache reads as zeros
                    if (key < p.u.len) {
                        tok = key;
                        blk = a.cache.fixed_block;
                        if (a.cache.block_table != nullptr) {
                            const int lb = (int)((uint32_t)key / (uint32_t)a.cache.block_tokens);
                            tok = key - lb * a.cache.block_tokens;
                            blk = __ldg(a.cache.block_table + (int64_t)p.u.b * a.cache.blocks_per_seq + lb);
                            if ((uint32_t)blk >= (uint32_t)a.cache.num_blocks) {
                                raise_bad_input(a.cache.status);
                                blk = a.cache.num_blocks;
                            }
                        }
                    }
                    tma_load_4d(ring + slot * kTileBytes + h * kHalfBytes + box * a.box_keys * 128, map, bar,
                                h * 64, a.head_first ? p.u.hk : tok, a.head_first ? tok : p.u.hk, blk, policy);
                }
                __syncwarp();
            };
            // The query tile goes first if its slot is free, else behind a ring full of keys and values: their
            // copies run while the products of the last piece still read its queries.
            const int lead = min(two ? 1 : 2, p.tiles);
            int kt = 0, vt = 0;
            const int q_at = q_fills + (two ? 2 : 1) <= q_slots ? 0 : min(kRing, 2 * p.tiles - 1);
            for (int i = 0; i < 2 * p.tiles && ok; ++i) {
                if (i == q_at) load_q();
                if (kt < min(vt + lead, p.tiles)) {
                    load(&map_k, kt++);
                } else {
                    load(&map_v, vt++);
                }
            }
        }
        if (ok) {
            // The last releases of the slots arrive by themselves, when the products that read them are complete; nothing else
            // waits for them, and the block's barriers must not be gone before.
            for (uint32_t f = fills > (uint32_t)kRing ? fills - kRing : 0; f < fills && ok; ++f) {
                ok = wait_warp(smem_u32(&s_kv_empty[f % kRing]), (f / kRing) & 1u, dead);
            }
            for (uint32_t f = q_fills > q_slots ? q_fills - q_slots : 0; f < q_fills && ok; ++f) {
                ok = wait_warp(smem_u32(&s_q_empty[f % q_slots]), (f / q_slots) & 1u, dead);
            }
        }
        if (!ok) {
            // Copies in flight land before the block ends (again with a limit).
            if (lane == 0) {
                volatile int fresh = 0;
                for (uint32_t f = fills > (uint32_t)kRing ? fills - kRing : 0; f < fills; ++f) {
                    wait_bar(smem_u32(&s_kv_full[f % kRing]), (f / kRing) & 1u, &fresh);
                }
                for (uint32_t f = q_fills > q_slots ? q_fills - q_slots : 0; f < q_fills; ++f) {
                    wait_bar(smem_u32(&s_q_full[f % q_slots]), (f / q_slots) & 1u, &fresh);
                }
            }
            __syncwarp();
        }
    } else if (warp == 9) {
        // ---- products ------------------------------------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t kShapeS = mma_shape(kTile, kTile, false);
            constexpr uint32_t kShapeO = mma_shape(kTile, kHeadDim, true);
            uint32_t ring_pos = 0, q_pos = 0;
            uint32_t jobs[2] = {0, 0}, pieces[2] = {0, 0};  // per stream, over all pieces
            bool ok = true;
            Piece p;
            while (ok && next_piece<QT>(a, tables, &pos, pos_end, &p)) {
                const bool two = two_tiles(p.u);
                const int count = two ? 2 * p.tiles : p.tiles;  // job j: stream j & 1, key tile j or j / 2
                const Order order = {p.tiles, two ? 1 : 2};
                for (int st = 0; st < (two ? 2 : 1) && ok; ++st) {
                    const uint32_t f = q_pos + st;
                    ok = wait_bar(smem_u32(&s_q_full[f % q_slots]), (f / q_slots) & 1u, dead);
                }
                auto issue_s = [&](int j) {
                    const int st = j & 1, t = two ? j >> 1 : j;
                    const uint32_t f = ring_pos + order.k(t), slot = f % kRing;
                    ok = ok && wait_bar(smem_u32(&s_kv_full[slot]), (f / kRing) & 1u, dead);
                    if (!ok) return;
                    const uint32_t q = matrix_lo(q_tiles + ((q_pos + (two ? st : 0)) % q_slots) * 2 * q_half, 16);
                    const uint32_t k = matrix_lo(ring + slot * kTileBytes, 16);
#pragma unroll
                    for (int i = 0; i < kHeadDim / 16; ++i) {
                        tc_mma_ss(tmem + kColS + st * 128, q + (i >> 2) * (q_half >> 4) + (i & 3) * 2,
                                  k + (i >> 2) * (kHalfBytes >> 4) + (i & 3) * 2, matrix_hi(1024), kShapeS, i > 0);
                    }
                    tc_commit(smem_u32(&s_s_full[st]));
                    if (!two || st == 1) tc_commit(smem_u32(&s_kv_empty[slot]));
                    if (j == count - 1) {
                        for (int i = 0; i < (two ? 2 : 1); ++i) tc_commit(smem_u32(&s_q_empty[(q_pos + i) % q_slots]));
                    }
                };
                issue_s(0);
                if (count > 1) issue_s(1);
                for (int j = 0; j < count && ok; ++j) {
                    const int st = j & 1, t = two ? j >> 1 : j;
                    const uint32_t f = ring_pos + order.v(t), slot = f % kRing;
                    ok = wait_bar(smem_u32(&s_kv_full[slot]), (f / kRing) & 1u, dead);
                    if (ok && j < 2 && pieces[st] > 0) {  // the last piece's O has been read
                        ok = wait_bar(smem_u32(&s_o_free[st]), (pieces[st] - 1) & 1u, dead);
                    }
                    ok = ok && wait_bar(smem_u32(&s_p_ready[st]), jobs[st] & 1u, dead);
                    ++jobs[st];
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v = matrix_lo(ring + slot * kTileBytes, kHalfBytes);
#pragma unroll
                    for (int i = 0; i < kTile / 16; ++i) {
                        tc_mma_ts(tmem + kColO + st * 128, tmem + kColS + st * 128 + i * 8, v + i * (2048 >> 4),
                                  matrix_hi(1024), kShapeO, j >= 2 || i > 0);
                    }
                    if (!two || st == 1) tc_commit(smem_u32(&s_kv_empty[slot]));
                    if (j + 2 >= count) {
                        tc_commit(smem_u32(&s_o_full[st]));
                        ++pieces[st];
                    } else {
                        issue_s(j + 2);
                    }
                }
                ring_pos += 2 * p.tiles;
                q_pos += two ? 2 : 1;
            }
            if (!ok) {
                // Products in flight finish before tensor memory is given back (with a limit).
                volatile int fresh = 0;
                tc_commit(smem_u32(&s_drain));
                wait_bar(smem_u32(&s_drain), 0, &fresh);
            }
        }
        __syncwarp();
    } else {
        // ---- weights ---------------------------------------------------------------------------------
        const int st = warp >> 2;             // stream
        const int row = threadIdx.x & 127;    // of the stream's query tile; lane of tensor memory
        const uint32_t my_lanes = tmem + ((uint32_t)(warp & 3) << 21);
        const uint32_t my_s = my_lanes + kColS + st * 128;
        const float scale = a.scale_log2;
        const int words = (a.cache.tokens + 31) / 32;
        uint32_t ring_pos = 0, jobs = 0, pieces[2] = {0, 0}, turn = 0;
        bool ok = true;
        int last_cta = -1;  // of the unit this CTA starts and others finish
        Piece p;
        while (ok && next_piece<QT>(a, tables, &pos, pos_end, &p)) {
            if (threadIdx.x == 0 && !p.whole && p.tile == 0) {
                last_cta = cut.owner(p.u.place + kUnitPad + p.u.tiles - 1);
                a.cut_units[2 * blockIdx.x] = make_int4(last_cta, p.u.b, p.u.hk, p.u.token0);
                a.cut_units[2 * blockIdx.x + 1] = make_int4(p.u.tokens, 0, 0, 0);
            }
            const bool two = two_tiles(p.u);
            const int count = two ? 2 * p.tiles : p.tiles;
            const Order order = {p.tiles, two ? 1 : 2};
            const int in_unit = row_token + (two ? st * a.tile_tokens : 0);
            const int token = p.u.token0 + in_unit;
            const bool live = row < a.tile_tokens * a.group && in_unit < p.u.tokens;
            const bool any_live = __any_sync(0xffffffffu, live);
            const int64_t mask_row = (int64_t)p.u.b * a.cache.tokens + token;
            const int base = p.u.len - p.u.n;

            // Bits of 32 keys from tree index `first` (negative: history) that this row sees.
            auto window = [&](int first) -> uint32_t {
                if (first <= -32) return 0xffffffffu;
                auto word = [&](int w) -> uint32_t {  // nodes 32 w .. 32 w + 31
                    if (w < 0) return 0xffffffffu;
                    if (w * 32 >= p.u.n) return 0u;
                    uint32_t bits = a.mask != nullptr ? __ldg(a.mask + mask_row * words + w)
                                    : token >= w * 32 + 31 ? 0xffffffffu
                                    : token < w * 32       ? 0u
                                                           : (2u << (token - w * 32)) - 1u;
                    if (p.u.n - w * 32 < 32) bits &= (1u << (p.u.n - w * 32)) - 1u;
                    return bits;
                };
                const int w = first >> 5;  // rounds down
                return __funnelshift_r(word(w), word(w + 1), first & 31);
            };

            float m = -INFINITY, l = 0.0f;  // m: of the raw scores
#pragma unroll 1
            for (int j = st; j < count && ok; j += 2, ++jobs) {
                const int t = two ? j >> 1 : j;
                const int key0 = (p.tile + t) * kTile;
                ok = wait_warp(smem_u32(&s_s_full[st]), jobs & 1u, dead);
                if (!ok) break;
                tc_fence_after();
                const bool tail = key0 + kTile > base;
                if (tail) {
                    // V: rows past the end become zeros, rows of nodes are looked over.
                    const uint32_t f = ring_pos + order.v(t), slot = f % kRing;
                    ok = wait_warp(smem_u32(&s_kv_full[slot]), (f / kRing) & 1u, dead);
                    if (!ok) break;
                    const int key = key0 + row;
                    uint4* v = reinterpret_cast<uint4*>(ring_ptr + slot * kTileBytes + row * 128);
                    bool clear = key >= p.u.len;
                    if (key >= base && !clear) {
#pragma unroll 1
                        for (int i = 0; i < 16; ++i) {
                            const uint4 x = v[(i >> 3) * (kHalfBytes / 16) + (i & 7)];
                            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                clear = clear || (e[c] & 0x7f80u) == 0x7f80u || (e[c] & 0x7f800000u) == 0x7f800000u;
                            }
                        }
                        // With two query tiles the other stream looks over the same row and may have zeroed part of it
                        // already: it names the row first, so a reader of its zeros finds the name.
                        uint32_t* named = &s_bad[turn & 1][(key - base) >> 5];
                        const uint32_t bit = 1u << ((key - base) & 31);
                        if (clear) {
                            atomicOr(named, bit);
                            __threadfence_block();
                        } else if (two) {
                            __threadfence_block();
                            clear = (*reinterpret_cast<volatile uint32_t*>(named) & bit) != 0;
                        }
                    }
                    if (clear) {
#pragma unroll 1
                        for (int i = 0; i < 16; ++i) v[(i >> 3) * (kHalfBytes / 16) + (i & 7)] = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                if (any_live) {
                    // Rolled loops over 64 columns, read from tensor memory twice: the whole body stays in the
                    // instruction cache next to the warp (128 columns in registers and unrolled ran at half the rate).
                    if (tail) {
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t sees = live ? window(key0 + 32 * c - base) : 0u;
                            uint32_t s[32];
                            __syncwarp();
                            tmem_load32(my_s + 32 * c, s);
                            tmem_loaded(s);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                if (!(sees >> i & 1u)) s[i] = 0xff800000u;
                            }
                            tmem_store32(my_s + 32 * c, s);
                        }
                        tmem_stored();
                    }
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        uint32_t s[2][32];
                        tmem_load32(my_s + 64 * half, s[0]);
                        tmem_load32(my_s + 64 * half + 32, s[1]);
                        tmem_loaded(s[0]);
                        tmem_loaded(s[1]);
                        float top[4] = {mx, mx, mx, mx};
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            top[i & 3] = fmaxf(top[i & 3], fmaxf(__uint_as_float(s[0][i]), __uint_as_float(s[1][i])));
                        }
                        mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    }
                    if (j < 2) {
                        m = mx;
                    } else {
                        const bool grow = (mx - m) * scale > kLazyMax || (m == -INFINITY && mx > m);
                        if (__any_sync(0xffffffffu, grow)) {
                            // S(j) was issued behind the product with the last P: O is at rest.
                            const float next = grow ? mx : m;
                            const float alpha = grow ? ex2_approx((m - next) * scale) : 1.0f;
                            m = next;
                            l *= alpha;
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t o[32];
                                const uint32_t at = my_lanes + kColO + st * 128 + 32 * c;
                                tmem_load32(at, o);
                                tmem_loaded(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                }
                                tmem_store32(at, o);
                            }
                        }
                    }
                    const float off = safe_max(m) * scale;
                    const Two factor = two_of(scale, scale), minus = two_of(-off, -off);
                    Two sum[2] = {two_of(0.0f, 0.0f), two_of(0.0f, 0.0f)};
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        uint32_t s[2][32], w[32];
                        tmem_load32(my_s + 64 * half, s[0]);
                        tmem_load32(my_s + 64 * half + 32, s[1]);
                        tmem_loaded(s[0]);
                        tmem_loaded(s[1]);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            float e0, e1;
                            split(fma2(two_of(s[i >> 4][2 * i & 31], s[i >> 4][(2 * i & 31) + 1]), factor, minus), &e0, &e1);
                            e0 = ex2_approx(e0);
                            e1 = ex2_approx(e1);
                            sum[i & 1] = add2(sum[i & 1], two_of(e0, e1));
                            w[i] = pack_bf16(e0, e1);
                        }
                        tmem_store32(my_s + 32 * half, w);
                    }
                    float l0, l1;
                    split(add2(sum[0], sum[1]), &l0, &l1);
                    l += l0 + l1;
                    tmem_stored();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_p_ready[st]));
            }
            ring_pos += 2 * p.tiles;
            // ---- the end of the piece ------------------------------------------------------------------
            const bool active1 = count > 1;
            ok = ok && wait_warp(smem_u32(&s_o_full[0]), pieces[0] & 1u, dead) &&
                 (!active1 || wait_warp(smem_u32(&s_o_full[1]), pieces[1] & 1u, dead));
            // Both warpgroups meet here, also when a wait ran out, and go on or leave together.
            s_ml[st][0][row] = m * scale;
            s_ml[st][1][row] = l;
            if (threadIdx.x < 4) s_bad[(turn + 1) & 1][threadIdx.x] = 0;
            tc_fence_before();
            ok = meet(ok);
            tc_fence_after();
            if (!ok) break;
            // Two tiles: this stream's rows, all channels. One tile: both streams' sums of the
            // rows, merged; the warpgroups take 64 channels each.
            float f0 = 1.0f, f1 = 0.0f, m_row, l_row;
            if (two) {
                m_row = s_ml[st][0][row];
                l_row = l;
            } else {
                const float m0 = s_ml[0][0][row], m1 = active1 ? s_ml[1][0][row] : -INFINITY;
                m_row = fmaxf(m0, m1);
                f0 = ex2_approx(m0 - safe_max(m_row));
                f1 = ex2_approx(m1 - safe_max(m_row));
                l_row = s_ml[0][1][row] * f0 + (active1 ? s_ml[1][1][row] * f1 : 0.0f);
            }
            if (any_live) {
                const int chunk0 = two ? 0 : 2 * st, chunks = two ? 4 : 2;
                const float inv = l_row == 0.0f ? 0.0f : 1.0f / l_row;
                const int head = p.u.hk * a.group + row_head;
                __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) +
                                     (mask_row * a.num_q_heads + head) * kHeadDim;
                float* rec = a.workspace + ((int64_t)(2 * blockIdx.x + (p.tile == 0 ? 1 : 0)) * QT + (two ? st : 0)) *
                                               a.tile_rows * kRecordCols;
                uint32_t bad[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) bad[i] = s_bad[turn & 1][i];
#pragma unroll 1
                for (int c = chunk0; c < chunk0 + chunks; ++c) {
                    uint32_t o[32];
                    float acc[32];
                    tmem_load32(my_lanes + kColO + (two ? st : 0) * 128 + 32 * c, o);
                    tmem_loaded(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[i] = __uint_as_float(o[i]) * f0;
                    if (!two && active1) {
                        tmem_load32(my_lanes + kColO + 128 + 32 * c, o);
                        tmem_loaded(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) acc[i] += __uint_as_float(o[i]) * f1;
                    }
                    if ((bad[0] | bad[1] | bad[2] | bad[3]) != 0 && live) {
                        // Nodes left out of the product: their weights again, then channel by channel.
                        for (int node = 0; node < p.u.n; ++node) {
                            if (!(s_bad[turn & 1][node >> 5] >> (node & 31) & 1u)) continue;
                            if (!tree_sees(a.mask, mask_row, words, token, node)) continue;
                            int64_t at = 0;
                            if (!tree_row(a.cache, p.u.b, base + node, &at)) continue;
                            at += (int64_t)p.u.hk * a.cache.stride_head;
                            const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.k_cache) + at;
                            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v_cache) + at;
                            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) +
                                                     mask_row * a.q_stride + head * kHeadDim;
                            float dot = 0.0f;
                            for (int d = 0; d < kHeadDim; ++d) dot += __bfloat162float(q[d]) * __bfloat162float(k[d]);
                            const float w = ex2_approx(dot * scale - safe_max(m_row));
#pragma unroll
                            for (int i = 0; i < 32; ++i) acc[i] += w * __bfloat162float(v[32 * c + i]);
                        }
                    }
                    if (live && p.whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 w;
                            w.x = pack_bf16(acc[8 * i] * inv, acc[8 * i + 1] * inv);
                            w.y = pack_bf16(acc[8 * i + 2] * inv, acc[8 * i + 3] * inv);
                            w.z = pack_bf16(acc[8 * i + 4] * inv, acc[8 * i + 5] * inv);
                            w.w = pack_bf16(acc[8 * i + 6] * inv, acc[8 * i + 7] * inv);
                            *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = w;
                        }
                    } else if (live) {
                        // [channel / 4][row][4]: a warp writes 512 contiguous bytes.
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            *reinterpret_cast<float4*>(rec + ((8 * c + i) * a.tile_rows + row) * 4) =
                                make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
                        }
                    }
                    __syncwarp();
                }
                if (live && !p.whole && (two || st == 0)) {
                    rec[kHeadDim * a.tile_rows + row] = m_row;
                    rec[(kHeadDim + 1) * a.tile_rows + row] = l_row;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&s_o_free[0]));
                if (active1) mbar_arrive(smem_u32(&s_o_free[1]));
            }
            ++pieces[0];
            if (active1) ++pieces[1];
            ++turn;
        }
        if (threadIdx.x == 0 && last_cta < 0) a.cut_units[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    __syncthreads();
    if (s_dead && threadIdx.x == 0 && a.cache.status != nullptr) atomicExch(a.cache.status, kStatusStageTimeout);
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, kColumns);
    }
}

int query_tiles(int32_t tokens, int32_t group) { return tokens * group > kTile ? 2 : 1; }

int rows_per_tile(int32_t tokens, int32_t group) {
    const int per = kTile / group, used = tokens < per ? tokens : per;
    return (used * group + 31) / 32 * 32;
}

template <int QT>
int launch(const TreeArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
           cudaStream_t stream) {
    const size_t smem = 1024 + kSlots * kTileBytes + table_bytes(a.batch);
    auto kernel = tree_attention_kernel<QT>;
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
    if (launch_pdl(kernel, dim3(a.ctas), dim3(kThreads), smem, stream, mq, mk, mv, a) != cudaSuccess) {
        return GQA_ERR_CUDA;
    }
    return launch_merge<QT, __nv_bfloat16>(a, stream) == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // namespace

// Records, then the descriptions of the cut units.
static size_t record_bytes(int32_t tokens, int32_t group, int32_t ctas) {
    return (size_t)2 * ctas * query_tiles(tokens, group) * rows_per_tile(tokens, group) * kRecordCols * sizeof(float);
}

size_t tree_attention_workspace(int32_t tokens, int32_t group, int32_t ctas) {
    return record_bytes(tokens, group, ctas) + 2 * (size_t)ctas * sizeof(int4);
}

int launch_tree_attention(TreeArgs a, const gqa_kv_layout& layout, int32_t sm_count, cudaStream_t stream) {
    a.ctas = sm_count;
    a.cut_units = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(a.workspace) +
                                          record_bytes(a.cache.tokens, a.group, sm_count));
    a.tile_tokens = kTile / a.group;
    a.tile_rows = rows_per_tile(a.cache.tokens, a.group);
    a.box_tokens = a.cache.tokens < a.tile_tokens ? a.cache.tokens : a.tile_tokens;
    // Bulk copies stay inside a block: the largest of 128, 64, 32 rows that divides it.
    a.box_keys = kTile;
    if (a.cache.block_table != nullptr && a.cache.blocks_per_seq > 1) {
        while (layout.block_tokens % a.box_keys != 0) a.box_keys /= 2;
    }
    // Places are 32-bit numbers.
    const int64_t per_seq = (int64_t)(ceil_div(a.cache.capacity, kTile) + kUnitPad) * a.num_kv_heads *
                            ceil_div(a.cache.tokens, a.tile_tokens);
    if (per_seq * a.batch > (1 << 30)) return GQA_ERR_SHAPE;
    if ((int64_t)a.batch * a.cache.tokens > INT32_MAX) return GQA_ERR_SHAPE;
    CUtensorMap mq, mk, mv;
    bool head_first = false;
    int rc = tree_cache_map(a.k_cache, layout, a.num_kv_heads, a.box_keys, &head_first, &mk);
    if (rc == GQA_OK) rc = tree_cache_map(a.v_cache, layout, a.num_kv_heads, a.box_keys, &head_first, &mv);
    if (rc == GQA_OK) {
        rc = tree_query_map(a.q, (int64_t)a.batch * a.cache.tokens, a.q_stride, a.num_q_heads, a.group, a.box_tokens, &mq);
    }
    if (rc != GQA_OK) return rc;
    a.head_first = head_first ? 1 : 0;
    return query_tiles(a.cache.tokens, a.group) == 2 ? launch<2>(a, mq, mk, mv, stream)
                                                     : launch<1>(a, mq, mk, mv, stream);
}

}  // namespace gqa

"""Tree drafting on the GPU: attention of the nodes, rotary append, verification, commit, and the four as a
decode loop runs them, each against its definition in FP64 (tree_helpers.py)."""
import math

import numpy as np
import pytest
import torch

import tree_helpers as TH
from tree_helpers import D, DEV

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gqa(built_lib):
    import llminfer_b200 as pkg
    return pkg


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- attention ------------------------------------------------------------------------------------

def attend(gqa, seed, lens, sizes, tokens, hq, hkv, block, dtype, kind, touch=None, capacity=None):
    """Runs tree_decode on seeded inputs and compares every element with the FP64 definition."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    batch = len(lens)
    capacity = capacity or max(max(lens), 1)
    cache = TH.Cache(gqa, rng, lens, capacity, hkv, block, dtype).fill(gen, lens)
    q = torch.randn(batch, tokens, hq, D, generator=gen).to(dtype)
    sees = []
    for n in sizes:
        if kind == "tree":
            sees.append(TH.ancestors(TH.random_parents(rng, n)) if n else np.zeros((0, 0), dtype=bool))
        elif kind == "causal":
            sees.append(np.tril(np.ones((n, n), dtype=bool)))
        elif kind == "none":
            sees.append(np.zeros((n, n), dtype=bool))
        else:
            sees.append(rng.random((n, n)) < 0.3)
    if touch:
        touch(cache, q, sees)
    mask = None if kind == "causal" else TH.pack_mask(sees, tokens)
    if mask is not None and tokens % 32:  # bits of nodes that do not exist mean nothing
        mask[..., -1] |= -(1 << (tokens % 32)) if tokens % 32 < 31 else -(1 << 31)
    k, v = cache.device()
    out = torch.full((batch, tokens, hq, D), 7.0, dtype=dtype, device=DEV)
    ws = gqa.tree_workspace(batch, tokens, hq, hkv, DEV, dtype)
    status = ints([0])
    gqa.tree_decode(q.to(DEV), k, v, out, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=ints(lens),
                    mask=None if mask is None else mask.to(DEV), tree_sizes=ints(sizes), block_table=cache.table,
                    workspace=ws, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    got = out.cpu().double()
    for b, n in enumerate(sizes):
        assert (got[b, n:] == 7.0).all(), "rows behind the tree's end changed"
        if n == 0:
            continue
        kb, vb = cache.rows("k", b, lens[b]), cache.rows("v", b, lens[b])
        want, spread, size = TH.attention(q[b, :n], kb, vb, lens[b] - n, sees[b])
        bound = TH.attention_bound(want, spread, size, lens[b], dtype)
        off = (got[b, :n] - want).abs()
        assert torch.isfinite(got[b, :n]).all()
        assert (off <= bound).all(), (b, float((off / bound).max()), torch.nonzero(off > bound)[0].tolist())


@pytest.mark.parametrize("kind", ["tree", "causal", "random"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,sizes,tokens,hq,hkv,block", [
    ([1], [1], 1, 8, 8, 0),                 # nothing but the root
    ([8], [8], 8, 32, 8, 0),                # no history
    ([100], [5], 5, 16, 8, 0),              # one ragged tile
    ([128], [8], 8, 32, 8, 0),              # a full tile, nodes at its end
    ([130], [9], 9, 32, 8, 0),              # nodes on both sides of a tile's edge
    ([257], [1], 1, 64, 8, 0),
    ([1111], [33], 33, 12, 2, 0),           # group 6, two mask words, 198 rows
    ([700], [64], 64, 16, 2, 0),            # group 8: 512 rows
    ([300], [128], 128, 7, 1, 0),           # group 7, the widest tree
    ([513, 64, 3, 0, 200], [8, 8, 3, 0, 1], 8, 32, 8, 64),
    ([96, 161, 1], [20, 7, 1], 20, 10, 2, 32),      # group 5, pages smaller than a tile
    ([97, 500, 289], [16, 16, 5], 16, 8, 2, 96),    # pages that end inside a tile
    ([1000, 255, 256, 1281], [12, 2, 12, 9], 12, 24, 8, 256),
])
def test_attention(gqa, lens, sizes, tokens, hq, hkv, block, dtype, kind):
    attend(gqa, sum(lens) + tokens * 7 + hq, lens, sizes, tokens, hq, hkv, block, dtype, kind)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_over_a_long_history_cut_over_many_blocks(gqa, dtype):
    attend(gqa, 5, [6000], [12], 12, 8, 1, 0, dtype, "tree")


@pytest.mark.parametrize("tokens,hq,hkv,length", [(36, 7, 1, 9001), (128, 8, 2, 5000), (33, 8, 1, 300)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_units_of_many_rows_merge_long_lists_of_pieces(gqa, tokens, hq, hkv, length, dtype):
    attend(gqa, tokens, [length], [tokens], tokens, hq, hkv, 0, dtype, "random")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing_are_zero(gqa, dtype):
    attend(gqa, 3, [6, 40], [6, 6], 6, 8, 2, 32, dtype, "none")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_nodes_may_hold_anything(gqa, dtype, bad):
    def touch(cache, q, sees):
        # Nodes 3 and 7 are seen by nobody, whatever their rows hold.
        for b in range(2):
            n = sees[b].shape[0]
            for j in (3, 7):
                sees[b][:, j] = False
                at = (0,) + cache.at(b, lens[b] - n + j)
                cache.k[at] = bad
                cache.v[at] = bad
    lens = [140, 70]
    attend(gqa, 11, lens, [14, 9], 14, 16, 2, 64, dtype, "random", touch)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_bad_row_reaches_only_those_that_see_it(gqa, dtype):
    """A node whose value row holds NaN and infinities: rows that see it carry them in those channels,
    all others are as if it were not there."""
    rng, gen = np.random.default_rng(2), torch.Generator().manual_seed(2)
    n, hq, hkv, length = 40, 16, 2, 150
    cache = TH.Cache(gqa, rng, [length], 192, hkv, 0, dtype).fill(gen, [length])
    sees = [rng.random((n, n)) < 0.4]
    at = (0,) + cache.at(0, length - n + 5)
    clean = cache.v[at].clone()
    cache.v[at][0, 9], cache.v[at][0, 77], cache.v[at][1, 3] = float("nan"), float("inf"), -float("inf")
    poisoned = cache.v[at].clone()
    q = torch.randn(1, n, hq, D, generator=gen).to(dtype)
    k, v = cache.device()
    out = torch.zeros(1, n, hq, D, dtype=dtype, device=DEV)
    ws = gqa.tree_workspace(1, n, hq, hkv, DEV, dtype)
    gqa.tree_decode(q.to(DEV), k, v, out, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=ints([length]),
                    mask=TH.pack_mask(sees, n).to(DEV), workspace=ws)
    got = out[0].cpu().double()
    cache.v[at] = torch.where(torch.isfinite(poisoned), poisoned, torch.zeros_like(clean))
    want, spread, size = TH.attention(q[0], cache.rows("k", 0, length), cache.rows("v", 0, length), length - n, sees[0])
    bound = TH.attention_bound(want, spread, size, length, dtype)
    for t in range(n):
        for h in range(hq):
            hit = [c for c in range(D) if not torch.isfinite(poisoned[h // 8, c])] if sees[0][t, 5] else []
            rest = [c for c in range(D) if c not in hit]
            assert ((got[t, h] - want[t, h]).abs() <= bound[t, h])[rest].all(), (t, h)
            for c in hit:
                assert (torch.isnan(got[t, h, c]) if torch.isnan(poisoned[h // 8, c]) else got[t, h, c] == poisoned[h // 8, c].double())


def test_attention_reads_queries_inside_packed_rows(gqa):
    rng, gen = np.random.default_rng(4), torch.Generator().manual_seed(4)
    hq, hkv, tokens, lens = 16, 4, 6, [90, 200]
    cache = TH.Cache(gqa, rng, lens, 256, hkv, 64, BF16).fill(gen, lens)
    k, v = cache.device()
    packed = torch.randn(2, tokens, hq + 2 * hkv, D, generator=gen).to(BF16).to(DEV)
    ws = gqa.tree_workspace(2, tokens, hq, hkv, DEV)
    outs = []
    for q in (packed[:, :, :hq], packed[:, :, :hq].contiguous()):
        out = torch.zeros(2, tokens, hq, D, dtype=BF16, device=DEV)
        gqa.tree_decode(q, k, v, out, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=ints(lens),
                        block_table=cache.table, workspace=ws)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().sum() > 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,sizes", [([65, 10], [4, 4]), ([20, 3], [4, 4]), ([20, 10], [5, 4]), ([20, 10], [4, -1])])
def test_attention_skips_and_reports_bad_lengths(gqa, lens, sizes, dtype):
    """Sequence 0 or 1 out of range (longer than its pages, shorter than its tree, sizes out of range):
    skipped, reported, the other one as always."""
    rng, gen = np.random.default_rng(6), torch.Generator().manual_seed(6)
    hq, hkv, tokens = 8, 2, 4
    ok = [n <= 64 and 0 <= s <= tokens and n >= s for n, s in zip(lens, sizes)]
    cache = TH.Cache(gqa, rng, [64, 64], 64, hkv, 32, dtype).fill(gen, [64, 64])
    q = torch.randn(2, tokens, hq, D, generator=gen).to(dtype)
    k, v = cache.device()
    out = torch.full((2, tokens, hq, D), 7.0, dtype=dtype, device=DEV)
    status = ints([0])
    gqa.tree_decode(q.to(DEV), k, v, out, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=ints(lens),
                    tree_sizes=ints(sizes), block_table=cache.table, status=status,
                    workspace=gqa.tree_workspace(2, tokens, hq, hkv, DEV, dtype))
    assert int(status) == 3
    got = out.cpu().double()
    for b in range(2):
        if not ok[b]:
            assert (got[b] == 7.0).all()
            continue
        n = sizes[b]
        want, spread, size = TH.attention(q[b, :n], cache.rows("k", b, lens[b]), cache.rows("v", b, lens[b]),
                                          lens[b] - n, np.tril(np.ones((n, n), dtype=bool)))
        assert ((got[b, :n] - want).abs() <= TH.attention_bound(want, spread, size, lens[b], dtype)).all()


def test_attention_reports_missing_blocks(gqa):
    rng, gen = np.random.default_rng(7), torch.Generator().manual_seed(7)
    cache = TH.Cache(gqa, rng, [64, 64], 64, 2, 32, BF16).fill(gen, [64, 64])
    cache.table[0, 0] = -1
    cache.table[1, 1] = 1000
    k, v = cache.device()
    q = torch.randn(2, 4, 8, D, generator=gen).to(BF16).to(DEV)
    status = ints([0])
    gqa.tree_decode(q, k, v, torch.zeros_like(q), num_kv_heads=2, layout=cache.layout, seq_lens_dev=ints([64, 64]),
                    block_table=cache.table, status=status, workspace=gqa.tree_workspace(2, 4, 8, 2, DEV))
    assert int(status) == 3


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_in_a_captured_graph_follows_lengths_and_masks(gqa, dtype):
    rng, gen = np.random.default_rng(8), torch.Generator().manual_seed(8)
    hq, hkv, tokens, cap = 16, 2, 10, 2048
    cache = TH.Cache(gqa, rng, [cap] * 3, cap, hkv, 64, dtype).fill(gen, [cap] * 3)
    k, v = cache.device()
    q = torch.randn(3, tokens, hq, D, generator=gen).to(dtype).to(DEV)
    lens, sizes = ints([100, 30, 2000]), ints([10, 10, 10])
    mask = torch.zeros(3, tokens, 1, dtype=torch.int32, device=DEV)
    out, ws = torch.zeros(3, tokens, hq, D, dtype=dtype, device=DEV), gqa.tree_workspace(3, tokens, hq, hkv, DEV, dtype)

    def call(o):
        gqa.tree_decode(q, k, v, o, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=lens, mask=mask,
                        tree_sizes=sizes, block_table=cache.table, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for l, s in (([100, 30, 2000], [10, 10, 10]), ([11, 2048, 700], [3, 10, 0]), ([1500, 1501, 5], [1, 10, 5])):
        lens.copy_(ints(l))
        sizes.copy_(ints(s))
        mask.random_(0, 1 << 10)
        out.zero_()
        graph.replay()
        eager = torch.zeros_like(out)
        call(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    assert out.abs().sum() > 0


def test_attention_on_two_streams_with_a_workspace_each(gqa):
    rng, gen = np.random.default_rng(9), torch.Generator().manual_seed(9)
    hq, hkv, tokens, cap = 16, 4, 16, 4096
    cache = TH.Cache(gqa, rng, [cap] * 2, cap, hkv, 64, BF16)
    k = torch.randn(cache.k.shape[1:], generator=gen).to(BF16).to(DEV)
    v = torch.randn(cache.k.shape[1:], generator=gen).to(BF16).to(DEV)
    qs = [torch.randn(2, tokens, hq, D, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    lens = [ints([4096, 3000]), ints([2500, 4000])]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [gqa.tree_workspace(2, tokens, hq, hkv, DEV) for _ in range(2)]

    def call(i, o):
        gqa.tree_decode(qs[i], k, v, o, num_kv_heads=hkv, layout=cache.layout, seq_lens_dev=lens[i],
                        block_table=cache.table, workspace=ws[i])

    want = [torch.zeros_like(qs[0]) for _ in range(2)]
    for i in range(2):
        call(i, want[i])
    torch.cuda.synchronize()
    got = [[torch.zeros_like(qs[0]) for _ in range(8)] for _ in range(2)]
    for r in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                call(i, got[i][r])
    torch.cuda.synchronize()
    for i in range(2):
        for r in range(8):
            assert torch.equal(got[i][r], want[i])


def test_attention_in_a_cache_beyond_32_bit_offsets(gqa):
    """A BF16 cache of more than 2^31 elements whose used blocks lie at both ends."""
    gen = torch.Generator().manual_seed(10)
    hkv, block, tokens, hq, length = 8, 256, 6, 16, 600
    blocks = (1 << 31) // (hkv * block * D) + 40
    k = torch.empty(blocks, hkv, block, D, dtype=BF16, device=DEV)
    v = torch.empty(blocks, hkv, block, D, dtype=BF16, device=DEV)
    used = [blocks - 1, 0, blocks - 7]
    rows = torch.randn(2, 3, hkv, block, D, generator=gen).to(BF16)
    for i, blk in enumerate(used):
        k[blk], v[blk] = rows[0, i].to(DEV), rows[1, i].to(DEV)
    q = torch.randn(1, tokens, hq, D, generator=gen).to(BF16)
    out = torch.zeros(1, tokens, hq, D, dtype=BF16, device=DEV)
    gqa.tree_decode(q.to(DEV), k, v, out, num_kv_heads=hkv, layout=gqa.layout_pool(blocks, block, hkv),
                    seq_lens_dev=ints([length]), block_table=ints([used]), workspace=gqa.tree_workspace(1, tokens, hq, hkv, DEV))
    flat = rows.permute(0, 1, 3, 2, 4).reshape(2, 3 * block, hkv, D)[:, :length]
    want, spread, size = TH.attention(q[0], flat[0], flat[1], length - tokens, np.tril(np.ones((tokens, tokens), dtype=bool)))
    assert ((out[0].cpu().double() - want).abs() <= TH.attention_bound(want, spread, size, length, BF16)).all()


# ---- rotary append --------------------------------------------------------------------------------

def rotate(x, weight, pos, freq, factor, style, eps):
    """x [n, heads, 128], pos [n]: the definition in FP64."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    half = freq.shape[0]
    i = torch.arange(half)
    a, c = (i, i + half) if style == "half" else (2 * i, 2 * i + 1)
    theta = pos.double()[:, None, None] * freq
    y = x.clone()
    y[..., a] = factor * (x[..., a] * theta.cos() - x[..., c] * theta.sin())
    y[..., c] = factor * (x[..., a] * theta.sin() + x[..., c] * theta.cos())
    reach = x.abs().clone()  # what the roundings of a rotated channel are relative to
    reach[..., a] = reach[..., c] = factor * (x[..., a].abs() + x[..., c].abs())
    return y, reach


def rotate_bound(y, reach, dtype):
    """sin and cos carry an angle off by half a step of a turn's fraction (2^-25 turns, 2^-22.3 rad) and
    two steps of their own, the norm a sum of 128 squares in a tree and rsqrt (about 12 roundings of 2^-24
    in all), the rotation three: below 2^-20 of the pair's size; then one rounding to the row type."""
    half_step = torch.finfo(dtype).eps / 2
    return half_step * y.abs() + 2.0 ** -20 * (1 + half_step) * reach + 1e-30


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("rotary,scaling,hq,hkv,tokens,lens,sizes,block,stretch", [
    (128, "none", 32, 8, 8, [1000], [8], 0, 0),
    (128, "yarn", 8, 8, 1, [131072], [1], 0, 0),
    (64, "linear", 7, 1, 33, [70, 33, 40], [33, 33, 5], 32, 0),
    (40, "ntk", 10, 2, 5, [5, 200000, 12, 0], [5, 3, 0, 0], 64, 1),
    (8, "none", 64, 8, 16, [500, 17], [16, 16], 96, 1),
])
def test_rope_append(gqa, dtype, style, norm, rotary, scaling, hq, hkv, tokens, lens, sizes, block, stretch):
    rng, gen = np.random.default_rng(rotary + tokens), torch.Generator().manual_seed(rotary + tokens)
    batch, eps = len(lens), 1e-5
    cap = (max(lens) + 95) // 96 * 96
    if max(lens) > 4096:  # far positions: all logical pages but the last share physical ones
        hkv = min(hkv, 2)
        hq = min(hq, 8)
    cache = TH.Cache(gqa, rng, lens, cap if not block else (max(lens) + block - 1) // block * block, hkv, block, dtype)
    k0 = torch.randn(cache.k.shape, generator=gen).to(dtype)
    v0 = torch.randn(cache.v.shape, generator=gen).to(dtype)
    freq, factor = gqa.rope_frequencies(rotary, scaling=scaling, factor=4.0, original_len=8192)
    wide = hq + 2 * hkv + stretch  # rows inside a packed QKV row when stretched
    packed = torch.randn(batch, tokens, wide, D, generator=gen).to(dtype)
    q, kn, vn = packed[:, :, :hq], packed[:, :, hq:hq + hkv], packed[:, :, hq + hkv:hq + 2 * hkv]
    depth = torch.from_numpy(rng.integers(0, max(tokens, 2), (batch, tokens)).astype(np.int32))
    weight = (1 + 0.2 * torch.randn(2 * D, generator=gen)).to(dtype) if norm else None
    k, v, dev = k0.to(DEV), v0.to(DEV), packed.to(DEV)
    dq, dk, dv = dev[:, :, :hq], dev[:, :, hq:hq + hkv], dev[:, :, hq + hkv:hq + 2 * hkv]
    if not stretch:
        dq, dk, dv = dq.contiguous(), dk.contiguous(), dv.contiguous()
    q_out = torch.full((batch, tokens, hq, D), 7.0, dtype=dtype, device=DEV)
    status = ints([0])
    gqa.rope_append(dq, dk, dv, k, v, layout=cache.layout, seq_lens_dev=ints(lens), freq=freq.to(DEV), q_out=q_out,
                    style=style, attn_factor=factor, qk_weight=None if weight is None else weight.to(DEV), eps=eps,
                    depth=depth.to(DEV), tree_sizes=ints(sizes), block_table=cache.table, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    got_q, k, v = q_out.cpu().double(), k.cpu(), v.cpu()
    for b, n in enumerate(sizes):
        assert (got_q[b, n:] == 7.0).all()
        pos = torch.full((n,), lens[b] - n) + depth[b, :n]
        want, reach = rotate(q[b, :n], None if weight is None else weight[:D], pos, freq, factor, style, eps)
        assert ((got_q[b, :n] - want).abs() <= rotate_bound(want, reach, dtype)).all()
        want, reach = rotate(kn[b, :n], None if weight is None else weight[D:], pos, freq, factor, style, eps)
        bound = rotate_bound(want, reach, dtype)
        for t in range(n):
            at = (0,) + cache.at(b, lens[b] - n + t)
            assert ((k[at].double() - want[t]).abs() <= bound[t]).all()
            assert torch.equal(v[at], vn[b, t])
            k0[at], v0[at] = k[at], v[at]
    assert torch.equal(k, k0) and torch.equal(v, v0), "rows of other slots changed"
    # In place, and over the strided rows themselves: the same bits.
    gqa.rope_append(dq, dk, dv, torch.zeros_like(k0).to(DEV), torch.zeros_like(v0).to(DEV), layout=cache.layout, seq_lens_dev=ints(lens),
                    freq=freq.to(DEV), style=style, attn_factor=factor, qk_weight=None if weight is None else weight.to(DEV), eps=eps,
                    depth=depth.to(DEV), tree_sizes=ints(sizes), block_table=cache.table)
    for b, n in enumerate(sizes):
        assert torch.equal(dq[b, :n].cpu().double(), got_q[b, :n])
        assert torch.equal(dq[b, n:].cpu(), q[b, n:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("style", ["half", "interleaved"])
def test_channels_that_are_not_rotated_pass_bit_for_bit(gqa, dtype, style):
    """Infinities, NaN and negative zeros among them touch no other channel."""
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 3, h, D, generator=gen).to(dtype) for h in (5, 3, 3))
    for rows in (q, k):
        rows[..., 64:68] = torch.tensor([float("inf"), -0.0, float("nan"), 1.0], dtype=dtype)
        rows[..., 120], rows[..., 121] = -float("inf"), -0.0
    layout = gqa.layout_reference(1, 32, 3)
    kc, vc = (torch.zeros(32 * 3 * D, dtype=dtype, device=DEV) for _ in range(2))
    out = torch.zeros(1, 3, 5, D, dtype=dtype, device=DEV)
    freq, _ = gqa.rope_frequencies(64, 1e4)
    gqa.rope_append(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, layout=layout, seq_lens_dev=ints([10]), freq=freq.to(DEV),
                    q_out=out, style=style)
    kind = torch.int16 if dtype is BF16 else torch.int32
    keys = kc.cpu().view(32, 3, D)[7:10]
    assert torch.equal(out[0].cpu().view(kind)[..., 64:], q[0].view(kind)[..., 64:])
    assert torch.equal(keys.view(kind)[..., 64:], k[0].view(kind)[..., 64:])
    assert torch.isfinite(out[..., :64]).all() and torch.isfinite(keys[..., :64]).all()


def test_rope_append_agrees_with_the_front_stage(gqa):
    """At near positions, rotate-half over the whole head with QK-Norm is what gqa_qk_norm_rope_append
    computes with FP32 angles: one unit in the last place of BF16."""
    gen = torch.Generator().manual_seed(21)
    hq, hkv, tokens, length = 16, 8, 4, 60
    layout = gqa.layout_reference(1, 64, hkv)
    q, kn, vn = (torch.randn(1, tokens, h, D, generator=gen).to(BF16).to(DEV) for h in (hq, hkv, hkv))
    w = (1 + 0.1 * torch.randn(2 * D, generator=gen)).to(BF16).to(DEV)
    caches = [torch.zeros(64 * hkv * D, dtype=BF16, device=DEV) for _ in range(4)]
    qa, qb = torch.zeros_like(q), torch.zeros_like(q)
    gqa.qk_norm_rope_append(q, kn, vn, w, caches[0], caches[1], layout=layout, positions=[length - tokens], q_out=qa)
    freq, factor = gqa.rope_frequencies(128)
    gqa.rope_append(q, kn, vn, caches[2], caches[3], layout=layout, seq_lens_dev=ints([length]), freq=freq.to(DEV),
                    q_out=qb, attn_factor=factor, qk_weight=w)
    assert torch.equal(caches[1], caches[3])
    for a, b in ((qa, qb), (caches[0], caches[2])):
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * a.float().abs() + 1e-5).all()


@pytest.mark.parametrize("lens,sizes", [([200], [4]), ([3], [4]), ([20], [5])])
def test_rope_append_skips_and_reports_bad_lengths(gqa, lens, sizes):
    layout = gqa.layout_reference(1, 64, 2)
    rows = torch.ones(1, 4, 2, D, dtype=BF16, device=DEV)
    k, v = (torch.zeros(64 * 2 * D, dtype=BF16, device=DEV) for _ in range(2))
    q_out, status = torch.zeros_like(rows), ints([0])
    freq, _ = gqa.rope_frequencies(128)
    gqa.rope_append(rows, rows, rows, k, v, layout=layout, seq_lens_dev=ints(lens), freq=freq.to(DEV), q_out=q_out,
                    tree_sizes=ints(sizes), status=status)
    assert int(status) == 3 and not k.any() and not v.any() and not q_out.any()


def test_rope_append_leaves_rows_without_a_block(gqa):
    layout = gqa.layout_pool(4, 32, 2)
    rows = torch.ones(1, 4, 2, D, dtype=BF16, device=DEV)
    k, v = (torch.zeros(4, 2, 32, D, dtype=BF16, device=DEV) for _ in range(2))
    status = ints([0])
    freq, _ = gqa.rope_frequencies(128)
    gqa.rope_append(rows, rows.clone(), rows.clone(), k, v, layout=layout, seq_lens_dev=ints([34]), freq=freq.to(DEV),
                    q_out=torch.zeros_like(rows), block_table=ints([[2, -1]]), status=status)
    assert int(status) == 3
    assert v[2, :, 30:].all() and v.float().sum() == 2 * 2 * D  # slots 30 and 31 only


# ---- verification ---------------------------------------------------------------------------------

def probabilities(gen, shape, dtype, sharp=2.0):
    return torch.softmax(sharp * torch.randn(shape, generator=gen), -1).to(dtype)


def run_verify(gqa, target, draft, tokens, parents, u, us, sizes, status=None):
    batch, nodes = tokens.shape
    path, kept, nxt = ints([[9] * nodes] * batch), ints([9] * batch), ints([9] * batch)
    gqa.tree_verify(target, draft, tokens.to(DEV), parents.to(DEV), u.to(DEV), us.to(DEV), path=path, kept=kept,
                    next_token=nxt, tree_sizes=ints(sizes), status=status)
    return path.cpu().tolist(), kept.cpu().tolist(), nxt.cpu().tolist()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("vocab,nodes,batch,shape", [
    (1, 4, 3, "tree"), (2, 9, 8, "tree"), (17, 128, 6, "tree"), (1000, 16, 9, "chain"), (4099, 33, 7, "tree"), (32000, 5, 4, "bush"),
    (50001, 64, 3, "bush")])
def test_verify(gqa, dtype, with_draft, vocab, nodes, batch, shape):
    seed = vocab + nodes
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    target = probabilities(gen, (batch, nodes, vocab), dtype)
    draft = probabilities(gen, (batch, nodes, vocab), dtype) if with_draft else None
    width = {"chain": 1, "tree": 4, "bush": nodes}[shape]
    parents = torch.tensor([TH.random_parents(rng, nodes, width) for _ in range(batch)], dtype=torch.int32)
    # Tokens at the rows' heavy ends, so that both outcomes occur; some siblings carry the same token.
    tokens = torch.zeros(batch, nodes, dtype=torch.int32)
    for b in range(batch):
        for t in range(1, nodes):
            row = (draft if draft is not None else target)[b, parents[b, t]].float()
            tokens[b, t] = int(torch.multinomial(row, 1, generator=gen))
    u, us = torch.rand(batch, nodes, generator=gen), torch.rand(batch, generator=gen)
    sizes = [int(rng.integers(1, nodes + 1)) for _ in range(batch)]
    sizes[0], sizes[-1] = nodes, 0 if batch > 1 else nodes
    got = run_verify(gqa, target.to(DEV), None if draft is None else draft.to(DEV), tokens, parents, u, us, sizes)
    for b in range(batch):
        path, nxt = TH.verify(target[b], None if draft is None else draft[b], tokens[b].tolist(), parents[b].tolist(),
                              sizes[b], u[b].double().tolist(), float(us[b].double()))
        assert got[0][b] == path + [-1] * (nodes - len(path)), b
        assert got[1][b] == len(path) and got[2][b] == nxt, b


def test_verify_reads_rows_with_strides_and_odd_alignment(gqa):
    rng, gen = np.random.default_rng(3), torch.Generator().manual_seed(3)
    batch, nodes, vocab = 3, 6, 999
    for dtype in (F32, BF16):
        for off_p, off_q in ((0, 0), (1, 1), (1, 2), (3, 0)):
            wide_p = probabilities(gen, (batch, nodes + 1, 1024), dtype).to(DEV)
            wide_q = probabilities(gen, (batch, nodes + 2, 1011), dtype).to(DEV)
            target, draft = wide_p[:, :nodes, off_p:off_p + vocab], wide_q[:, 1:nodes + 1, off_q:off_q + vocab]
            parents = torch.tensor([TH.random_parents(rng, nodes) for _ in range(batch)], dtype=torch.int32)
            tokens = torch.from_numpy(rng.integers(0, vocab, (batch, nodes)).astype(np.int32))
            u, us = torch.rand(batch, nodes, generator=gen), torch.rand(batch, generator=gen)
            got = run_verify(gqa, target, draft, tokens, parents, u, us, [nodes] * batch)
            for b in range(batch):
                path, nxt = TH.verify(target[b].cpu(), draft[b].cpu(), tokens[b].tolist(), parents[b].tolist(), nodes,
                                      u[b].double().tolist(), float(us[b].double()))
                assert got[0][b][: len(path)] == path and got[1][b] == len(path) and got[2][b] == nxt


def test_verify_edges(gqa):
    """One node a sequence but for the last four: random numbers at their ends, rows that are zero, hold NaN,
    negative numbers or infinities; residuals that are empty; rows of unvisited nodes full of NaN."""
    vocab, nan, inf = 70, float("nan"), float("inf")
    rows = torch.zeros(12, 3, vocab)
    rows[:, :, 5], rows[:, :, 60] = 0.25, 0.75
    rows[2, 0] = 0.0                                    # nothing to sample
    rows[3, 0, :4], rows[3, 0, 61:] = nan, -1.0         # NaN and negative entries count as 0
    rows[4, 0, 10] = inf
    draft = rows.clone()
    tokens = torch.full((12, 3), 5, dtype=torch.int32)
    parents = torch.tensor([[-1, 0, 0]] * 12, dtype=torch.int32)
    u = torch.zeros(12, 3)
    us = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.5, 0.3, 0.5, nan, 1.0, 0.5, 0.2, 0.9, 0.5, 0.5])
    sizes = [1] * 7 + [3, 3, 3, 3, 0]
    # 7: p = q and u at its upper end: always accepted. 8: the token has no probability: rejected twice; with
    # p = q nothing is left, p itself is sampled. 9: q = 0 at the token and p > 0: accepted. 10: bad tokens.
    u[7] = 1.0 - 2.0 ** -24
    rows[7, 2] = nan  # never visited
    tokens[8] = 6
    tokens[9], draft[9, :, 5] = 5, 0.0
    tokens[10, 1], tokens[10, 2] = -1, vocab
    status = ints([0])
    got = run_verify(gqa, rows.to(DEV), draft.to(DEV), tokens, parents, u, us, sizes, status)
    assert int(status) == 3  # the row of zeros and the bad tokens
    assert got[2][:4] == [5, 60, -1, 60]
    assert got[2][4] in (10, 60)  # an infinite entry: any entry that is not 0
    assert got[2][5] == 60 and got[2][6] == 60  # a threshold that nothing passes: the last one
    assert got[1] == [1] * 7 + [2, 1, 2, 1, 0]
    assert got[0][7] == [0, 1, -1] and got[0][9] == [0, 1, -1] and got[0][11] == [-1, -1, -1]
    assert got[2][8] == 5 and got[2][10] == 60 and got[2][11] == -1


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_of_many_sequences_over_a_large_vocabulary(gqa, with_draft):
    """So many sequences that each gets one block, and more rounds of a warp's segment than are kept
    (64 of 32 vectors): samples among the first rounds, the last ones, and a threshold nothing passes."""
    gen = torch.Generator().manual_seed(12)
    batch, nodes, vocab = 150, 2, 140001
    target = torch.softmax(2.0 * torch.randn(batch, nodes, vocab, generator=gen), -1)
    draft = torch.softmax(2.0 * torch.randn(batch, nodes, vocab, generator=gen), -1) if with_draft else None
    parents = torch.tensor([[-1, 0]] * batch, dtype=torch.int32)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=gen).int()
    u, us = torch.rand(batch, nodes, generator=gen), torch.rand(batch, generator=gen)
    us[0], us[1], us[2] = 0.0, 1.0 - 2.0 ** -24, 1.0
    got = run_verify(gqa, target.to(DEV), None if draft is None else draft.to(DEV), tokens, parents, u, us, [nodes] * batch)
    for b in range(batch):
        path, nxt = TH.verify(target[b], None if draft is None else draft[b], tokens[b].tolist(), parents[b].tolist(), nodes,
                              u[b].double().tolist(), float(us[b].double()))
        assert got[0][b][: len(path)] == path and got[1][b] == len(path) and got[2][b] == nxt, b


def test_verify_emits_tokens_as_the_target_would(gqa):
    """The first token behind the root, accepted or sampled, over many seeded draws of two drafts from the
    draft's row: its frequencies are the target's, to five standard deviations of a count."""
    gen = torch.Generator().manual_seed(77)
    batch, vocab = 40000, 6
    p = torch.tensor([0.4, 0.05, 0.25, 0.1, 0.2, 0.0])
    q = torch.tensor([0.1, 0.3, 0.2, 0.2, 0.1, 0.1])
    target = torch.zeros(batch, 3, vocab)
    target[:] = p
    draft = torch.zeros(batch, 3, vocab)
    draft[:] = q
    tokens = torch.multinomial(q.expand(batch, vocab), 3, replacement=True, generator=gen).int()
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32).expand(batch, 3).contiguous()
    u, us = torch.rand(batch, 3, generator=gen), torch.rand(batch, generator=gen)
    path, kept, nxt = run_verify(gqa, target.to(DEV), draft.to(DEV), tokens, parents, u, us, [3] * batch)
    first = np.array([tokens[b, path[b][1]] if kept[b] > 1 else nxt[b] for b in range(batch)])
    count = np.bincount(first, minlength=vocab)
    assert count[5] == 0
    for x in range(5):
        mean = batch * float(p[x])
        assert abs(count[x] - mean) <= 5 * math.sqrt(mean * (1 - float(p[x]))), (x, count[x], mean)


# ---- commit -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layers,hkv,tokens,lens,sizes,block", [
    (1, 8, 1, [1], [1], 0), (3, 8, 8, [40], [8], 0), (2, 1, 128, [200], [128], 0),
    (4, 2, 16, [70, 33, 16, 20, 64], [16, 16, 16, 4, 0], 32), (36, 8, 33, [100, 64], [33, 30], 96)])
def test_commit(gqa, dtype, layers, hkv, tokens, lens, sizes, block):
    rng, gen = np.random.default_rng(tokens), torch.Generator().manual_seed(tokens)
    cache = TH.Cache(gqa, rng, lens, max(lens) if block else max(lens) + 3, hkv, block, dtype, layers)
    k0, v0 = (torch.randn(cache.k.shape, generator=gen).to(dtype) for _ in range(2))
    path = np.full((len(lens), tokens), -1, dtype=np.int32)
    kept = []
    for b, n in enumerate(sizes):
        m = int(rng.integers(1, n + 1)) if n else 0
        rest = 1 + np.sort(rng.permutation(max(n - 1, 0))[: max(m - 1, 0)])
        path[b, :m] = np.concatenate([[0], rest])[:m]
        kept.append(m)
    k, v, new, status = k0.to(DEV), v0.to(DEV), ints([-5] * len(lens)), ints([0])
    gqa.tree_commit(k, v, num_kv_heads=hkv, layout=cache.layout, layers=layers, seq_lens_dev=ints(lens), seq_lens_out=new,
                    path=torch.from_numpy(path).to(DEV), kept=ints(kept), tree_sizes=ints(sizes), block_table=cache.table, status=status)
    assert int(status) == 0
    wk, wv = k0.clone(), v0.clone()
    for b, n in enumerate(sizes):
        base = lens[b] - n
        for i in range(kept[b]):
            src, dst = (slice(None),) + cache.at(b, base + int(path[b, i])), (slice(None),) + cache.at(b, base + i)
            wk[dst], wv[dst] = k0[src], v0[src]
        assert int(new[b]) == base + kept[b]
    assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)


@pytest.mark.parametrize("path,kept", [([0, 2, 1, -1], 3), ([0, 1, 1, -1], 3), ([0, 4, -1, -1], 2), ([-1, 0, 1, 2], 2),
                                       ([0, 1, 2, 3], 5), ([0, 1, 2, 3], -1)])
def test_commit_skips_and_reports_paths_that_do_not_ascend(gqa, path, kept):
    gen = torch.Generator().manual_seed(1)
    layout = gqa.layout_reference(1, 32, 2)
    k = torch.randn(32 * 2 * D, generator=gen).to(BF16).to(DEV)
    before, new, status = k.clone(), ints([0]), ints([0])
    gqa.tree_commit(k, k.clone(), num_kv_heads=2, layout=layout, seq_lens_dev=ints([20]), path=ints([path]), kept=ints([kept]),
                    seq_lens_out=new, status=status)
    assert int(status) == 3 and torch.equal(k, before) and int(new) == 20


# ---- the four in a row --------------------------------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
def test_decode_loop(gqa, captured):
    """Three steps of a tree-drafted loop over a two-layer model of nothing but attention. After each step
    the caches hold what appending the accepted tokens one by one leaves, and the nodes on the path got
    the attention output that single-token decoding computes for them."""
    rng, gen = np.random.default_rng(31), torch.Generator().manual_seed(31)
    hq, hkv, tokens, batch, block, layers, vocab = 16, 4, 12, 3, 64, 2, 50
    pool = gqa.KvPool(64, block, hkv, batch, 8)
    layout = pool.layout()
    history = [70, 31, 5]
    for b in range(batch):
        pool.reserve(b, history[b] + 3 * tokens)
    table = pool.table().to(DEV)
    k = torch.zeros(layers, 64, hkv, block, D, dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    freq, factor = gqa.rope_frequencies(96, scaling="yarn", factor=2.0, original_len=64)
    freq = freq.to(DEV)
    w = (1 + 0.1 * torch.randn(2 * D, generator=gen)).to(BF16).to(DEV)

    def rows(n, heads):
        return torch.randn(batch, n, heads, D, generator=gen).to(BF16).to(DEV)

    # The history: appended through the same entry point, at consecutive positions.
    for layer in range(layers):
        qh, kh, vh = rows(70, hq), rows(70, hkv), rows(70, hkv)
        gqa.rope_append(qh, kh, vh, k[layer], v[layer], layout=layout, seq_lens_dev=ints(history), freq=freq, attn_factor=factor,
                        qk_weight=w, tree_sizes=ints(history), block_table=table)
    plain_k, plain_v = k.clone(), v.clone()
    lens, new_lens = ints([0] * batch), ints([0] * batch)
    sizes, mask = ints([0] * batch), ints([[[0]] * tokens] * batch)
    depth, par = ints([[0] * tokens] * batch), ints([[0] * tokens] * batch)
    q, kn, vn = ([torch.zeros(batch, tokens, h, D, dtype=BF16, device=DEV) for _ in range(layers)] for h in (hq, hkv, hkv))
    q_rot = [torch.zeros_like(q[0]) for _ in range(layers)]
    out = [torch.zeros_like(q[0]) for _ in range(layers)]
    target, draft = (torch.zeros(batch, tokens, vocab, device=DEV) for _ in range(2))
    words, path = ints([[0] * tokens] * batch), ints([[0] * tokens] * batch)
    kept, nxt, status = ints([0] * batch), ints([0] * batch), ints([0])
    u, us = torch.zeros(batch, tokens, device=DEV), torch.zeros(batch, device=DEV)
    ws = gqa.tree_workspace(batch, tokens, hq, hkv, DEV)

    def step():
        for layer in range(layers):
            gqa.rope_append(q[layer], kn[layer], vn[layer], k[layer], v[layer], layout=layout, seq_lens_dev=lens, freq=freq,
                            q_out=q_rot[layer], attn_factor=factor, qk_weight=w, depth=depth, tree_sizes=sizes, block_table=table,
                            status=status)
            gqa.tree_decode(q_rot[layer], k[layer], v[layer], out[layer], num_kv_heads=hkv, layout=layout, seq_lens_dev=lens,
                            mask=mask, tree_sizes=sizes, block_table=table, workspace=ws, status=status)
        gqa.tree_verify(target, draft, words, par, u, us, path=path, kept=kept, next_token=nxt, tree_sizes=sizes, status=status)
        gqa.tree_commit(k, v, num_kv_heads=hkv, layout=layout, layers=layers, seq_lens_dev=lens, path=path, kept=kept,
                        seq_lens_out=new_lens, tree_sizes=sizes, block_table=table, status=status)

    graph = None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()  # sizes are 0: nothing is done
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    for turn in range(3):
        n = [int(rng.integers(6, tokens + 1)) for _ in range(batch)]
        trees = [TH.random_parents(rng, tokens, 3) for _ in range(batch)]
        m, d = gqa.tree_masks(torch.tensor(trees), torch.tensor(n))
        sizes.copy_(ints(n)); mask.copy_(m); depth.copy_(d); par.copy_(ints(trees))
        lens.copy_(ints([history[b] + n[b] for b in range(batch)]))
        for layer in range(layers):
            q[layer].copy_(rows(tokens, hq)); kn[layer].copy_(rows(tokens, hkv)); vn[layer].copy_(rows(tokens, hkv))
        target.copy_(probabilities(gen, (batch, tokens, vocab), F32, 1.0))
        draft.copy_(target)
        draft.mul_(0.9).add_(0.1 / vocab)  # near the target: long paths
        words.copy_(torch.randint(0, vocab, (batch, tokens), generator=gen).int())
        u.copy_(torch.rand(batch, tokens, generator=gen)); us.copy_(torch.rand(batch, generator=gen))
        if captured:
            graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        assert int(status) == 0
        for b in range(batch):
            want, token = TH.verify(target[b].cpu(), draft[b].cpu(), words[b].tolist(), trees[b], n[b],
                                    u[b].double().cpu().tolist(), float(us[b].double()))
            assert path[b, : len(want)].tolist() == want and int(kept[b]) == len(want) and int(nxt[b]) == token
            # The accepted tokens one by one, at consecutive slots.
            for i, node in enumerate(want):
                one = ints([history[b] + i + 1])
                for layer in range(layers):
                    qo = torch.zeros(1, 1, hq, D, dtype=BF16, device=DEV)
                    gqa.rope_append(q[layer][b:b + 1, node:node + 1], kn[layer][b:b + 1, node:node + 1], vn[layer][b:b + 1, node:node + 1],
                                    plain_k[layer], plain_v[layer], layout=layout, seq_lens_dev=one, freq=freq, q_out=qo,
                                    attn_factor=factor, qk_weight=w, block_table=table[b:b + 1].contiguous())
                    assert torch.equal(qo[0, 0], q_rot[layer][b, node])
                    single = torch.zeros(1, hq, D, dtype=BF16, device=DEV)
                    gqa.decode(qo[:, 0], plain_k[layer], plain_v[layer], single, num_kv_heads=hkv, layout=layout,
                               seq_lens=[history[b] + i + 1], seq_lens_dev=one, block_table=table[b:b + 1].contiguous(),
                               workspace=gqa.binding.workspace_for(1, hq, hkv, DEV))
                    # Both carry two roundings of 2^-8 (weights, output) of values whose weighted mean size is below 4.
                    assert ((single[0].float() - out[layer][b, node].float()).abs() <= 4 * 2.0 ** -8 * 4).all()
            history[b] += len(want)
            assert int(new_lens[b]) == history[b]
            for layer in range(layers):
                for p in range(history[b]):
                    blk, at = int(table[b, p // block]), p % block
                    assert torch.equal(k[layer, blk, :, at], plain_k[layer, blk, :, at])
                    assert torch.equal(v[layer, blk, :, at], plain_v[layer, blk, :, at])


def test_draft_tree_runs_the_four_calls(gqa):
    """DraftTree is the four calls on buffers of its own: the same bits, and the next plan starts from
    the lengths the last commit left."""
    gen = torch.Generator().manual_seed(41)
    hq, hkv, tokens, batch, vocab = 16, 4, 10, 2, 40
    layout = gqa.layout_pool(8, 64, hkv)
    table = ints([[0, 1, 2, 3], [4, 5, 6, 7]])
    freq, factor = gqa.rope_frequencies(128)
    freq = freq.to(DEV)
    trees = torch.tensor([[-1, 0, 0, 1, 1, 2, 3, 3, 4, 5], [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8]])
    sizes, history = torch.tensor([10, 7]), torch.tensor([60, 100])
    start = [torch.randn(8, hkv, 64, D, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    tree = gqa.DraftTree(batch, tokens, hq, hkv, DEV)
    plain = [c.clone() for c in start]
    own = [c.clone() for c in start]
    for turn in range(2):
        q, kn, vn = (torch.randn(batch, tokens, h, D, generator=gen).to(BF16).to(DEV) for h in (hq, hkv, hkv))
        target = probabilities(gen, (batch, tokens, vocab), F32, 1.0).to(DEV)
        draft = (0.9 * target + 0.1 / vocab)
        words = torch.randint(0, vocab, (batch, tokens), generator=gen).int().to(DEV)
        u, us = torch.rand(batch, tokens, generator=gen).to(DEV), torch.rand(batch, generator=gen).to(DEV)
        tree.plan(trees, sizes, history if turn == 0 else None)
        rot, out = torch.zeros_like(q), torch.zeros_like(q)
        tree.append(q, kn, vn, own[0], own[1], layout=layout, freq=freq, attn_factor=factor, q_out=rot, block_table=table)
        tree.attend(rot, own[0], own[1], out, layout=layout, block_table=table)
        tree.verify(target, draft, words, u, us)
        tree.commit(own[0], own[1], layout=layout, block_table=table)
        lens = ints([int(h) + int(s) for h, s in zip(history, sizes)])
        mask, depth = gqa.tree_masks(trees, sizes)
        rot2, out2 = torch.zeros_like(q), torch.zeros_like(q)
        ws = gqa.tree_workspace(batch, tokens, hq, hkv, DEV)
        gqa.rope_append(q, kn, vn, plain[0], plain[1], layout=layout, seq_lens_dev=lens, freq=freq, attn_factor=factor, q_out=rot2,
                        depth=depth.to(DEV), tree_sizes=ints(sizes.tolist()), block_table=table)
        gqa.tree_decode(rot2, plain[0], plain[1], out2, num_kv_heads=hkv, layout=layout, seq_lens_dev=lens, mask=mask.to(DEV),
                        tree_sizes=ints(sizes.tolist()), block_table=table, workspace=ws)
        path, kept, nxt, new = ints([[0] * tokens] * batch), ints([0] * batch), ints([0] * batch), ints([0] * batch)
        gqa.tree_verify(target, draft, words, trees.int().to(DEV), u, us, path=path, kept=kept, next_token=nxt, tree_sizes=ints(sizes.tolist()))
        gqa.tree_commit(plain[0], plain[1], num_kv_heads=hkv, layout=layout, seq_lens_dev=lens, path=path, kept=kept, seq_lens_out=new,
                        tree_sizes=ints(sizes.tolist()), block_table=table)
        assert int(tree.status) == 0
        for a, b in ((rot, rot2), (out, out2), (own[0], plain[0]), (own[1], plain[1]), (tree.path, path), (tree.kept, kept),
                     (tree.next_token, nxt), (tree.history, new)):
            assert torch.equal(a, b)
        history = new.cpu()
    with pytest.raises(ValueError, match="parents"):
        tree.plan(trees[:, :5])

"""Tree drafting on the GPU over caches that lie otherwise than one pool or one block: K and V side by side, blocks
of odd lengths behind a table, as many sequences as a call takes, FP32 queries inside packed rows."""
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


def check(got, q, k, v, lens, sizes, sees, dtype):
    """Every element of got [batch, tokens, hq, 128] against the definition; k, v: lists of [len, hkv, 128]."""
    for b, n in enumerate(sizes):
        want, spread, size = TH.attention(q[b, :n], k[b], v[b], lens[b] - n, sees[b])
        bound = TH.attention_bound(want, spread, size, lens[b], dtype)
        off = (got[b, :n].cpu().double() - want).abs()
        assert (off <= bound).all(), (b, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_k_and_v_side_by_side(gqa, dtype):
    """[block][K or V][head][token][channel], all four calls: the same bits as in caches of their own."""
    gen = torch.Generator().manual_seed(1)
    hq, hkv, tokens, block, blocks, layers = 8, 2, 9, 32, 9, 3
    lens, table = [70, 130], ints([[0, 7, 2, 8, -1], [1, 3, 4, 5, 6]])
    both = torch.randn(layers, blocks, 2, hkv, block, D, generator=gen).to(dtype).to(DEV)
    apart = [both[:, :, i].clone() for i in range(2)]
    pool = gqa.layout_pool(blocks, block, hkv)
    wide = gqa.KvLayout(block, blocks, 2 * pool.stride_block, pool.stride_token, pool.stride_head)
    q, kn, vn = (torch.randn(2, tokens, h, D, generator=gen).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    freq, _ = gqa.rope_frequencies(128)
    freq, ws = freq.to(DEV), gqa.tree_workspace(2, tokens, hq, hkv, DEV, dtype)
    results = []
    for k, v, layout in ((both[:, :, 0], both[:, :, 1], wide), (*apart, pool)):
        rot, out, new = torch.zeros_like(q), torch.zeros_like(q), ints([0, 0])
        kw = dict(layout=layout, seq_lens_dev=ints(lens), block_table=table)
        gqa.rope_append(q, kn, vn, k[1], v[1], freq=freq, q_out=rot, **kw)
        gqa.tree_decode(rot, k[1], v[1], out, num_kv_heads=hkv, workspace=ws, **kw)
        gqa.tree_commit(k, v, num_kv_heads=hkv, layers=layers, layer_stride=blocks * layout.stride_block, path=ints([[0, 3, 8] + [-1] * 6] * 2),
                        kept=ints([3, 3]), seq_lens_out=new, **kw)
        results.append((rot, out, new, k.clone(), v.clone()))
    assert results[0][1].abs().sum() > 0
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("length", [1, 100, 129, 333])
def test_one_block_of_any_length_for_each_sequence(gqa, dtype, length):
    """A table of one block per sequence: the block need not be whole chunks or tiles of keys."""
    gen, rng = torch.Generator().manual_seed(length), np.random.default_rng(length)
    hq, hkv, tokens = 12, 2, min(7, length)
    layout, blocks = gqa.layout_reference(3, length, hkv), [2, 0]
    k, v = (torch.full((3, length, hkv, D), float("nan"), dtype=dtype) for _ in range(2))
    lens = [length, max(tokens, length // 2)]
    for b in range(2):
        k[blocks[b], :lens[b]] = torch.randn(lens[b], hkv, D, generator=gen).to(dtype)
        v[blocks[b], :lens[b]] = torch.randn(lens[b], hkv, D, generator=gen).to(dtype)
    sees = [TH.ancestors(TH.random_parents(rng, tokens)) for _ in range(2)]
    q = torch.randn(2, tokens, hq, D, generator=gen).to(dtype)
    out, status = torch.zeros(2, tokens, hq, D, dtype=dtype, device=DEV), ints([0])
    gqa.tree_decode(q.to(DEV), k.to(DEV), v.to(DEV), out, num_kv_heads=hkv, layout=layout, seq_lens_dev=ints(lens), mask=TH.pack_mask(sees, tokens).to(DEV),
                    block_table=ints([[b] for b in blocks]), workspace=gqa.tree_workspace(2, tokens, hq, hkv, DEV, dtype), status=status)
    assert int(status) == 0
    check(out, q, [k[blocks[b], :lens[b]] for b in range(2)], [v[blocks[b], :lens[b]] for b in range(2)], lens, [tokens] * 2, sees, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_as_many_sequences_as_a_call_takes(gqa, dtype):
    gen, rng = torch.Generator().manual_seed(2), np.random.default_rng(2)
    batch, hq, hkv, tokens, block = 1024, 4, 1, 3, 32
    sizes = [int(n) for n in rng.integers(0, tokens + 1, batch)]
    lens = [n + int(rng.integers(0, 2 * block - tokens + 1)) for n in sizes]
    table = rng.permutation(2 * batch).reshape(batch, 2)
    k, v = (torch.randn(2 * batch, hkv, block, D, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(batch, tokens, hq, D, generator=gen).to(dtype)
    out, status = torch.full((batch, tokens, hq, D), 7.0, dtype=dtype, device=DEV), ints([0])
    gqa.tree_decode(q.to(DEV), k.to(DEV), v.to(DEV), out, num_kv_heads=hkv, layout=gqa.layout_pool(2 * batch, block, hkv), seq_lens_dev=ints(lens),
                    tree_sizes=ints(sizes), block_table=ints(table.tolist()), workspace=gqa.tree_workspace(batch, tokens, hq, hkv, DEV, dtype), status=status)
    assert int(status) == 0
    rows = lambda c, b: c[torch.from_numpy(table[b])].permute(0, 2, 1, 3).reshape(2 * block, hkv, D)[: lens[b]]
    check(out, q, [rows(k, b) for b in range(batch)], [rows(v, b) for b in range(batch)], lens, sizes, [np.tril(np.ones((n, n), dtype=bool)) for n in sizes], dtype)
    got = out.cpu()
    assert all((got[b, n:] == 7.0).all() for b, n in enumerate(sizes))


def test_fp32_queries_inside_packed_rows(gqa):
    gen = torch.Generator().manual_seed(4)
    hq, hkv, tokens, lens = 16, 4, 6, [90, 200]
    layout, table = gqa.layout_pool(8, 64, hkv), ints([[0, 3, 5, 6], [7, 1, 2, 4]])
    k, v = (torch.randn(8, hkv, 64, D, generator=gen).to(DEV) for _ in range(2))
    packed = torch.randn(2, tokens, hq + 2 * hkv, D, generator=gen).to(DEV)
    ws = gqa.tree_workspace(2, tokens, hq, hkv, DEV, F32)
    outs = []
    for q in (packed[:, :, :hq], packed[:, :, :hq].contiguous()):
        outs.append(torch.zeros(2, tokens, hq, D, device=DEV))
        gqa.tree_decode(q, k, v, outs[-1], num_kv_heads=hkv, layout=layout, seq_lens_dev=ints(lens), block_table=table, workspace=ws)
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().sum() > 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_between_rows(gqa, dtype):
    """Queries and outputs that lie in one buffer without sharing an element: the same bits as apart."""
    gen = torch.Generator().manual_seed(8)
    hq, hkv, tokens = 4, 2, 6
    rows = torch.randn(2, tokens, 3 * hq, D, generator=gen).to(dtype).to(DEV)
    q, q_out = rows[:, :, :hq], rows[:, :, 2 * hq:]
    before = rows.clone()
    kn, vn = (torch.randn(2, tokens, hkv, D, generator=gen).to(dtype).to(DEV) for _ in range(2))
    k, v = (torch.zeros(4, hkv, 32, D, dtype=dtype, device=DEV) for _ in range(2))
    freq, _ = gqa.rope_frequencies(128)
    kw = dict(layout=gqa.layout_pool(4, 32, hkv), seq_lens_dev=ints([40, 20]), freq=freq.to(DEV), block_table=ints([[0, 1], [2, 3]]))
    apart = torch.zeros(2, tokens, hq, D, dtype=dtype, device=DEV)
    gqa.rope_append(q.contiguous(), kn, vn, k, v, q_out=apart, **kw)
    gqa.rope_append(q, kn, vn, k, v, q_out=q_out, **kw)
    assert torch.equal(q_out, apart) and torch.equal(rows[:, :, : 2 * hq], before[:, :, : 2 * hq]) and apart.abs().sum() > 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("entry", [-1, 4, 1 << 30])
def test_positions_without_a_block_are_rows_of_zeros(gqa, dtype, entry):
    gen = torch.Generator().manual_seed(9)
    hq, hkv, tokens, length = 8, 2, 5, 110
    k, v = (torch.randn(4, hkv, 32, D, generator=gen).to(dtype) for _ in range(2))
    q, status = torch.randn(1, tokens, hq, D, generator=gen).to(dtype), ints([0])
    out = torch.zeros(1, tokens, hq, D, dtype=dtype, device=DEV)
    gqa.tree_decode(q.to(DEV), k.to(DEV), v.to(DEV), out, num_kv_heads=hkv, layout=gqa.layout_pool(4, 32, hkv), seq_lens_dev=ints([length]),
                    block_table=ints([[3, entry, 0, 1]]), workspace=gqa.tree_workspace(1, tokens, hq, hkv, DEV, dtype), status=status)
    assert int(status) == 3
    rows = lambda c: torch.cat([c[3], torch.zeros_like(c[0]), c[0], c[1]], 1).transpose(0, 1)[:length]
    check(out, q, [rows(k)], [rows(v)], [length], [tokens], [np.tril(np.ones((tokens, tokens), dtype=bool))], dtype)


@pytest.mark.parametrize("tokens", [8, 40])
def test_launches_back_to_back(gqa, tokens):
    """Blocks follow one another on an SM without a pause: each leaves only when all that was to arrive in its memory has."""
    gen = torch.Generator().manual_seed(tokens)
    hq, hkv, batch = 32, 8, 3
    k, v = (torch.randn(batch, 700, hkv, D, generator=gen).to(BF16).to(DEV) for _ in range(2))
    q = torch.randn(batch, tokens, hq, D, generator=gen).to(BF16).to(DEV)
    layout, table, ws = gqa.layout_reference(batch, 700, hkv), ints([[0], [1], [2]]), gqa.tree_workspace(batch, tokens, hq, hkv, DEV)
    lens = [ints([tokens, 129, 700]), ints([128, tokens + 1, 300]), ints([650, 513, 40])]

    def call(out, n):
        gqa.tree_decode(q, k, v, out, num_kv_heads=hkv, layout=layout, seq_lens_dev=lens[n], block_table=table, workspace=ws)

    want = [torch.zeros_like(q) for _ in lens]
    for i, w in enumerate(want):
        call(w, i)
        torch.cuda.synchronize()
    got = [torch.zeros_like(q) for _ in range(90)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i, g in enumerate(got):
            call(g, i % 3)
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        for i, g in enumerate(got):
            assert torch.equal(g, want[i % 3]), i

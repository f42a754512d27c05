"""Tree drafting on the GPU, what lies between the four calls: plans from buffers that the caller goes on to
use, commits that are refused."""
import pytest
import torch

from tree_helpers import D, DEV

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
PARENTS = torch.tensor([[-1, 0, 0, 1, 1, 2]] * 2)


@pytest.fixture(scope="module")
def gqa(built_lib):
    import llminfer_b200 as pkg
    return pkg


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_plan_is_done_with_its_inputs_when_it_returns(gqa, kind):
    """A serving loop refills its pinned buffers for the next step while the stream is still busy."""
    tree = gqa.DraftTree(2, 6, 8, 2, DEV)
    parents, sizes, history = (t.to(kind).pin_memory() for t in (PARENTS, torch.tensor([6, 4]), torch.tensor([20, 30])))
    tree.plan(PARENTS)  # what a first call loads keeps it waiting for the stream
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # the stream is at work for some 50 ms
    tree.plan(parents, sizes, history)
    for t in (parents, sizes, history):
        t.zero_()
    torch.cuda.synchronize()
    mask, depth = gqa.tree_masks(PARENTS, torch.tensor([6, 4]))
    assert torch.equal(tree.parents.cpu(), PARENTS.int()) and tree.sizes.tolist() == [6, 4]
    assert tree.history.tolist() == [20, 30] and tree.lens.tolist() == [26, 34]
    assert torch.equal(tree.mask.cpu(), mask) and torch.equal(tree.depth.cpu(), depth)


@pytest.mark.parametrize("history,path,kept,missing", [
    (40, [0, 3, 2, -1, -1, -1], 3, False),   # does not ascend
    (40, [0, 1, 2, 3, 5, 4], 6, False),      # as many as there are, out of order
    (40, [0, 1, 2, 3, 4, 5], 7, False),      # more than there are
    (40, [0, 1, 2, 3, 4, 5], -1, False),
    (40, [0, 2, -1, -1, -1, -1], 2, True),   # the slots have no block
    (62, [0, 2, -1, -1, -1, -1], 2, False),  # the tree reaches beyond the sequence's blocks
])
def test_a_refused_commit_leaves_the_history(gqa, history, path, kept, missing):
    """Nodes that nobody accepted do not become history: the next plan starts where this one did."""
    gen = torch.Generator().manual_seed(5)
    layout = gqa.layout_pool(4, 32, 2)
    k, v = (torch.randn(4, 2, 32, D, generator=gen).to(BF16).to(DEV) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    tree = gqa.DraftTree(2, 6, 8, 2, DEV)
    tree.plan(PARENTS, None, torch.tensor([20, history]))
    tree.path.copy_(ints([[0, 2, 5, -1, -1, -1], path]))
    tree.kept.copy_(ints([3, kept]))
    tree.commit(k, v, layout=layout, block_table=ints([[0, 1], [2, -1 if missing else 3]]))
    assert int(tree.status) == 3
    assert tree.history.tolist() == [23, history]
    for c, c0 in ((k, k0), (v, v0)):
        for i, node in enumerate([0, 2, 5]):
            c0[0, :, 20 + i] = c0[0, :, 20 + node].clone()
        assert torch.equal(c, c0)
    tree.plan(PARENTS, torch.tensor([6, 5]))
    assert tree.lens.tolist() == [29, history + 5]


def test_the_history_of_an_accepted_commit(gqa):
    """All nodes, some, the root, none of an empty tree: the same lengths from both forms of the call."""
    layout = gqa.layout_pool(4, 32, 2)
    k, v = (torch.zeros(4, 2, 32, D, dtype=BF16, device=DEV) for _ in range(2))
    table, parents = ints([[0], [1], [2], [3]]), PARENTS[:1].expand(4, 6)
    tree = gqa.DraftTree(4, 6, 8, 2, DEV)
    tree.plan(parents, torch.tensor([6, 6, 3, 0]), torch.tensor([26, 5, 0, 7]))
    tree.path.copy_(ints([[0, 1, 2, 3, 4, 5], [0, 1, 3, -1, -1, -1], [0, -1, -1, -1, -1, -1], [-1] * 6]))
    tree.kept.copy_(ints([6, 3, 1, 0]))
    plain = ints([0] * 4)
    gqa.tree_commit(k, v, num_kv_heads=2, layout=layout, seq_lens_dev=tree.lens, path=tree.path, kept=tree.kept, seq_lens_out=plain,
                    tree_sizes=tree.sizes, block_table=table)
    tree.commit(k, v, layout=layout, block_table=table)
    assert int(tree.status) == 0
    assert tree.history.tolist() == plain.tolist() == [32, 8, 1, 7]


@pytest.mark.parametrize("path,kept", [([0, 1, -1, -1, -1, -1], 2), ([0, 1, 3, -1, -1, -1], 3)])
@pytest.mark.parametrize("missing", [-1, 4])
def test_commit_refuses_kept_rows_without_a_block(gqa, path, kept, missing):
    """Rows that stay where they are must have a place too: no other call could have written them."""
    layout = gqa.layout_pool(4, 32, 2)
    k, v = (torch.ones(4, 2, 32, D, dtype=BF16, device=DEV) for _ in range(2))
    new, status = ints([0]), ints([0])
    kw = dict(num_kv_heads=2, layout=layout, path=ints([path]), kept=ints([kept]), seq_lens_out=new, block_table=ints([[2, missing]]), status=status)
    gqa.tree_commit(k, v, seq_lens_dev=ints([37]), **kw)   # nodes in slots 31 .. 36
    assert int(status) == 3 and int(new) == 37 and (k == 1).all() and (v == 1).all()
    status.zero_()
    gqa.tree_commit(k, v, seq_lens_dev=ints([37]), keep_history=True, **kw)
    assert int(status) == 3 and int(new) == 31
    status.zero_()
    gqa.tree_commit(k, v, seq_lens_dev=ints([32]), **kw)   # 26 .. 31
    assert int(status) == 0 and int(new) == 26 + kept


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_commit_of_one_layer_in_a_buffer_of_odd_size(gqa, dtype):
    """With one layer there is no distance between layers to be aligned."""
    gen = torch.Generator().manual_seed(6)
    layout = gqa.layout_reference(1, 32, 2)
    k, v = (torch.randn(32 * 2 * D + 3, generator=gen).to(dtype).to(DEV) for _ in range(2))
    want = [c.clone() for c in (k, v)]
    for c in want:
        c[: 32 * 2 * D].view(32, 2, D)[17] = c[: 32 * 2 * D].view(32, 2, D)[18].clone()
    new = ints([0])
    gqa.tree_commit(k, v, num_kv_heads=2, layout=layout, seq_lens_dev=ints([20]), path=ints([[0, 2, -1, -1]]), kept=ints([2]),
                    seq_lens_out=new)
    assert int(new) == 18 and torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_a_block_other_than_the_first(gqa, dtype):
    """Without a block table the caches may be any block of a larger one: the same bits as in a cache of its own,
    and the other blocks stay as they are."""
    gen = torch.Generator().manual_seed(7)
    hq, hkv, tokens, cap, vocab = 8, 2, 6, 200, 30
    parents = PARENTS[:1]
    freq, _ = gqa.rope_frequencies(64)
    freq = freq.to(DEV)
    caches = [torch.randn(3, cap, hkv, D, generator=gen).to(dtype).to(DEV) for _ in range(2)]
    before = [c.clone() for c in caches]
    q, kn, vn = (torch.randn(1, tokens, h, D, generator=gen).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    target = torch.softmax(torch.randn(1, tokens, vocab, generator=gen), -1).to(DEV)
    words = torch.randint(0, vocab, (1, tokens), generator=gen).int().to(DEV)
    u = torch.full((1, tokens), 1e-6, device=DEV)  # nearly every draft is taken
    results = []
    for block in (0, 2):
        k, v = caches if block else [c[2].clone() for c in caches]
        tree = gqa.DraftTree(1, tokens, hq, hkv, DEV, dtype)
        tree.plan(parents, None, torch.tensor([150]))
        kw = dict(layout=gqa.layout_reference(3 if block else 1, cap, hkv), fixed_block=block)
        rot, out = torch.zeros_like(q), torch.zeros_like(q)
        tree.append(q, kn, vn, k, v, freq=freq, q_out=rot, **kw)
        tree.attend(rot, k, v, out, **kw)
        tree.verify(target, None, words, u, torch.full((1,), 0.5, device=DEV))
        tree.commit(k, v, **kw)
        assert int(tree.status) == 0 and int(tree.kept) > 1
        results.append([rot, out, tree.path, tree.next_token, tree.history] + [(c[2] if block else c) for c in (k, v)])
    assert out.abs().sum() > 0
    for a, b in zip(*results):
        assert torch.equal(a, b)
    for c, c0 in zip(caches, before):
        assert torch.equal(c[:2], c0[:2]) and not torch.equal(c[2], c0[2])

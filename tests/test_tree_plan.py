"""Tree drafting without a GPU: what DraftTree.plan takes and leaves in the buffers, refusals."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from test_tree_host import COMMON, _fill


@pytest.fixture(scope="module")
def gqa(built_lib):
    import llminfer_b200 as pkg
    return pkg


@pytest.fixture
def tree(monkeypatch, gqa):
    """A DraftTree of two sequences on the host: plan() needs no GPU."""
    from llminfer_b200 import binding as B
    monkeypatch.setattr(B, "tree_workspace", lambda *a: torch.zeros(16, dtype=torch.uint8))
    return gqa.DraftTree(2, 4, 8, 2, "cpu")


PARENTS = torch.tensor([[-1, 0, 0, 1], [-1, 0, 1, 2]])


@pytest.mark.parametrize("history", [torch.tensor([5]), torch.tensor(5), torch.tensor([5, 6, 7]), torch.tensor([[5, 6]])])
def test_plan_refuses_a_history_of_another_shape(tree, history):
    """One number is not spread over all sequences."""
    with pytest.raises(ValueError, match="history"):
        tree.plan(PARENTS, None, history)


@pytest.mark.parametrize("history", [torch.tensor([5.5, 6.0]), torch.tensor([True, False])])
def test_plan_refuses_a_history_that_is_not_whole_numbers(tree, history):
    with pytest.raises(TypeError, match="history"):
        tree.plan(PARENTS, None, history)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_plan_fills_the_buffers(tree, kind):
    tree.plan(PARENTS.to(kind), torch.tensor([4, 2], dtype=kind), torch.tensor([5, 6], dtype=kind))
    assert tree.lens.tolist() == [9, 8] and tree.history.tolist() == [5, 6] and tree.sizes.tolist() == [4, 2]
    assert torch.equal(tree.parents, PARENTS.int())
    tree.plan(PARENTS)  # from the lengths that are there
    assert tree.lens.tolist() == [9, 10] and tree.sizes.tolist() == [4, 4]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(path=None), -1), (dict(num_layers=0), -3), (dict(seq_lens_out=0x2000, kept=0x2000), -8)])
def test_tree_commit_history_refuses_what_tree_commit_refuses(gqa, kw, code):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeCommitParams(), gqa, **{**dict(num_layers=1, seq_lens_out=0x3000), **kw})
    assert gqa.lib().gqa_tree_commit_history(C.byref(p)) == code
    assert gqa.lib().gqa_tree_commit_history(None) == -1


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("block,blocks,code", [(64, (1 << 25) - 1, -3), (32, (1 << 26) - 1, -3), (64, 1 << 25, -3)])
def test_tree_decode_refuses_positions_that_tiles_of_keys_would_carry_past_32_bits(gqa, dtype, block, blocks, code):
    """Capacities of 2^31 - 64, 2^31 - 32 and 2^31: the end of the last tile of 128 keys is no 32-bit number."""
    from llminfer_b200 import binding as B
    p = _fill(B._TreeDecodeParams(), gqa, dtype=dtype, workspace_bytes=1 << 40, out=0x2000, blocks_per_seq=blocks,
              layout=gqa.layout_pool(8, block, 2).c())
    assert gqa.lib().gqa_tree_decode(C.byref(p)) == code


ROW = 4 * 128 * 2  # bytes of a token's queries below


@pytest.mark.parametrize("offset,stride", [(16, 0), (-16, 0), (7 * ROW, 0), (-7 * ROW, 0), (-8 * ROW + 16, 0), (ROW, 1024), (ROW - 16, 1024), (14 * ROW, 1024)])
def test_tree_decode_refuses_output_that_reaches_into_the_queries(gqa, offset, stride):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeDecodeParams(), gqa, workspace_bytes=1 << 40, q=0x100000, out=0x100000 + offset, q_token_stride=stride)
    assert gqa.lib().gqa_tree_decode(C.byref(p)) == -8


@pytest.mark.parametrize("offset,stride,out_stride", [(16, 0, 0), (-16, 0, 0), (ROW, 0, 0), (-7 * ROW, 0, 0), (ROW - 16, 1280, 1280), (6 * ROW, 1280, 512),
                                                      (-2 * ROW, 512, 1280)])
def test_rope_append_refuses_rows_that_reach_into_one_another(gqa, offset, stride, out_stride):
    """In place is row on row; any other way to share memory overwrites rows that are still to be read."""
    from llminfer_b200 import binding as B
    p = _fill(B._RopeParams(), gqa, rotary_dim=128, eps=1e-6, attn_factor=1.0, q=0x100000, q_out=0x100000 + offset, q_token_stride=stride,
              q_out_token_stride=out_stride)
    assert gqa.lib().gqa_rope_append(C.byref(p)) == -8


@pytest.mark.parametrize("name,size", [("seq_lens_dev", 2), ("tree_sizes_dev", 2), ("kept", 2), ("path", 8)])
def test_tree_commit_refuses_lengths_that_reach_into_its_inputs(gqa, name, size):
    """Two sequences of four nodes: outputs that begin below an input's end or end above its beginning."""
    from llminfer_b200 import binding as B
    for at in (-1, 1, size - 1):
        p = _fill(B._TreeCommitParams(), gqa, num_layers=1, seq_lens_out=0x3000 + 4 * at, **{name: 0x3000})
        for call in (gqa.lib().gqa_tree_commit, gqa.lib().gqa_tree_commit_history):
            assert call(C.byref(p)) == -8, at


@pytest.mark.parametrize("rotary,base,factor,original,fast,slow", [
    (128, 1e6, 4.0, 32768, 32.0, 1.0), (128, 1e6, 40.0, 4096, 32.0, 1.0), (64, 1e4, 2.0, 2048, 16.0, 2.0), (8, 1e4, 8.0, 131072, 32.0, 1.0)])
def test_yarn_interpolates_linearly_in_turns(gqa, rotary, base, factor, original, fast, slow):
    """Every pair, those between the ramp's ends among them: a pair that turns r times over the trained context keeps
    (r - slow) / (fast - slow) of its frequency, cut to 0 .. 1, and divides the rest by the factor. Both sides take some ten
    FP64 roundings, of numbers at most 4 times the result: below 1e-14."""
    f, a = gqa.rope_frequencies(rotary, base=base, scaling="yarn", factor=factor, original_len=original, beta_fast=fast, beta_slow=slow)
    plain = base ** (-2.0 * np.arange(rotary // 2) / rotary)
    keep = np.clip((original * plain / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
    assert rotary < 64 or ((keep > 0) & (keep < 1)).sum() >= 4
    np.testing.assert_allclose(f.numpy(), plain * (keep + (1.0 - keep) / factor), rtol=1e-14)
    assert a == pytest.approx(0.1 * math.log(factor) + 1.0, rel=2.0 ** -24)

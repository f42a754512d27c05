"""Tree drafting, what needs no GPU: struct layouts, masks, frequencies, refusals of the entry points
before any CUDA call, refusals of the binding."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import tree_helpers as TH

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def gqa(built_lib):
    import llminfer_b200 as pkg
    return pkg


def test_struct_layouts_match_the_header(gqa, tmp_path):
    from llminfer_b200 import binding as B
    mirrors = {"gqa_rope_params": B._RopeParams, "gqa_tree_decode_params": B._TreeDecodeParams,
               "gqa_tree_verify_params": B._TreeVerifyParams,
               "gqa_tree_commit_params": B._TreeCommitParams}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "gqa_b200.h"', "int main(void) {"]
    for name, mirror in mirrors.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _ in mirror._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    lines += ["return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.strip().splitlines())
    for name, mirror in mirrors.items():
        assert int(got[name]) == C.sizeof(mirror), name
        for field, _ in mirror._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(mirror, field).offset, (name, field)


def test_packed_blocks_match_the_structs(gqa):
    """The blocks the binding packs in one go have every field where the structures have it."""
    from llminfer_b200 import binding as B

    def flat(kind):
        for name, t in kind._fields_:
            yield from (((name, f) for f, _ in t._fields_) if t is B._Layout else ((name,),))

    for block, kind in ((B._ROPE, B._RopeParams), (B._TREE_DECODE, B._TreeDecodeParams),
                        (B._TREE_VERIFY, B._TreeVerifyParams), (B._TREE_COMMIT, B._TreeCommitParams)):
        names = list(flat(kind))
        assert block.size == C.sizeof(kind)
        p = kind.from_buffer_copy(block.pack(*range(1, len(names) + 1)))
        for i, name in enumerate(names):
            v = p
            for f in name:
                v = getattr(v, f)
            assert v == i + 1, name


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 64, 127, 128])
def test_masks_and_depths(gqa, tokens):
    rng = np.random.default_rng(tokens)
    sizes = [tokens, max(1, tokens // 2), 0]
    par = np.full((3, tokens), 99, dtype=np.int32)  # entries behind a tree's end are ignored
    sees = []
    for b, n in enumerate(sizes):
        tree = TH.random_parents(rng, n)[:n]
        par[b, :n] = tree
        sees.append(TH.ancestors(tree))
    mask, depth = gqa.tree_masks(torch.from_numpy(par), torch.tensor(sizes))
    assert torch.equal(mask, TH.pack_mask(sees, tokens))
    for b, n in enumerate(sizes):
        assert depth[b, :n].tolist() == [int(sees[b][t].sum()) - 1 for t in range(n)]
        assert not depth[b, n:].any()


@pytest.mark.parametrize("row", [[0, 0], [-1, 1], [-1, -1], [-1, 2]])
def test_masks_refuse_parents_out_of_order(gqa, row):
    with pytest.raises(gqa.GqaError) as e:
        gqa.tree_masks(torch.tensor([row]))
    assert e.value.status == -5


def test_masks_refuse_shapes_and_sizes(gqa):
    for par, sizes, code in ((torch.zeros(1, 129), None, -3),
                             (torch.zeros(0, 4), None, -1),  # an empty tensor has no address
                             (torch.tensor([[-1, 0]]), torch.tensor([3]), -5),
                             (torch.tensor([[-1, 0]]), torch.tensor([-1]), -5)):
        with pytest.raises(gqa.GqaError) as e:
            gqa.tree_masks(par, sizes)
        assert e.value.status == code
    with pytest.raises(ValueError):
        gqa.tree_masks(torch.tensor([[-1, 0]]), torch.tensor([1, 1]))


def test_frequencies(gqa):
    f, a = gqa.rope_frequencies(128)
    i = np.arange(64)
    plain = 1e6 ** (-2.0 * i / 128)
    np.testing.assert_allclose(f.numpy(), plain, rtol=1e-14)
    assert a == 1.0
    f, a = gqa.rope_frequencies(64, base=1e4, scaling="linear", factor=8.0)
    np.testing.assert_allclose(f.numpy(), 1e4 ** (-2.0 * np.arange(32) / 64) / 8, rtol=1e-14)
    f, a = gqa.rope_frequencies(64, base=1e4, scaling="ntk", factor=8.0)
    base = 1e4 * 8.0 ** (64 / 62)
    np.testing.assert_allclose(f.numpy(), base ** (-2.0 * np.arange(32) / 64), rtol=1e-13)
    # The slowest pair is stretched by exactly the factor, the fastest not at all.
    np.testing.assert_allclose(f.numpy()[[0, 31]] * np.array([1, 8.0]), 1e4 ** np.array([0, -62 / 64]), rtol=1e-13)
    f, a = gqa.rope_frequencies(128, scaling="yarn", factor=4.0, original_len=32768)
    turns = 32768 * plain / (2 * math.pi)
    assert np.array_equal(f.numpy()[turns >= 32], plain[turns >= 32]) or np.allclose(
        f.numpy()[turns >= 32], plain[turns >= 32], rtol=1e-14)
    np.testing.assert_allclose(f.numpy()[turns <= 1], plain[turns <= 1] / 4, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((f.numpy()[mid] > plain[mid] / 4) & (f.numpy()[mid] < plain[mid])).all()
    assert a == pytest.approx(0.1 * math.log(4.0) + 1.0, rel=1e-7)


@pytest.mark.parametrize("kw,code", [
    (dict(rotary_dim=4), -3), (dict(rotary_dim=20), -3), (dict(rotary_dim=136), -3),
    (dict(scaling="linear", factor=0.5), -5), (dict(scaling="ntk", factor=float("nan")), -5),
    (dict(scaling="linear", factor=float("inf")), -5), (dict(scaling="yarn", factor=4.0), -5),
    (dict(scaling="yarn", factor=4.0, original_len=4096, beta_fast=1.0, beta_slow=2.0), -5)])
def test_frequencies_refuse(gqa, kw, code):
    with pytest.raises(gqa.GqaError) as e:
        gqa.rope_frequencies(**kw)
    assert e.value.status == code


FAKE = 0x1000  # aligned, never touched: every call below is refused first


def _layout(gqa, block=64):
    return gqa.layout_pool(8, block, 2).c()


def _fill(p, gqa, **kw):
    p.dtype, p.batch, p.tokens = 2, 2, 4
    for name, value in (("num_q_heads", 4), ("num_kv_heads", 2), ("head_dim", 128), ("blocks_per_seq", 2)):
        if hasattr(p, name):
            setattr(p, name, value)
    if hasattr(p, "layout"):
        p.layout = _layout(gqa)
    for name, kind in p._fields_:
        if kind is C.c_void_p and name not in ("status_dev", "stream"):
            setattr(p, name, FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


COMMON = [(dict(dtype=3), -2), (dict(batch=0), -3), (dict(tokens=0), -3), (dict(tokens=129), -3),
          (dict(num_kv_heads=0), -3), (dict(head_dim=64), -3), (dict(k_cache=None), -1), (dict(v_cache=None), -1),
          (dict(seq_lens_dev=None), -1), (dict(k_cache=0x1008), -4), (dict(blocks_per_seq=0), -3),
          (dict(block_table_dev=None), -3), (dict(block_table_dev=None, batch=1, fixed_block=8), -5),
          (dict(block_table_dev=None, batch=1, fixed_block=-1), -5), (dict(blocks_per_seq=1 << 26), -3)]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(num_q_heads=0), -3), (dict(q=None), -1), (dict(q_out=None), -1), (dict(k_new=None), -1),
    (dict(v_new=None), -1), (dict(freq_dev=None), -1), (dict(rotary_dim=12), -3), (dict(rotary_dim=0), -3),
    (dict(rotary_dim=136), -3), (dict(style=2), -8), (dict(q_token_stride=500), -3), (dict(k_token_stride=255), -3),
    (dict(q_token_stride=516), -4), (dict(qk_weight=0x1004), -4), (dict(freq_dev=0x1004), -4),
    (dict(q_token_stride=1024), -3)])  # in place (q_out is q) with another stride
def test_rope_append_refuses(gqa, kw, code):
    from llminfer_b200 import binding as B
    p = _fill(B._RopeParams(), gqa, **{**dict(rotary_dim=128, style=0, eps=1e-6, attn_factor=1.0), **kw})
    assert gqa.lib().gqa_rope_append(C.byref(p)) == code


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(num_q_heads=0), -3), (dict(num_q_heads=5), -3), (dict(num_q_heads=18), -8), (dict(batch=1025), -8),
    (dict(q=None), -1), (dict(out=None), -1), (dict(workspace=None), -1), (dict(q=0x1002), -4), (dict(out=0x1002), -4),
    (dict(q_token_stride=500), -3), (dict(q_token_stride=516), -4)])
def test_tree_decode_refuses(gqa, kw, code):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeDecodeParams(), gqa, **{**dict(workspace_bytes=1 << 40), **kw})
    assert gqa.lib().gqa_tree_decode(C.byref(p)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), -2), (dict(batch=0), -3), (dict(tokens=0), -3), (dict(tokens=129), -3), (dict(vocab=0), -3),
    (dict(target=None), -1), (dict(tokens_dev=None), -1), (dict(parents_dev=None), -1), (dict(u_accept=None), -1),
    (dict(u_sample=None), -1), (dict(path=None), -1), (dict(kept=None), -1), (dict(next_token=None), -1),
    (dict(target=0x1001), -4), (dict(draft=0x1001), -4), (dict(target_node_stride=-4), -3)])
def test_tree_verify_refuses(gqa, kw, code):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeVerifyParams(), gqa, **{**dict(vocab=100), **kw})
    assert gqa.lib().gqa_tree_verify(C.byref(p)) == code


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(path=None), -1), (dict(kept=None), -1), (dict(seq_lens_out=None), -1), (dict(num_layers=0), -3),
    (dict(num_layers=2, layer_stride=0), -3), (dict(num_layers=2, layer_stride=4), -4), (dict(batch=65536), -3),
    (dict(seq_lens_out=0x2000, seq_lens_dev=0x2000), -8)])
def test_tree_commit_refuses(gqa, kw, code):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeCommitParams(), gqa, **{**dict(num_layers=1, seq_lens_out=0x3000), **kw})
    assert gqa.lib().gqa_tree_commit(C.byref(p)) == code


def test_null_parameter_blocks(gqa):
    for name in ("gqa_rope_append", "gqa_tree_decode", "gqa_tree_verify", "gqa_tree_commit"):
        assert getattr(gqa.lib(), name)(None) == -1
    assert gqa.lib().gqa_tree_masks(None, None, 1, 1, None, None) == -1


def test_workspace_sizes(gqa):
    size = gqa.lib().gqa_tree_workspace_bytes
    assert size(2, 1, 8, 32, 8, 148) > 0 and size(1, 1, 8, 32, 8, 148) > 0
    for bad in ((3, 1, 8, 32, 8, 148), (2, 0, 8, 32, 8, 148), (2, 1025, 8, 32, 8, 148), (2, 1, 129, 32, 8, 148),
                (2, 1, 8, 30, 8, 148), (2, 1, 8, 72, 8, 148), (2, 1, 8, 0, 8, 148)):
        assert size(*bad) == 0, bad


def test_binding_refuses_wrong_tensors(monkeypatch, gqa):
    """Types, shapes, devices and strides are refused in Python, before a call; host tensors stand in
    for tensors on another device than the current one."""
    from llminfer_b200 import binding as B
    monkeypatch.setattr(B.torch.cuda, "current_device", lambda: 0)
    host = torch.zeros(1, 4, 4, 128, dtype=torch.bfloat16)
    lens = torch.zeros(1, dtype=torch.int32)
    lay = gqa.layout_pool(8, 64, 2)
    with pytest.raises(ValueError, match="current device"):
        gqa.tree_decode(host, host, host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens)
    with pytest.raises(ValueError, match="current device"):
        gqa.tree_verify(torch.zeros(1, 4, 9), None, lens, lens, lens, lens, path=lens, kept=lens, next_token=lens)
    monkeypatch.setattr(B.torch.cuda, "current_device", lambda: -1)  # what get_device() says of host tensors
    with pytest.raises(TypeError):
        gqa.tree_decode(host, host.float(), host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens)
    with pytest.raises(TypeError, match="seq_lens_dev"):
        gqa.tree_decode(host, host, host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens.long())
    with pytest.raises(ValueError, match="mask"):
        gqa.tree_decode(host, host, host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens,
                        mask=torch.zeros(1, 4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="packed"):
        gqa.tree_decode(host.transpose(1, 2), host, host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens)
    with pytest.raises(ValueError, match="packed"):
        gqa.tree_decode(host[:, :1].expand(1, 4, 4, 128), host, host, host, num_kv_heads=2, layout=lay, seq_lens_dev=lens)
    with pytest.raises(ValueError, match="share memory"):
        gqa.tree_verify(torch.zeros(1, 1, 9).expand(1, 4, 9), None, lens, lens, lens, lens, path=lens, kept=lens,
                        next_token=lens)
    with pytest.raises(ValueError, match="contiguous"):
        gqa.tree_verify(torch.zeros(2, 4, 9), None, torch.zeros(4, 2, dtype=torch.int32).t(), lens, lens, lens,
                        path=lens, kept=lens, next_token=lens)


@pytest.mark.parametrize("alias", ["kept", "path", "tree_sizes_dev"])
def test_tree_commit_refuses_lengths_on_top_of_its_inputs(gqa, alias):
    """Blocks of one launch read the inputs while another writes the lengths."""
    from llminfer_b200 import binding as B
    p = _fill(B._TreeCommitParams(), gqa, num_layers=1, seq_lens_out=0x3000, **{alias: 0x3000})
    assert gqa.lib().gqa_tree_commit(C.byref(p)) == -8


def test_commit_wants_a_stride_for_layers_that_are_not_packed(monkeypatch, gqa):
    """Half of a cache that holds K and V side by side has its layers twice as far apart as its size says."""
    from llminfer_b200 import binding as B
    monkeypatch.setattr(B.torch.cuda, "current_device", lambda: -1)
    both = torch.zeros(3, 2, 64 * 2 * 128, dtype=torch.bfloat16)
    ints = torch.zeros(1, dtype=torch.int32)
    kw = dict(num_kv_heads=2, layout=gqa.layout_reference(1, 64, 2), seq_lens_dev=ints, path=torch.zeros(1, 4, dtype=torch.int32),
              kept=ints, seq_lens_out=ints)
    for k, v, layers in ((both[:, 0], both[:, 1], 3), (both[:, 0].contiguous(), both[:, 1], 3), (both, both, 5)):
        with pytest.raises(ValueError, match="layer_stride"):
            gqa.tree_commit(k, v, layers=layers, **kw)
    with pytest.raises(gqa.GqaError):  # no layers
        gqa.tree_commit(both, both, layers=0, stream=0, **kw)


def test_rope_append_wants_a_row_of_frequencies(monkeypatch, gqa):
    from llminfer_b200 import binding as B
    monkeypatch.setattr(B.torch.cuda, "current_device", lambda: -1)
    q = torch.zeros(1, 4, 4, 128)
    lens = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="freq"):
        gqa.rope_append(q, q, q, q, q, layout=gqa.layout_reference(1, 64, 4), seq_lens_dev=lens,
                        freq=torch.zeros(8, 2, dtype=torch.float64))


def test_tree_decode_refuses_output_on_top_of_the_queries(gqa):
    from llminfer_b200 import binding as B
    p = _fill(B._TreeDecodeParams(), gqa, workspace_bytes=1 << 40)
    assert p.q == p.out and gqa.lib().gqa_tree_decode(C.byref(p)) == -8

"""FP64 references and inputs of the tree-drafting tests."""
from __future__ import annotations

import math

import numpy as np
import torch

D = 128
DEV = "cuda:0"


def random_parents(rng, tokens, width=4):
    par = [-1] + [max(0, t - 1 - int(rng.integers(0, width))) for t in range(1, tokens)]
    return par


def ancestors(parents):
    """sees[t][j] for one tree."""
    n = len(parents)
    sees = np.zeros((n, n), dtype=bool)
    for t in range(n):
        if parents[t] >= 0:
            sees[t] = sees[parents[t]]
        sees[t, t] = True
    return sees


def pack_mask(sees, tokens):
    """[batch, tokens, words] int32 words from a list of [n, n] truth values."""
    words = (tokens + 31) // 32
    out = np.zeros((len(sees), tokens, words), dtype=np.uint32)
    for b, s in enumerate(sees):
        for t in range(s.shape[0]):
            for j in np.nonzero(s[t])[0]:
                out[b, t, j // 32] |= np.uint32(1 << (int(j) % 32))
    return torch.from_numpy(out.view(np.int32))


class Cache:
    """K and V caches whose unused rows hold NaN: paged in random order, or one block."""

    def __init__(self, gqa, rng, lens, capacity, hkv, block, dtype, layers=1):
        self.block, self.hkv, self.dtype = block, hkv, dtype
        batch = len(lens)
        if block:
            per = (capacity + block - 1) // block
            blocks = batch * per + 2
            order = rng.permutation(blocks)[: batch * per].reshape(batch, per)
            table = np.full((batch, per), -1, dtype=np.int64)
            for b, n in enumerate(lens):
                need = (n + block - 1) // block
                table[b, :need] = order[b, :need]
            self.table_host = table
            self.table = torch.from_numpy(table.astype(np.int32)).to(DEV)
            self.layout = gqa.layout_pool(blocks, block, hkv)
            shape = (layers, blocks, hkv, block, D)
        else:
            assert batch == 1
            self.table_host, self.table = None, None
            self.layout = gqa.layout_reference(1, capacity, hkv)
            shape = (layers, 1, capacity, hkv, D)
        self.k = torch.full(shape, float("nan"), dtype=dtype)
        self.v = torch.full(shape, float("nan"), dtype=dtype)

    def at(self, b, pos):
        """Index of row (b, pos) in [layer, ...]: use cache[(layer,) + at] -> [hkv, 128]."""
        if self.block:
            return (int(self.table_host[b, pos // self.block]), slice(None), pos % self.block)
        return (0, pos)

    def fill(self, gen, lens):
        for b, n in enumerate(lens):
            for pos in range(n):
                i = (slice(None),) + self.at(b, pos)
                self.k[i] = torch.randn(self.k[i].shape, generator=gen).to(self.dtype)
                self.v[i] = torch.randn(self.v[i].shape, generator=gen).to(self.dtype)
        return self

    def rows(self, which, b, n, layer=0):
        """[n, hkv, 128] of sequence b (host)."""
        c = getattr(self, which)[layer]
        if n == 0:
            return c.new_zeros((0, self.hkv, D))
        return torch.stack([c[self.at(b, p)] for p in range(n)])

    def device(self):
        return self.k.to(DEV), self.v.to(DEV)


def attention(q, k, v, base, sees):
    """One sequence in FP64: q [n, hq, 128], k/v [base + n, hkv, 128], sees [n, n]. Returns the output,
    the weighted sum of |v| and the largest sum of |q_i k_i| of a visible key, per (node, head)."""
    n, hq, _ = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(n, hq, D, dtype=torch.float64)
    spread = torch.zeros(n, hq, D, dtype=torch.float64)
    size = torch.zeros(n, hq, 1, dtype=torch.float64)
    for t in range(n):
        keys = list(range(base)) + [base + j for j in range(n) if sees[t][j]]
        if not keys:
            continue
        for h in range(hq):
            kk, vv = k[keys, h // group], v[keys, h // group]
            w = torch.softmax(kk @ q[t, h] / math.sqrt(D), 0)
            out[t, h] = w @ vv
            spread[t, h] = w @ vv.abs()
            size[t, h, 0] = (kk.abs() @ q[t, h].abs()).max()
    return out, spread, size


def attention_bound(out, spread, size, keys, dtype):
    """How far a kernel that follows the definition may be off, element by element.

    Scores are FP32 sums of 128 products: off by at most 129 * 2^-24 * sum |q_i k_i|, times 1 / sqrt(128)
    and log2(e); their scaling, the maximum's subtraction and 2^x add three roundings of numbers below that
    sum and 2^-21 of the value. A weight's relative error is that (times ln 2) for itself and
    once more through the normalisation; sums over the keys add keys * 2^-24. With BF16 rows the weights are
    rounded to BF16 (2^-8, half a step) and so is the output."""
    eps = 2.0 ** -24
    score = size / math.sqrt(D) * (129 + 3) * eps
    weight = 2 * (score + 2.0 ** -21) + 2 * (keys + 16) * eps
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * out.abs() + (2.0 ** -8 + weight) * (1 + 2.0 ** -7) * spread + 1e-30
    return eps * out.abs() + weight * spread + 1e-30


def verify(target, draft, tokens, parents, n, u, us):
    """One sequence by the definition, residuals normalised one after another. Host tensors/arrays."""
    if n == 0:
        return [], -1
    clean = lambda x: np.where(np.isnan(x) | (x < 0), 0.0, x)
    node, path = 0, [0]
    while True:
        p = clean(target[node].double().numpy())
        q = clean(draft[node].double().numpy()) if draft is not None else None
        step = None
        for t in range(node + 1, n):
            if parents[t] != node or not 0 <= tokens[t] < len(p):
                continue
            x = tokens[t]
            if u[t] * (q[x] if q is not None else 1.0) < p[x]:
                step = t
                break
            less = np.maximum(p - q, 0.0) if q is not None else np.where(np.arange(len(p)) == x, 0.0, p)
            total = less.sum()
            p = less / total if total > 0 else less
        if step is None:
            break
        node = step
        path.append(step)
    if not p.sum() > 0:
        p = clean(target[node].double().numpy())
        if not p.sum() > 0:
            return path, -1
    upto = np.cumsum(p)
    past = np.nonzero((upto > us * upto[-1]) & (p > 0))[0]
    return path, int(past[0]) if len(past) else int(np.nonzero(p > 0)[0][-1])

"""Cases of the tree-drafted decode step: rope_append, tree_decode, tree_verify, tree_commit.

A decode loop that drafts several tokens as a tree runs, per step: the rotary stage that appends the
drafted tokens' key and value rows behind the cache (rope_append), attention of all nodes over prefix and
ancestors (tree_decode), the verification of the draft against the target's probabilities
(tree_verify), and the move of the accepted path's cache rows to the front of the draft's slots
(tree_commit). `run` computes one of them, in elementary torch operations or (own) with the framework.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
D = 128
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one user, a short draft: latency
        dict(name="attend b1 t8 1K", op="attend", batch=1, tokens=8, hq=32, hkv=8, lo=1024, hi=1024, block=0, shape="tree"),
        # a serving batch of unequal histories in 256-token pages
        dict(name="attend b16 t16 ragged", op="attend", batch=16, tokens=16, hq=32, hkv=8, lo=256, hi=8192, block=256, shape="tree"),
        # a wide tree over a long history: 512 rows for each KV head, arithmetic as heavy as the bytes
        dict(name="attend b1 t64 32K", op="attend", batch=1, tokens=64, hq=64, hkv=8, lo=32768, hi=32768, block=256, shape="tree"),
        # the longest context the framework is measured on, a short chain
        dict(name="attend b4 t8 128K", op="attend", batch=4, tokens=8, hq=64, hkv=8, lo=131072, hi=131072, block=256, shape="chain"),
        # one user's draft: latency
        dict(name="rope b1 t8", op="rope", batch=1, tokens=8, hq=32, hkv=8, dtype="bf16", style="half", rotary=128, scaling="none", hi=4000, norm=True, block=0),
        # FP32 rows, interleaved pairs, half of the head
        dict(name="rope b16 t13 fp32", op="rope", batch=16, tokens=13, hq=16, hkv=8, dtype="fp32", style="interleaved", rotary=64, scaling="linear", hi=30000, norm=False, block=256),
        # a large batch of wide trees far out in a stretched context
        dict(name="rope b64 t64 yarn", op="rope", batch=64, tokens=64, hq=64, hkv=8, dtype="bf16", style="half", rotary=128, scaling="yarn", hi=131072, norm=True, block=256),
        # one user, a chain: latency
        dict(name="verify b1 t8 32K words", op="verify", batch=1, tokens=8, vocab=32000, dtype="fp32", draft="probs", shape="chain"),
        # a serving batch of trees
        dict(name="verify b16 t32 128K words", op="verify", batch=16, tokens=32, vocab=128000, dtype="fp32", draft="probs", shape="tree"),
        # a large batch, drafts looked up and not sampled, BF16 probabilities, an odd vocabulary
        dict(name="verify b64 t16 lookup", op="verify", batch=64, tokens=16, vocab=151643, dtype="bf16", draft="none", shape="tree"),
        # one user, all layers of a model
        dict(name="commit b1 36 layers", op="commit", batch=1, tokens=8, accepted=4, layers=36, hkv=8, dtype="bf16", hi=200, block=0),
        # a large batch of wide trees
        dict(name="commit b32 t64 36 layers", op="commit", batch=32, tokens=64, accepted=9, layers=36, hkv=8, dtype="bf16", hi=150, block=64),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "rope", "verify", "verify", "commit"])
    if op == "attend":
        hq, hkv = rng.choice([(16, 8), (32, 8), (64, 8), (40, 8), (24, 4), (12, 2), (7, 1), (8, 8)])
        block = rng.choice([0, 32, 64, 96, 256])
        hi = _span(rng, 40, 131072)
        tokens = min(_span(rng, 1, 128), hi)
        batch = 1 if block == 0 else _span(rng, 1, 48)
        while batch * hi > 524288 or batch * hi * hq * tokens > 64 * 64 * 32768:
            if batch > 1:
                batch = max(1, batch // 2)
            else:
                tokens = max(1, tokens // 2)
        lo = hi if batch == 1 else max(tokens, _span(rng, max(1, hi // 16), hi))
        return dict(op=op, batch=batch, tokens=tokens, hq=hq, hkv=hkv, lo=lo, hi=hi, block=block, shape=rng.choice(["tree", "chain"]))
    if op == "rope":
        hq, hkv = rng.choice([(16, 8), (32, 8), (64, 8), (40, 8), (7, 1)])
        block = rng.choice([0, 64, 256])
        return dict(op=op, batch=1 if block == 0 else _span(rng, 1, 64), tokens=_span(rng, 1, 64), hq=hq, hkv=hkv, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    style=rng.choice(["half", "interleaved"]), rotary=rng.choice([128, 128, 96, 64, 32]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), hi=_span(rng, 300, 131072), norm=rng.choice([True, False]), block=block)
    if op == "verify":
        batch, tokens, vocab = _span(rng, 1, 64), _span(rng, 1, 64), _span(rng, 1000, 152000)
        while batch * tokens * vocab > 16 * 32 * 128000:
            batch, tokens = max(1, batch // 2), max(2, tokens * 2 // 3)
        return dict(op=op, batch=batch, tokens=tokens, vocab=vocab, dtype=rng.choice(["fp32", "fp32", "bf16"]), draft=rng.choice(["probs", "probs", "none"]),
                    shape=rng.choice(["chain", "tree"]))
    tokens = _span(rng, 2, 64)
    block = rng.choice([0, 32, 64])
    return dict(op=op, batch=1 if block == 0 else _span(rng, 1, 32), tokens=tokens, accepted=rng.randint(1, min(tokens, 9)), layers=rng.randint(1, 36),
                hkv=rng.choice([8, 8, 4, 1]), dtype=rng.choice(["bf16", "bf16", "fp32"]), hi=_span(rng, 70, 190), block=block)


# ---- inputs -----------------------------------------------------------------------------------

def _trees(r, batch, tokens, shape):
    """Sizes [batch] and parents [batch, tokens] (-1 at the root): a chain, or a random tree whose
    nodes hang from one of the nodes shortly before them. Sizes differ between the sequences."""
    sizes = np.full(batch, tokens, dtype=np.int32)
    if batch > 1:
        sizes = np.maximum(1, tokens - r.randint(0, tokens // 2 + 1, batch)).astype(np.int32)
    t = np.arange(tokens)
    if shape == "chain":
        parents = np.tile(t - 1, (batch, 1))
    else:
        parents = np.maximum(0, t[None] - 1 - r.randint(0, 4, (batch, tokens)))
    parents[:, 0] = -1
    return sizes, parents.astype(np.int32)


def _ancestors(parents):
    """Mask [batch, tokens, tokens] (node sees itself and its ancestors) and depths [batch, tokens]."""
    batch, tokens = parents.shape
    seen = np.zeros((batch, tokens, tokens), dtype=bool)
    depth = np.zeros((batch, tokens), dtype=np.int32)
    rows = np.arange(batch)
    for t in range(tokens):
        if t > 0:
            seen[:, t] = seen[rows, parents[:, t]]
            depth[:, t] = depth[rows, parents[:, t]] + 1
        seen[:, t, t] = True
    return seen, depth


def _bits(seen):
    """The mask in 32-bit words: bit j % 32 of word j / 32 of row t."""
    batch, tokens, _ = seen.shape
    words = (tokens + 31) // 32
    padded = np.zeros((batch, tokens, words * 32), dtype=np.uint64)
    padded[:, :, :tokens] = seen
    shift = (np.uint64(1) << np.arange(32, dtype=np.uint64))
    return (padded.reshape(batch, tokens, words, 32) * shift).sum(-1).astype(np.uint32).view(np.int32)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _pages(r, batch, positions, block):
    """Block table of a paged cache in random order, or None: one block that holds the sequence."""
    if block == 0:
        return None, 1, (positions + 31) // 32 * 32
    per = (positions + block - 1) // block
    order = r.permutation(batch * per + 3)[: batch * per].astype(np.int32)
    return _dev(order.reshape(batch, per)), batch * per + 3, block


def _frequencies(rotary, scaling, factor=4.0, original=32768, base=1e6):
    """Radians per position of each pair, and the factor on sine and cosine."""
    i = np.arange(rotary // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rotary / (rotary - 2.0))
    f = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = original * f / (2 * np.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    r = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op, batch, tokens = case["op"], case["batch"], case["tokens"]
    s = dict(case)
    sizes, parents = _trees(r, batch, tokens, case.get("shape", "tree"))
    seen, depth = _ancestors(parents)
    s["sizes_host"] = sizes
    s["sizes"], s["parents"], s["depth"] = _dev(sizes), _dev(parents), _dev(depth)
    if op == "verify":
        return _prepare_verify(s, r, g)
    dtype = torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16
    hkv = case["hkv"]
    if op == "attend":
        lens = np.maximum(sizes, r.randint(case["lo"], case["hi"] + 1, batch)) if case["lo"] < case["hi"] else np.full(batch, case["hi"])
        capacity = case["hi"]
    else:
        lens = sizes + r.randint(0, case["hi"] + 1, batch)
        capacity = case["hi"] + tokens
        if op == "rope" and case["block"]:  # far positions, of which the cache holds the last pages in earnest
            lens = sizes + r.randint(case["hi"] // 2, case["hi"] + 1, batch)
    s["lens"] = _dev(lens.astype(np.int32))
    s["lens_host"] = lens.astype(np.int64)
    if op == "rope" and case["block"]:
        # Only the pages that the new rows touch exist; the table's other entries share one page.
        block, per = case["block"], (capacity + case["block"] - 1) // case["block"]
        table = np.zeros((batch, per), dtype=np.int32)
        own_pages = (tokens + block - 1) // block + 1
        order = 1 + r.permutation(batch * own_pages).astype(np.int32).reshape(batch, own_pages)
        first = (lens - sizes) // block
        for k in range(own_pages):
            at = np.minimum(first + k, per - 1)
            table[np.arange(batch), at] = order[:, k]
        s["table"], s["blocks"], s["block_tokens"] = _dev(table), 1 + batch * own_pages, block
    else:
        s["table"], s["blocks"], s["block_tokens"] = _pages(r, batch, capacity, case["block"])
    layers = case.get("layers", 1)
    shape = (layers, s["blocks"], hkv, s["block_tokens"], D) if s["table"] is not None else (layers, s["blocks"], s["block_tokens"], hkv, D)
    if layers == 1:
        shape = shape[1:]
    s["k"] = torch.randn(shape, generator=g, device=DEV, dtype=dtype)
    s["v"] = torch.randn(shape, generator=g, device=DEV, dtype=dtype)
    if op == "attend":
        s["q"] = torch.randn((batch, tokens, case["hq"], D), generator=g, device=DEV, dtype=dtype)
        s["out"] = torch.zeros_like(s["q"])
        s["seen"], s["mask"] = _dev(seen), _dev(_bits(seen))
    elif op == "rope":
        s["q"] = torch.randn((batch, tokens, case["hq"], D), generator=g, device=DEV, dtype=dtype)
        s["q_out"] = torch.zeros_like(s["q"])
        s["k_new"] = torch.randn((batch, tokens, hkv, D), generator=g, device=DEV, dtype=dtype)
        s["v_new"] = torch.randn((batch, tokens, hkv, D), generator=g, device=DEV, dtype=dtype)
        s["weight"] = (1.0 + 0.1 * torch.randn(2 * D, generator=g, device=DEV)).to(dtype) if case["norm"] else None
        freq, s["factor"] = _frequencies(case["rotary"], case["scaling"])
        s["freq"] = _dev(freq)
    else:
        path = np.full((batch, tokens), -1, dtype=np.int32)
        kept = np.minimum(case["accepted"], sizes).astype(np.int32)
        for b in range(batch):
            rest = 1 + np.sort(r.permutation(sizes[b] - 1)[: kept[b] - 1])
            path[b, : kept[b]] = np.concatenate([[0], rest])
        s["path"], s["kept"] = _dev(path), _dev(kept)
        s["new_lens"] = torch.zeros_like(s["lens"])
    return s


def _prepare_verify(s, r, g):
    batch, tokens, vocab = s["batch"], s["tokens"], s["vocab"]
    dtype = torch.bfloat16 if s["dtype"] == "bf16" else torch.float32
    logits = torch.randn((batch, tokens, vocab), generator=g, device=DEV).mul_(3.0)
    s["target"] = torch.softmax(logits, -1).to(dtype)
    words = torch.zeros((batch, tokens), dtype=torch.int32, device=DEV)
    rows = torch.arange(batch, device=DEV)
    if s["draft"] == "probs":
        logits += torch.randn((batch, tokens, vocab), generator=g, device=DEV).mul_(0.8)
        s["probs"] = torch.softmax(logits, -1).to(dtype)
        source = s["probs"]
    else:
        s["probs"] = None
        source = s["target"]
    for t in range(1, tokens):  # every node is drawn from the draft's row at its parent
        words[:, t] = torch.multinomial(source[rows, s["parents"][:, t].long()].float(), 1, generator=g)[:, 0].int()
    s["words"] = words
    s["u_accept"] = torch.rand((batch, tokens), generator=g, device=DEV)
    s["u_sample"] = torch.rand(batch, generator=g, device=DEV)
    s["path"] = torch.zeros((batch, tokens), dtype=torch.int32, device=DEV)
    s["kept"] = torch.zeros(batch, dtype=torch.int32, device=DEV)
    s["next"] = torch.zeros(batch, dtype=torch.int32, device=DEV)
    return s


# ---- the framework's calls ----------------------------------------------------------------------

def _handle(s):
    """Layout and scratch, which a program makes once."""
    h = s.get("handle")
    if h is None:
        import llminfer_b200 as gqa
        h = s["handle"] = dict(gqa=gqa)
        if s["op"] != "verify":
            if s["table"] is not None:
                h["layout"] = gqa.layout_pool(s["blocks"], s["block_tokens"], s["hkv"])
            else:
                h["layout"] = gqa.layout_reference(s["blocks"], s["block_tokens"], s["hkv"])
        if s["op"] == "attend":
            h["workspace"] = gqa.tree_workspace(s["batch"], s["tokens"], s["hq"], s["hkv"], DEV)
    return h


def _run_own(s):
    h = _handle(s)
    gqa = h["gqa"]
    if s["op"] == "attend":
        gqa.tree_decode(s["q"], s["k"], s["v"], s["out"], num_kv_heads=s["hkv"], layout=h["layout"], seq_lens_dev=s["lens"], mask=s["mask"],
                        tree_sizes=s["sizes"], block_table=s["table"], workspace=h["workspace"])
        return s["out"]
    if s["op"] == "rope":
        gqa.rope_append(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], layout=h["layout"], seq_lens_dev=s["lens"], freq=s["freq"], q_out=s["q_out"],
                        style=s["style"], attn_factor=s["factor"], qk_weight=s["weight"], eps=EPS, depth=s["depth"], tree_sizes=s["sizes"],
                        block_table=s["table"])
        return s["q_out"], s["k"], s["v"]
    if s["op"] == "verify":
        gqa.tree_verify(s["target"], s["probs"], s["words"], s["parents"], s["u_accept"], s["u_sample"], path=s["path"], kept=s["kept"],
                        next_token=s["next"], tree_sizes=s["sizes"])
        return s["path"], s["kept"], s["next"]
    gqa.tree_commit(s["k"], s["v"], num_kv_heads=s["hkv"], layout=h["layout"], layers=s["layers"], seq_lens_dev=s["lens"], path=s["path"], kept=s["kept"],
                    seq_lens_out=s["new_lens"], tree_sizes=s["sizes"], block_table=s["table"])
    return s["k"], s["v"], s["new_lens"]


# ---- the plain forms ----------------------------------------------------------------------------

def _rows(s, cache):
    """The cache as [batch, hkv, positions, 128]."""
    if s["table"] is None:
        return cache.permute(0, 2, 1, 3)
    picked = cache[s["table"].long()]  # [batch, pages, hkv, block, 128]
    b, n, h, t, d = picked.shape
    return picked.permute(0, 2, 1, 3, 4).reshape(b, h, n * t, d)


def _attend(s):
    batch, tokens, hq, hkv = s["batch"], s["tokens"], s["hq"], s["hkv"]
    group = hq // hkv
    k, v = _rows(s, s["k"]).float(), _rows(s, s["v"]).float()
    length = k.shape[2]
    lens, sizes = s["lens"].long(), s["sizes"].long()
    base = (lens - sizes)[:, None, None]
    at = torch.arange(length, device=DEV)[None, None, :]
    node = torch.arange(tokens, device=DEV)
    inside = (at - base).clamp(0, tokens - 1).expand(batch, tokens, length)
    sees = (at < base) | ((at < lens[:, None, None]) & torch.gather(s["seen"], 2, inside))  # [batch, tokens, length]
    q = s["q"].float().view(batch, tokens, hkv, group, D).permute(0, 2, 1, 3, 4).reshape(batch, hkv, tokens * group, D)
    scores = (q @ k.transpose(-1, -2)).view(batch, hkv, tokens, group, length).mul_(D ** -0.5)
    scores.masked_fill_(~sees[:, None, :, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((at[0] < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = (p.view(batch, hkv, tokens * group, length) @ v).view(batch, hkv, tokens, group, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(batch, tokens, hq, D).to(s["q"].dtype)
    live = (node[None, :] < sizes[:, None])[:, :, None, None]
    s["out"].copy_(torch.where(live, o, s["out"]))
    return s["out"]


def _rotate(s, x, weight):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    start = (s["lens"] - s["sizes"]).double()
    theta = (start[:, None] + s["depth"].double())[:, :, None] * s["freq"]
    sin, cos = (theta.sin() * s["factor"]).float()[:, :, None], (theta.cos() * s["factor"]).float()[:, :, None]
    rotary, half = s["rotary"], s["rotary"] // 2
    y = x.clone()
    if s["style"] == "half":
        a, b = x[..., :half], x[..., half:rotary]
        y[..., :half], y[..., half:rotary] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _rope(s):
    weight = s["weight"]
    q = _rotate(s, s["q"], None if weight is None else weight[:D]).to(s["q"].dtype)
    k = _rotate(s, s["k_new"], None if weight is None else weight[D:]).to(s["k"].dtype)
    batch, tokens = s["batch"], s["tokens"]
    node = torch.arange(tokens, device=DEV)[None]
    live = node < s["sizes"][:, None]
    s["q_out"].copy_(torch.where(live[:, :, None, None], q, s["q_out"]))
    # Rows behind a tree's end are written where its last row goes, with that row's values.
    last = torch.minimum(node.expand(batch, tokens), s["sizes"][:, None] - 1).long()
    slot = (s["lens"] - s["sizes"])[:, None] + last
    seq = torch.arange(batch, device=DEV)[:, None]
    k, v = k[seq, last], s["v_new"][seq, last]
    if s["table"] is None:
        s["k"][0, slot[0].long()], s["v"][0, slot[0].long()] = k[0], v[0]
    else:
        block = s["block_tokens"]
        page = s["table"][seq, (slot // block).long()].long()
        s["k"][page, :, (slot % block).long()] = k
        s["v"][page, :, (slot % block).long()] = v
    return s["q_out"], s["k"], s["v"]


def _verify(s):
    batch, tokens, vocab = s["batch"], s["tokens"], s["vocab"]
    seq = torch.arange(batch, device=DEV)
    node = torch.zeros(batch, dtype=torch.long, device=DEV)
    used = torch.zeros(batch, dtype=torch.float64, device=DEV)
    left = torch.ones(batch, dtype=torch.float64, device=DEV)
    gone = torch.zeros((batch, vocab), dtype=torch.bool, device=DEV)
    kept = torch.ones(batch, dtype=torch.long, device=DEV)
    path = torch.full((batch, tokens + 1), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0

    def residual():
        p = s["target"][seq, node].double()
        if s["probs"] is not None:
            return (p - used[:, None] * s["probs"][seq, node].double()).clamp_(min=0.0)
        return torch.where(gone, torch.zeros_like(p), p)

    for t in range(1, tokens):  # the walk: each test depends on the one before
        tested = (s["parents"][:, t] == node) & (t < s["sizes"])
        word = s["words"][:, t].long()
        q = s["probs"][seq, node, word].double() if s["probs"] is not None else torch.ones_like(left)
        taken = tested & (s["u_accept"][:, t].double() * q * left < residual()[seq, word])
        refused = tested & ~taken
        path[seq, torch.where(taken, kept, torch.full_like(kept, tokens))] = t
        kept = kept + taken
        node = torch.where(taken, torch.full_like(node, t), node)
        used = torch.where(taken, torch.zeros_like(used), torch.where(refused, used + left, used))
        gone[seq, word] |= refused
        gone &= ~taken[:, None]
        left = torch.where(taken, torch.ones_like(left), torch.where(refused, residual().sum(-1), left))
    rest = residual()
    total = rest.sum(-1, keepdim=True)
    rest = torch.where(total > 0, rest, s["target"][seq, node].double())
    upto = rest.cumsum(-1)
    past = upto > s["u_sample"].double()[:, None] * rest.sum(-1, keepdim=True)
    s["path"].copy_(path[:, :tokens])
    s["kept"].copy_(kept)
    s["next"].copy_(past.int().argmax(-1))
    return s["path"], s["kept"], s["next"]


def _commit(s):
    tokens, block, layers = s["tokens"], s["block_tokens"], s["layers"]
    to = torch.arange(tokens, device=DEV)[None].expand(s["batch"], tokens)
    moves = to < s["kept"][:, None]
    # Rows that stay are written with their own values; slots past the tree's end stand for its last.
    to = torch.minimum(to, s["sizes"][:, None] - 1)
    start = (s["lens"] - s["sizes"])[:, None]
    src, dst = (start + torch.where(moves, s["path"], to)).long(), (start + to).long()
    seq = torch.arange(s["batch"], device=DEV)[:, None]
    every = torch.arange(layers, device=DEV)[:, None, None]

    def move(cache):
        cache = cache if layers > 1 else cache[None]
        if s["table"] is None:
            cache[every, 0, dst] = cache[every, 0, src]
        else:
            cache = cache.permute(0, 1, 3, 2, 4)
            cache[every, s["table"][seq, dst // block].long(), dst % block] = cache[every, s["table"][seq, src // block].long(), src % block]

    move(s["k"])
    move(s["v"])
    s["new_lens"].copy_(s["lens"] - s["sizes"] + s["kept"])
    return s["k"], s["v"], s["new_lens"]


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "rope": _rope, "verify": _verify, "commit": _commit}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op, batch, tokens = case["op"], case["batch"], case["tokens"]
    nodes = batch * tokens if batch == 1 else batch * (tokens - 0.25 * tokens)  # mean over the sizes
    if op == "attend":
        keys = batch * 0.5 * (case["lo"] + case["hi"])
        return {"bytes": keys * case["hkv"] * D * 4 + nodes * case["hq"] * D * 4, "flops": 4.0 * (nodes / batch) * case["hq"] * D * keys}
    if op == "rope":
        size = 4 if case["dtype"] == "fp32" else 2
        heads = case["hq"] + 2 * case["hkv"]
        return {"bytes": nodes * heads * D * 2 * size, "flops": nodes * (case["hq"] + case["hkv"]) * D * 7.0}
    if op == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = 2 if case["draft"] == "probs" else 1  # the last node's rows
        return {"bytes": float(batch * rows * case["vocab"] * size), "flops": batch * case["vocab"] * 3.0}
    size = 4 if case["dtype"] == "fp32" else 2
    moved = max(batch * (case["accepted"] - 1), 1)
    return {"bytes": float(moved * case["layers"] * case["hkv"] * D * size * 4), "flops": 0.0}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _place(s, b, slot):
    if s["table"] is None:
        return 0, slot
    return int(s["table"][b, slot // s["block_tokens"]]), slot % s["block_tokens"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "rope": _exact_rope, "verify": _exact_verify, "commit": _exact_commit}[s["op"]](s)


def _exact_attend(s):
    group = s["hq"] // s["hkv"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for b in range(s["batch"]):
        n, length = int(s["sizes_host"][b]), int(s["lens_host"][b])
        for h in range(s["hkv"]):
            if s["table"] is None:
                k, v = s["k"][0, :length, h], s["v"][0, :length, h]
            else:
                pages = s["table"][b].long()
                k, v = s["k"][pages, h].reshape(-1, D)[:length], s["v"][pages, h].reshape(-1, D)[:length]
            k, v = k.double(), v.double()
            q = s["q"][b, :n, h * group:(h + 1) * group].double()
            w = torch.einsum("tgd,ld->tgl", q, k) / math.sqrt(D)
            w[:, :, length - n:].masked_fill_(~s["seen"][b, :n, :n][:, None, :], -math.inf)
            out[b, :n, h * group:(h + 1) * group] = torch.einsum("tgl,ld->tgd", torch.softmax(w, -1), v)
    return out


def _exact_rope(s):
    weight, half = s["weight"], s["rotary"] // 2
    q, k, v = s["q_out"].double(), s["k"].double(), s["v"].double()
    for name, heads in (("q", s["hq"]), ("k_new", s["hkv"])):
        x = s[name].double()
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * weight.double()[(0 if name == "q" else D):][:D]
        turned = x.clone()
        pair = torch.arange(half, device=DEV)
        first, second = (pair, pair + half) if s["style"] == "half" else (2 * pair, 2 * pair + 1)
        where = torch.from_numpy(s["lens_host"] - s["sizes_host"]).to(DEV)[:, None] + s["depth"]
        turn = torch.polar(torch.full((half,), float(s["factor"]), dtype=torch.float64, device=DEV), torch.zeros(half, dtype=torch.float64, device=DEV))
        angle = where.double()[..., None] * s["freq"]
        z = torch.complex(x[..., first], x[..., second]) * (turn * torch.exp(1j * angle))[:, :, None]
        turned[..., first], turned[..., second] = z.real, z.imag
        for b in range(s["batch"]):
            n, length = int(s["sizes_host"][b]), int(s["lens_host"][b])
            if name == "q":
                q[b, :n] = turned[b, :n]
                continue
            for t in range(n):
                block, at = _place(s, b, length - n + t)
                if s["table"] is None:
                    k[block, at], v[block, at] = turned[b, t], s["v_new"][b, t].double()
                else:
                    k[block, :, at], v[block, :, at] = turned[b, t], s["v_new"][b, t].double()
    return q, k, v


def _exact_verify(s):
    batch, tokens = s["batch"], s["tokens"]
    path, kept, then = np.full((batch, tokens), -1, dtype=np.int32), np.zeros(batch, dtype=np.int32), np.zeros(batch, dtype=np.int32)
    parents, words = s["parents"].cpu().numpy(), s["words"].cpu().numpy()
    u, w = s["u_accept"].double().cpu().numpy(), s["u_sample"].double().cpu().numpy()
    for b in range(batch):
        node, way = 0, [0]
        while True:
            p = s["target"][b, node].double().cpu().numpy()
            q = s["probs"][b, node].double().cpu().numpy() if s["probs"] is not None else None
            step = None
            for t in range(node + 1, int(s["sizes_host"][b])):
                if parents[b, t] != node:
                    continue
                x = words[b, t]
                if u[b, t] * (q[x] if q is not None else 1.0) < p[x]:
                    step = t
                    break
                less = p - q if q is not None else np.where(np.arange(len(p)) == x, 0.0, p)
                less = np.maximum(less, 0.0)
                p = less / less.sum() if less.sum() > 0 else less
            if step is None:
                break
            node = step
            way.append(step)
        if not p.sum() > 0:
            p = s["target"][b, node].double().cpu().numpy()
        upto = np.cumsum(p)
        path[b, : len(way)], kept[b], then[b] = way, len(way), np.searchsorted(upto, w[b] * upto[-1], side="right")
    return _dev(path), _dev(kept), _dev(then)


def _exact_commit(s):
    k, v = s["k"].clone(), s["v"].clone()
    lens = np.zeros(s["batch"], dtype=np.int32)
    path, kept = s["path"].cpu().numpy(), s["kept"].cpu().numpy()
    for b in range(s["batch"]):
        start = int(s["lens_host"][b]) - int(s["sizes_host"][b])
        for i in range(int(kept[b])):
            (b0, t0), (b1, t1) = _place(s, b, start + int(path[b, i])), _place(s, b, start + i)
            for new, old in ((k, s["k"]), (v, s["v"])):
                if s["table"] is None:
                    new[..., b1, t1, :, :] = old[..., b0, t0, :, :]
                else:
                    new[..., b1, :, t1, :] = old[..., b0, :, t0, :]
        lens[b] = start + int(kept[b])
    return k.double(), v.double(), _dev(lens)

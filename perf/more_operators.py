"""The operators that check a tree of drafted tokens in one pass: a decode step that takes
several tokens per sequence instead of one.

* ``append``: ``kernels.paged_rope_append``, queries and keys rotated to their positions and
  the keys and values of several tokens per sequence stored in the paged cache.
* ``attend``: ``kernels.paged_tree_attention``, each drafted token over its sequence's cache,
  its ancestors and itself.
* ``sample``: ``kernels.sample_tokens``, a token from each row of logits with temperature,
  top-k, top-p and min-p, from given uniform numbers.
* ``accept``: ``kernels.accept_draft_tree``, the walk down the tree along the sampled tokens,
  and the kept tokens' keys and values closed up in the cache of every layer.

Heads, vocabularies and block size are those of the repository's configurations (Qwen2-1.5B:
12 / 2 heads, Qwen2-7B: 28 / 4), or generic.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

sys.path.insert(0, os.path.join(os.getcwd(), "grpo-training-engine_amd"))

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
MOST_APPEND = 8 * 2048 * 36 * 128  # values of the largest listed cases
MOST_PAIRS = 64 * 32 * 28 * 2500  # node, head, token
MOST_CACHE = 64 * 4096 * 4
MOST_LOGITS = 512 * 151936
MOST_MOVED = 28 * 64 * 4


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # a group of 8 that checks three drafted tokens each, float32 tables
        dict(name="append_8x4", kind="append", batch=8, nodes=4, hq=12, hkv=2, dim=128, block=16,
             dtype="bf16", table="f32", full=True),
        # trees of up to 61 nodes, some with fewer
        dict(name="append_32x61", kind="append", batch=32, nodes=61, hq=28, hkv=4, dim=128,
             block=16, dtype="f16", table="f16", full=False),
        # chunks of eight long prompts
        dict(name="append_8x2048", kind="append", batch=8, nodes=2048, hq=28, hkv=4, dim=128,
             block=16, dtype="bf16", table="bf16", full=True),
        # a group of 8, three drafted tokens each, short contexts
        dict(name="attend_8x4", kind="attend", batch=8, nodes=4, hq=12, hkv=2, dim=128, block=16,
             dtype="bf16", context=700, tree="chain", full=True),
        # one sequence's tree over a long context, of no round size
        dict(name="attend_1x61_long", kind="attend", batch=1, nodes=61, hq=28, hkv=4, dim=128,
             block=16, dtype="f16", context=30011, tree="random", full=True),
        # a group of 32 with trees of 16, ragged
        dict(name="attend_32x16", kind="attend", batch=32, nodes=16, hq=12, hkv=2, dim=128,
             block=16, dtype="bf16", context=1500, tree="random", full=False),
        # the larger model's group of 64 with trees of 32
        dict(name="attend_64x32", kind="attend", batch=64, nodes=32, hq=28, hkv=4, dim=128,
             block=16, dtype="bf16", context=2500, tree="random", full=True),
        # the newest token of a group of 8, the trainer's settings
        dict(name="sample_8", kind="sample", rows=8, vocab=151936, dtype="bf16", std=2.0,
             temperature=0.7, top_k=0, top_p=0.9, min_p=0.0),
        # float32 logits of a vocabulary of odd size, every filter, settings of each row's own
        dict(name="sample_37_f32", kind="sample", rows=37, vocab=50257, dtype="f32", std=1.5,
             temperature="rows", top_k="rows", top_p="rows", min_p="rows"),
        # every node of 32 trees of 16
        dict(name="sample_512", kind="sample", rows=512, vocab=151936, dtype="bf16", std=2.0,
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.02),
        # a group of 8, two chains of three tokens each, 28 layers
        dict(name="accept_8x7", kind="accept", batch=8, chains=2, depth=3, hkv=2, dim=128,
             block=16, layers=28, dtype="bf16"),
        # 64 sequences with trees of 61 nodes
        dict(name="accept_64x61", kind="accept", batch=64, chains=10, depth=6, hkv=4, dim=128,
             block=16, layers=28, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


HEADS = [(12, 2), (28, 4), (8, 8), (16, 2), (14, 2), (12, 1)]


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "sample", "sample", "accept"])
    hq, hkv = rng.choice(HEADS)
    dim, block = rng.choice([64, 128, 128]), rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        batch = _log_int(rng, 1, 64)
        most = MOST_APPEND // (2 * batch * (hq + 2 * hkv) * dim)
        return dict(kind=kind, batch=batch, nodes=_log_int(rng, 1, min(2048, most)), hq=hq,
                    hkv=hkv, dim=dim, block=block, dtype=dtype,
                    table=rng.choice(["f32", dtype]), full=rng.random() < 0.5)
    if kind == "attend":
        batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        most = min(MOST_PAIRS // (2 * batch * nodes * hq), MOST_CACHE // (2 * batch * hkv), 32000)
        return dict(kind=kind, batch=batch, nodes=nodes, hq=hq, hkv=hkv, dim=dim, block=block,
                    dtype=dtype, context=_log_int(rng, 16, most),
                    tree=rng.choice(["chain", "random", "random"]), full=rng.random() < 0.5)
    if kind == "sample":
        vocab = rng.choice([151936, 152064, 32000, 50257, _log_int(rng, 1000, 152064)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        rows = _log_int(rng, 1, min(512, MOST_LOGITS // (vocab * BYTES[dtype])))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype,
                    std=rng.choice([0.5, 1.5, 3.0]),
                    temperature=rng.choice([1.0, 0.7, "rows"]),
                    top_k=rng.choice([0, 0, 50, rng.randint(1, 1000), "rows"]),
                    top_p=rng.choice([1.0, 0.9, 0.95, "rows"]),
                    min_p=rng.choice([0.0, 0.0, 0.05, "rows"]))
    chains = rng.randint(1, 10)
    batch = rng.randint(1, 64)
    return dict(kind=kind, batch=batch, chains=chains, depth=rng.randint(1, 60 // chains),
                hkv=hkv, dim=dim, block=block,
                layers=rng.randint(1, max(1, min(28, MOST_MOVED // (2 * batch * hkv)))),
                dtype=dtype)


# ----------------------------------------------------------------- inputs --

MAX_POS = 32768


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _randint(g, lo, hi, shape):
    """Integers lo .. hi, both among them."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda")


def _tables(c, g, lens, spare):
    """(number of blocks, shuffled block table) for the sequences' longest length."""
    width = -(-(spare + lens) // c["block"])
    blocks = c["batch"] * width + 3
    at = torch.randperm(blocks, generator=g, device="cuda")[:c["batch"] * width]
    return blocks, at.view(c["batch"], width).int()


def _cache(c, g, blocks, *layers):
    shape = (*layers, blocks, c["hkv"], c["block"], c["dim"])
    dt = DTYPES[c["dtype"]]
    return _randn(g, *shape, dtype=dt), _randn(g, *shape, dtype=dt)


def _counts(c, g):
    """Nodes in use of each sequence: all of them, or from half of them on."""
    n = c["nodes"]
    return _randint(g, n if c["full"] else (n + 1) // 2, n, (c["batch"],)).int()


def _rotation(c):
    """cos and sin of Qwen2's angles, [positions, dim]."""
    half = torch.arange(0, c["dim"], 2, device="cuda").double() / c["dim"]
    a = torch.arange(MAX_POS, device="cuda").double()[:, None] * 1e6 ** -half
    a = torch.cat((a, a), 1)
    return a.cos().to(DTYPES[c["table"]]), a.sin().to(DTYPES[c["table"]])


def _parents(c, g):
    """Each node's parent, an earlier node (-1: none): a chain, or a tree whose nodes hang
    off any earlier one."""
    b, t = c["batch"], c["nodes"]
    at = torch.arange(t, device="cuda")
    if c["tree"] == "chain":
        return (at - 1).int().expand(b, t).contiguous()
    u = torch.rand(b, t, generator=g, device="cuda")
    return torch.where(at > 0, (u * at).floor().clamp(max=at - 1), -1).int()


def _accept_state(c, g):
    """Chains of drafted tokens off node 0, and the tokens that the model sampled at each
    node: along one chain the drafted ones, up to some depth."""
    b, n, depth = c["batch"], c["chains"], c["depth"]
    t = 1 + n * depth
    at = torch.arange(t, device="cuda")
    parents = torch.where((at - 1) % depth == 0, 0, at - 1)
    parents[0] = -1
    drafted = _randint(g, 0, 151935, (b, t))
    sampled = _randint(g, 151936, 152063, (b, t))  # no drafted token's id
    chain, good = _randint(g, 0, n - 1, (b,)), _randint(g, 0, depth, (b,))
    first = 1 + chain * depth
    for d in range(depth):
        node = (first + d - 1 if d else torch.zeros_like(first))[:, None]
        token = torch.where((good > d)[:, None], drafted.gather(1, first[:, None] + d),
                            sampled.gather(1, node))
        sampled.scatter_(1, node, token)
    lens = _randint(g, 40, 90, (b,)).int()
    blocks, table = _tables(c, g, 90, t)
    k, v = _cache(c, g, blocks, c["layers"])
    return dict(parents=parents.int().expand(b, t).contiguous(), drafted=drafted,
                sampled=sampled, lens=lens, table=table, k=k, v=v)


def _row_settings(c, g):
    """The settings that are each row's own, one tensor each."""
    m, dev = c["rows"], "cuda"
    s = {k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    u = torch.rand(4, m, generator=g, device=dev)
    if s["temperature"] == "rows":
        s["temperature"] = torch.where(u[0] < 0.2, 0.0, 0.4 + u[0])
    if s["top_k"] == "rows":
        s["top_k"] = torch.where(u[1] < 0.3, 0.0, u[1] * 400).int()
    if s["top_p"] == "rows":
        s["top_p"] = torch.where(u[2] < 0.2, 1.0, 0.5 + u[2] / 2)
    if s["min_p"] == "rows":
        s["min_p"] = torch.where(u[3] < 0.5, 0.0, u[3] / 10)
    return s


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c=c)
    if c["kind"] == "sample":
        dt = DTYPES[c["dtype"]]
        s["logits"] = _randn(g, c["rows"], c["vocab"], std=c["std"], dtype=dt)
        # some tokens stand out, as they do in a model's logits
        up = _randint(g, 0, c["vocab"] - 1, (c["rows"], 1))
        up = (up + torch.arange(32, device="cuda") * (c["vocab"] // 37)) % c["vocab"]
        height = torch.rand(up.shape, generator=g, device="cuda") * 6 * c["std"]
        s["logits"].scatter_(1, up, height.to(dt))
        s["draws"] = torch.rand(c["rows"], generator=g, device="cuda", dtype=torch.float64)
        s.update(_row_settings(c, g))
        return s
    if c["kind"] == "accept":
        s.update(_accept_state(c, g))
        return s
    dt, b, t, d = DTYPES[c["dtype"]], c["batch"], c["nodes"], c["dim"]
    s["counts"] = _counts(c, g)
    if c["kind"] == "append":
        most = min(300, MAX_POS - t)
        s["lens"] = _randint(g, 0, most, (b,)).int()
        s["positions"] = s["lens"][:, None] + torch.arange(t, device="cuda").int()
        blocks, s["table"] = _tables(c, g, most, t)
        # the rows of a projection that makes q, k and v together
        qkv = _randn(g, b, t, (c["hq"] + 2 * c["hkv"]) * d, dtype=dt).view(b, t, -1, d)
        s["q"], s["k_new"], s["v_new"] = qkv.split((c["hq"], c["hkv"], c["hkv"]), 2)
        s["cos"], s["sin"] = _rotation(c)
    else:
        n = c["context"]
        s["lens"] = _randint(g, n if b == 1 else n // 2, n if b == 1 else n + n // 2, (b,)).int()
        blocks, s["table"] = _tables(c, g, n + n // 2, t)
        s["parents"] = _parents(c, g)
        s["q"] = _randn(g, b, t, c["hq"], d, dtype=dt)
    s["k"], s["v"] = _cache(c, g, blocks)
    return s


# ------------------------------------------------------------- plain forms --

def _slots(table, block, slots):
    """(block id, place in the block) of slots [B, n] of each sequence."""
    slots = slots.long()
    return table.long().gather(1, slots // block), slots % block


def _plain_append(s):
    c, t, half = s["c"], s["c"]["nodes"], s["c"]["dim"] // 2
    at = torch.arange(t, device="cuda")
    used = (at < s["counts"][:, None])
    cos = s["cos"][s["positions"].long()].float()[:, :, None]
    sin = s["sin"][s["positions"].long()].float()[:, :, None]

    def turned(x):
        x = x.float()
        lo, hi = x[..., :half], x[..., half:]
        return torch.cat((lo * cos[..., :half] - hi * sin[..., :half],
                          hi * cos[..., half:] + lo * sin[..., half:]), -1)

    dt = s["q"].dtype
    q = torch.where(used[..., None, None], turned(s["q"]), 0.0).to(dt)
    blk, off = _slots(s["table"], c["block"], s["lens"][:, None] + at)
    keep = used[..., None, None]
    # unused rows store again what their slots hold
    s["k"][blk, :, off] = torch.where(keep, turned(s["k_new"]).to(dt), s["k"][blk, :, off])
    s["v"][blk, :, off] = torch.where(keep, s["v_new"], s["v"][blk, :, off])
    return [q, s["k"], s["v"]]


def _sees(parents):
    """[B, T, T]: node i has node j as ancestor, or is it."""
    b, t = parents.shape
    at = torch.arange(t, device=parents.device)
    m = (at[:, None] == at).expand(b, t, t)
    up = parents.long()
    for i in range(1, t):  # a parent's row is complete before its children's
        p = up[:, i].clamp(min=0)
        row = m[torch.arange(b, device=up.device), p] & (up[:, i] >= 0)[:, None]
        m = torch.cat((m[:, :i], (m[:, i] | row)[:, None], m[:, i + 1:]), 1)
    return m


def _plain_attend(s):
    c = s["c"]
    b, t, hq, hkv, d = c["batch"], c["nodes"], c["hq"], c["hkv"], c["dim"]
    most = c["context"] * (2 if b == 1 else 3) // 2 + t
    most = min(most, s["table"].shape[1] * c["block"])
    slot = torch.arange(most, device="cuda")
    blk, off = _slots(s["table"], c["block"], slot.expand(b, most))
    used = torch.arange(t, device="cuda") < s["counts"][:, None]
    node = slot - s["lens"][:, None]  # [B, most]
    tree = _sees(s["parents"]).gather(2, node.clamp(0, t - 1)[:, None].expand(b, t, most))
    on = (node < 0)[:, None] | (tree & ((node >= 0) & (node < t))[:, None])
    on = on & used[:, :, None]
    out = torch.empty(b, t, hq, d, device="cuda", dtype=s["q"].dtype)
    for lo in range(0, b, 8):  # some sequences at a time
        at = slice(lo, lo + 8)
        k = s["k"][blk[at], :, off[at]].float().permute(0, 2, 3, 1).contiguous()
        v = s["v"][blk[at], :, off[at]].float().permute(0, 2, 1, 3).contiguous()
        n = k.shape[0]
        q = s["q"][at].float().view(n, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)
        x = (q.reshape(n, hkv, -1, d) @ k) * (1 / math.sqrt(d))
        x = x.view(n, hkv, t, -1, most).masked_fill_(~on[at][:, None, :, None], -math.inf)
        e = (x - x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
        o = e.view(n, hkv, -1, most) @ v
        o = o / e.sum(-1).view(n, hkv, -1, 1).clamp(min=1e-30)
        o = o.view(n, hkv, t, -1, d).permute(0, 2, 1, 3, 4)
        out[at] = o.reshape(n, t, hq, d).to(out.dtype)
    return [out]


def _per_row(v, rows):
    """A setting as float64 [rows, 1]."""
    if not torch.is_tensor(v):
        v = torch.full((rows,), v, device="cuda", dtype=torch.float64)
    return v.double()[:, None]


def _plain_sample(s):
    m, v = s["logits"].shape
    t, k, p, least = (_per_row(s[n], m) for n in ("temperature", "top_k", "top_p", "min_p"))
    k = torch.where(t > 0, torch.where(k > 0, k, v), 1.0)
    x, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    # in 64 bits: sums over a vocabulary, and values next to the filters' borders
    x = x.double()
    w = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp_()
    rank = torch.arange(v, device="cuda")
    w = torch.where(rank < k, w, 0.0)
    mass = w.cumsum(1)
    keep = (rank < k) & (w >= least) & ((mass - w < p * mass[:, -1:]) | (rank == 0) | (p >= 1))
    kept = keep.sum(1)
    total = mass.gather(1, kept[:, None] - 1)
    pick = (mass <= s["draws"][:, None] * total).sum(1)
    pick = torch.minimum(pick, kept - 1)
    return [order.gather(1, pick[:, None])[:, 0], kept.int()]


def _plain_accept(s):
    c = s["c"]
    b, t = s["drafted"].shape
    at = torch.arange(t, device="cuda")
    cur = torch.zeros(b, 1, dtype=torch.int64, device="cuda")
    live = torch.ones(b, 1, dtype=torch.bool, device="cuda")
    path = torch.full((b, t), -1, dtype=torch.int64, device="cuda")
    tokens = torch.zeros(b, t, dtype=torch.int64, device="cuda")
    count = torch.zeros(b, 1, dtype=torch.int64, device="cuda")
    for step in range(c["depth"] + 1):
        token = s["sampled"].gather(1, cur)
        path[:, step] = torch.where(live, cur, -1)[:, 0]
        tokens[:, step] = torch.where(live, token, 0)[:, 0]
        count = count + live
        child = (s["parents"] == cur) & (s["drafted"] == token)
        live = live & child.any(1, keepdim=True)
        cur = torch.where(child, at, t).amin(1, keepdim=True).clamp(max=t - 1)
    source = torch.where(path >= 0, path, at)  # others stay where they are
    source, slot = source + s["lens"][:, None], at + s["lens"][:, None]
    blk, off = _slots(s["table"], c["block"], source)
    to_blk, to_off = _slots(s["table"], c["block"], slot)
    for x in (s["k"], s["v"]):
        x[:, to_blk, :, to_off] = x[:, blk, :, off]
    return [tokens, count[:, 0].int(), path.int(), s["k"], s["v"]]


# --------------------------------------------------------- the framework's --

def _own(s):
    from grpo_mi355x import kernels

    kind = s["c"]["kind"]
    if kind == "append":
        q = kernels.paged_rope_append(s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], s["k"],
                                      s["v"], s["table"], s["lens"], counts=s["counts"],
                                      positions=s["positions"])
        return [q, s["k"], s["v"]]
    if kind == "attend":
        return [kernels.paged_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"],
                                             s["parents"], counts=s["counts"])]
    if kind == "sample":
        return list(kernels.sample_tokens(s["logits"], s["draws"], temperature=s["temperature"],
                                          top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                          return_kept=True))
    tokens, count, path = kernels.accept_draft_tree(s["drafted"], s["parents"], s["sampled"],
                                                    s["lens"], s["k"], s["v"], s["table"])
    return [tokens, count, path, s["k"], s["v"]]


PLAIN = {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample,
         "accept": _plain_accept}


def run(state):
    return _own(state) if own else PLAIN[state["c"]["kind"]](state)


# -------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * BYTES[c["dtype"]], flops=6 * n)  # the weight, the sums
    size = BYTES[c["dtype"]]
    if c["kind"] == "accept":
        # the mean walk accepts half of a chain; the first token stays where it is
        moved = c["batch"] * c["depth"] / 2 * (c["chains"] - 1) / c["chains"]
        return dict(bytes=4 * moved * c["layers"] * c["hkv"] * c["dim"] * size
                    + 20 * c["batch"] * (1 + c["chains"] * c["depth"]), flops=0)
    n = c["batch"] * c["nodes"] * (1 if c["full"] else 0.75)
    if c["kind"] == "append":
        values = n * (c["hq"] + 2 * c["hkv"]) * c["dim"]
        return dict(bytes=2 * values * size, flops=3 * n * (c["hq"] + c["hkv"]) * c["dim"])
    tokens = c["batch"] * c["context"]
    return dict(bytes=size * c["dim"] * (2 * c["hkv"] * (tokens + n) + 2 * c["hq"] * n),
                flops=4 * c["hq"] * c["dim"] * n * c["context"])


# ------------------------------------------------- the definition, 64 bits --

def _exact_append(s):
    c = s["c"]
    half = c["dim"] // 2
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k, v = s["k"].double(), s["v"].double()
    place = torch.arange(c["block"] * s["table"].shape[1], device="cuda")
    for b in range(c["batch"]):
        n, first = int(s["counts"][b]), int(s["lens"][b])
        pos = s["positions"][b, :n].long()
        # a pair of values as one complex number, each half's table entries its own
        cs, sn = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
        at = place[first:first + n]
        blk, off = s["table"][b].long()[at // c["block"]], at % c["block"]
        for x, to in ((s["q"], None), (s["k_new"], k)):
            z = x[b, :n].double()
            swapped = torch.cat((-z[..., half:], z[..., :half]), -1)
            y = z * cs + swapped * sn
            if to is None:
                q[b, :n] = y
            else:
                to[blk, :, off] = y
        v[blk, :, off] = s["v_new"][b, :n].double()
    return [q, k, v]


def _exact_attend(s):
    c = s["c"]
    g = c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    parents, lens, counts = (s[n].tolist() for n in ("parents", "lens", "counts"))
    for b in range(c["batch"]):
        n, most = lens[b], lens[b] + c["nodes"]
        ids = s["table"][b].long()
        k = s["k"][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :most].double()
        v = s["v"][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :most].double()
        hidden = np.zeros((c["nodes"], c["nodes"]), bool)
        for i in range(c["nodes"]):
            j = i
            while j >= 0:
                hidden[i, j] = True
                j = parents[b][j]
        hidden = ~torch.from_numpy(hidden).cuda()
        for h in range(c["hkv"]):
            q = s["q"][b, :counts[b], h * g:(h + 1) * g].double()
            x = torch.matmul(q, k[h].t().contiguous()) / c["dim"] ** 0.5
            x[..., n:] = x[..., n:].masked_fill(hidden[:counts[b], None], -math.inf)
            out[b, :counts[b], h * g:(h + 1) * g] = torch.softmax(x, -1) @ v[h]
    return [out]


def _exact_sample(s):
    tokens, kept = [], []
    rows, vocab = s["logits"].shape

    def of(name, i):
        return float(s[name][i]) if torch.is_tensor(s[name]) else s[name]

    for i in range(rows):
        z = s["logits"][i].double()
        t = of("temperature", i)
        if t <= 0:
            tokens.append(int((z == z.max()).nonzero()[0]))
            kept.append(1)
            continue
        order = torch.argsort(-z, stable=True)
        k = int(of("top_k", i))
        if k > 0:
            order = order[:k]
        p = torch.softmax(z[order] / t, 0)
        n = len(p)
        if of("top_p", i) < 1:  # the shortest head that holds top_p of the mass
            n = int(torch.searchsorted(torch.cumsum(p, 0), of("top_p", i))) + 1
        n = max(1, min(n, int((p / p[0] >= of("min_p", i)).sum()), len(p)))
        c = torch.cumsum(p[:n], 0)
        at = int(torch.searchsorted(c, c[-1] * s["draws"][i], right=True))
        tokens.append(int(order[min(at, n - 1)]))
        kept.append(n)
    return [torch.tensor(tokens, device="cuda"),
            torch.tensor(kept, dtype=torch.int32, device="cuda")]


def _exact_accept(s):
    c = s["c"]
    b, t = s["drafted"].shape
    up, drafted, sampled = (s[n].tolist() for n in ("parents", "drafted", "sampled"))
    path, tokens, counts = np.full((b, t), -1), np.zeros((b, t), np.int64), []
    k, v = s["k"], s["v"]
    flat = s["table"].long()
    for i in range(b):
        walk, node = [], 0
        while node is not None:
            walk.append(node)
            want = sampled[i][node]
            node = next((j for j in range(t) if up[i][j] == node and drafted[i][j] == want), None)
        n = len(walk)
        path[i, :n], tokens[i, :n] = walk, [sampled[i][j] for j in walk]
        counts.append(n)
        at = torch.tensor(walk, device="cuda") + int(s["lens"][i])
        to = torch.arange(n, device="cuda") + int(s["lens"][i])
        for x in (k, v):
            x[:, flat[i][to // c["block"]], :, to % c["block"]] = \
                x[:, flat[i][at // c["block"]], :, at % c["block"]].clone()
    return [torch.from_numpy(tokens).cuda(), torch.tensor(counts, dtype=torch.int32).cuda(),
            torch.from_numpy(path).int().cuda(), k, v]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample,
            "accept": _exact_accept}[case["kind"]](s)

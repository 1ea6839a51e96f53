"""Float64 restatement of the operators that check a tree of drafted tokens (numpy)."""

from __future__ import annotations

import numpy as np


def parent_of(parents, i: int) -> int:
    """Node ``i``'s parent: an earlier node, or -1."""
    p = i - 1 if parents is None else int(parents[i])
    return p if 0 <= p < i else -1


def sees(parents, t: int) -> np.ndarray:
    """bool [t, t]: node i has node j as an ancestor, or is it."""
    m = np.eye(t, dtype=bool)
    for i in range(t):
        p = parent_of(parents, i)
        if p >= 0:
            m[i] |= m[p]
    return m


def slot_of(table, slot: int, block: int, num_blocks: int):
    """(block, place) of a sequence's slot, None where the table has no block for it."""
    if not 0 <= slot < len(table) * block:
        return None
    blk = int(table[slot // block])
    return (blk, slot % block) if 0 <= blk < num_blocks else None


def used_nodes(counts, b: int, t: int, context: int) -> int:
    n = t if counts is None else max(0, min(int(counts[b]), t))
    return 0 if context < 0 else n


def rotate(x, cos, sin):
    """x [..., D] by the table rows cos, sin [D]."""
    h = x.shape[-1] // 2
    return np.concatenate([x[..., :h] * cos[:h] - x[..., h:] * sin[:h],
                           x[..., h:] * cos[h:] + x[..., :h] * sin[h:]], -1)


def rope_append(q, k, v, cos, sin, kc, vc, tables, lens, counts=None, positions=None):
    """(rotated q, k cache, v cache), float64; the caches are copies."""
    b_, t_ = q.shape[:2]
    nb, _, bs, _ = kc.shape
    out, kc, vc = np.zeros(q.shape), kc.astype(np.float64), vc.astype(np.float64)
    for b in range(b_):
        for t in range(used_nodes(counts, b, t_, int(lens[b]))):
            pos = int(lens[b]) + t if positions is None else int(positions[b, t])
            pos = min(max(pos, 0), len(cos) - 1)
            out[b, t] = rotate(q[b, t], cos[pos], sin[pos])
            at = slot_of(tables[b], int(lens[b]) + t, bs, nb)
            if at:
                kc[at[0], :, at[1]] = rotate(k[b, t], cos[pos], sin[pos])
                vc[at[0], :, at[1]] = v[b, t]
    return out, kc, vc


def tree_attention(q, kc, vc, tables, lens, parents=None, counts=None, scale=None):
    """(out, per value the attended |v| weighted as v is): float64 [B, T, Hq, D] both."""
    b_, t_, hq, d = q.shape
    nb, hkv, bs, _ = kc.shape
    scale = 1 / np.sqrt(d) if scale is None else scale
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(b_):
        n = int(lens[b])
        up = None if parents is None else parents[b]
        tree = sees(up, t_)
        for t in range(used_nodes(counts, b, t_, n)):
            slots = [*range(n), *(n + j for j in range(t_) if tree[t, j])]
            at = [s for s in (slot_of(tables[b], s, bs, nb) for s in slots) if s]
            if not at:
                continue
            blk, off = np.array(at).T
            for h in range(hq):
                g = h // (hq // hkv)
                x = kc[blk, g, off] @ q[b, t, h] * scale
                w = np.exp(x - x.max())
                out[b, t, h] = w @ vc[blk, g, off] / w.sum()
                size[b, t, h] = w @ np.abs(vc[blk, g, off]) / w.sum()
    return out, size


def accept(drafted, parents, sampled, lens, kc, vc, tables, counts=None, eos=None, pad=0):
    """(tokens, accepted, path, k cache, v cache); caches [layers, ...], copies."""
    b_, t_ = drafted.shape
    _, nb, _, bs, _ = kc.shape
    kc, vc = kc.copy(), vc.copy()
    tokens, path = np.full((b_, t_), pad, np.int64), np.full((b_, t_), -1, np.int32)
    accepted = np.zeros(b_, np.int32)
    for b in range(b_):
        n, walk = used_nodes(counts, b, t_, int(lens[b])), []
        cur = 0 if n else -1
        while cur >= 0:
            walk.append(cur)
            want = int(sampled[b, cur])
            child = [j for j in range(n) if parent_of(parents[b], j) == cur
                     and int(drafted[b, j]) == want]
            cur = child[0] if child and want >= 0 and want != eos else -1
        accepted[b] = len(walk)
        moved = []
        for j, i in enumerate(walk):
            tokens[b, j], path[b, j] = sampled[b, i], i
            src = slot_of(tables[b], int(lens[b]) + i, bs, nb)
            dst = slot_of(tables[b], int(lens[b]) + j, bs, nb)
            if src and dst:
                moved.append((dst, kc[:, src[0], :, src[1]].copy(), vc[:, src[0], :, src[1]].copy()))
        for (blk, off), k, v in moved:
            kc[:, blk, :, off], vc[:, blk, :, off] = k, v
    return tokens, accepted, path, kc, vc


def sample(x, u: float, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, kept tokens) of one row of logits."""
    x = np.asarray(x, dtype=np.float64)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0
    top = x[order[0]]
    if not temperature > 0 or top_p <= 0 or min_p > 1:
        return int(order[0]), 1
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(x[order] == top, 0.0, (x[order] - top) / temperature))
    mass = np.cumsum(w)
    n = len(order)
    if top_p < 1:
        n = min(n, int(np.searchsorted(mass, top_p * mass[-1])) + 1)
    if min_p > 0:
        n = min(n, int((w >= min_p).sum()))
    n = max(n, 1)
    at = int(np.searchsorted(mass[:n], u * mass[n - 1], side="right"))
    return int(order[min(at, n - 1)]), n

"""The policy update's operators in float64 numpy.

``token_logprobs`` and ``policy_loss`` with their gradients, restating the log-softmax of
the reference's fused loss (``src/triton_kernels/grpo_loss.py:47-139``) and its
two-sided clipped objective (``src/grpo/algorithm.py:115-254``) from their formulas, and
the counter-based dropout mask (Philox4x32-10, Salmon et al. 2011).
"""

from __future__ import annotations

import numpy as np


def token_logprobs(logits, ids, mask, temperature=1.0):
    """(logp, entropy, softmax) of float64 logits [R, V]; 0 in rows not counted."""
    rows, vocab = logits.shape
    logp, ent = np.zeros(rows), np.zeros(rows)
    p = np.zeros((rows, vocab))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if not mask[r]:
                continue
            z = np.asarray(logits[r], np.float64) / temperature
            z = z - z.max()
            lse = np.log(np.exp(z).sum())
            p[r] = np.exp(z - lse)
            logp[r] = z[ids[r]] - lse if 0 <= ids[r] < vocab else np.nan
            ent[r] = -np.sum(np.where(p[r] > 0, p[r] * (z - lse), 0.0)) if not np.isnan(
                lse) else np.nan
    return logp, ent, p


def logits_grad(p, ids, mask, coef, temperature=1.0):
    """coef / T (1[v = id] - p) per row, 0 in rows not counted."""
    g = np.zeros_like(p)
    for r in range(p.shape[0]):
        if mask[r]:
            g[r] = -p[r] * (coef[r] / temperature)
            if 0 <= ids[r] < p.shape[1]:
                g[r, ids[r]] += coef[r] / temperature
    return g


def policy_loss(logp, old, adv, mask, ref=None, eps_low=0.2, eps_high=0.2, delta=np.inf,
                beta=0.0, normalizer="tokens"):
    """(loss, metrics[4], d loss / d logp) over [B, S]; old None: logp itself."""
    logp = np.asarray(logp, np.float64)
    old = logp if old is None else np.asarray(old, np.float64)
    adv = np.asarray(adv, np.float64)
    adv = np.broadcast_to(adv[:, None] if adv.ndim == 1 else adv, logp.shape)
    total, sums, grad = 0.0, np.zeros(4), np.zeros(logp.shape)
    tokens, seqs = int(mask.sum()), int(mask.any(1).sum())
    for b, s in zip(*np.nonzero(mask)):
        w = 1 / normalizer if not isinstance(normalizer, str) else 1 / tokens \
            if normalizer == "tokens" else 1 / (mask[b].sum() * seqs)
        r, a = np.exp(logp[b, s] - old[b, s]), adv[b, s]
        free, clip = min(r, delta) * a, min(max(r, 1 - eps_low), 1 + eps_high) * a
        inside = 1 - eps_low <= r <= 1 + eps_high
        moves = (free <= clip and r <= delta) or (clip <= free and inside)
        d, kl = -a * r if moves else 0.0, 0.0
        if ref is not None:
            q = ref[b, s] - logp[b, s]
            kl = np.exp(q) - q - 1
            d = d + beta * (1 - np.exp(q))
        total += w * (beta * kl - min(free, clip))
        sums += (r, 0.0 if moves else 1.0, kl, old[b, s] - logp[b, s])
        grad[b, s] = w * d
    return total, sums / max(tokens, 1), grad


def philox(counter, key):
    """The four words of each Philox4x32-10 block: counter [n, 4], key (2) of uint32."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(counter)[:, i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low,
             (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype(np.uint32)


def dropout_factors(numel, p, seed, offset):
    """What each of ``numel`` elements is multiplied by: 0 or 65536 / (65536 - t)."""
    t = int(np.floor(p * 65536 + 0.5))
    seed, offset = int(seed) % 2 ** 64, int(offset) % 2 ** 64
    i = np.arange(-(-numel // 8), dtype=np.uint64)
    ctr = np.stack([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32),
                    np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)], 1)
    w = philox(ctr, (seed & 0xFFFFFFFF, seed >> 32))
    u = np.stack([w & 0xFFFF, w >> 16], 2).reshape(-1)[:numel]
    return np.where(u >= t, 65536.0 / (65536 - t), 0.0)

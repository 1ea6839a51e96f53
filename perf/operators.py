"""The operators of a policy update: what stands between the rollout's tokens and the
gradients of the LoRA layers.

* ``logp``: ``kernels.token_logprobs``, the log-probabilities of given tokens under a
  vocabulary of logits, with the entropy of each position, alone (the old and the
  reference policy) or with the logits' gradient.
* ``policy``: ``kernels.grpo_policy_loss``, the clipped policy loss with a KL term over
  per-token log-probabilities, and its gradient.
* ``loss``: ``kernels.fused_grpo_loss``, that loss straight from the logits, and their gradient.
* ``dropout``: ``kernels.counter_dropout``, dropout whose mask comes from a counter-based
  generator and is never stored, forward and backward.
* ``lora``: ``kernels.lora_fused_forward`` with that dropout on the adapter's input, forward
  and backward (gradients of the input and of both adapters).

Vocabularies and widths are those of the repository's configurations (Qwen2-1.5B and
Qwen2-7B), or generic.
"""

from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

sys.path.insert(0, os.path.join(os.getcwd(), "grpo-training-engine_amd"))

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS_LOW, EPS_HIGH, DELTA = 0.2, 0.28, 4.0
MOST_LOGITS = 8 * 512 * 151936  # values of the largest listed case
MOST_TOKENS = 64 * 4096
MOST_DROPOUT = 16384 * 3584


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # the log-probability of the newest token of a group of 8
        dict(name="logp_8", kind="logp", batch=8, seq=1, vocab=151936, dtype="bf16",
             temperature=0.7, fill=1.0, train=False),
        # the old policy's over the responses of a group of 8, of no round length
        dict(name="logp_3992", kind="logp", batch=8, seq=499, vocab=151936, dtype="bf16",
             temperature=1.0, fill=0.75, train=False),
        # trained through, float32 logits, rows at odd addresses
        dict(name="logp_train_f32", kind="logp", batch=3, seq=331, vocab=50257, dtype="f32",
             temperature=1.0, fill=0.75, train=True),
        # the loss of a group of 8 whose log-probabilities are there already
        dict(name="policy_4096", kind="policy", batch=8, seq=512, beta=0.04,
             normalizer="tokens", fill=0.75),
        # ... of 64 long responses
        dict(name="policy_262144", kind="policy", batch=64, seq=4096, beta=0.04,
             normalizer="sequences", fill=0.75),
        # a micro-batch of 4 short sequences, no reference policy
        dict(name="loss_256", kind="loss", batch=4, seq=64, vocab=151936, dtype="bf16",
             temperature=1.0, beta=0.0, normalizer="tokens", fill=0.75),
        # ragged responses over a small vocabulary of odd size
        dict(name="loss_1665_f16", kind="loss", batch=5, seq=333, vocab=32003, dtype="f16",
             temperature=0.7, beta=0.04, normalizer="sequences", fill=0.75),
        # a whole group of 8
        dict(name="loss_4096", kind="loss", batch=8, seq=512, vocab=151936, dtype="bf16",
             temperature=1.0, beta=0.04, normalizer="tokens", fill=0.75),
        # one layer's input of 8 tokens
        dict(name="dropout_8", kind="dropout", rows=8, cols=1536, dtype="bf16", p=0.05),
        # ... of a group's whole batch at the larger model
        dict(name="dropout_16384", kind="dropout", rows=16384, cols=3584, dtype="bf16", p=0.1),
        # a projection of a micro-batch of 4 short sequences
        dict(name="lora_256", kind="lora", batch=4, seq=64, inp=1536, out=1536, rank=16,
             dtype="bf16", p=0.05),
        # ... of a group of 8 at the larger model
        dict(name="lora_4184", kind="lora", batch=8, seq=523, inp=3584, out=3584, rank=16,
             dtype="bf16", p=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_logits(rng):
    vocab = rng.choice([151936, 152064, 32000, 50257, _log_int(rng, 1000, 152064)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    batch, most = rng.randint(1, 8), MOST_LOGITS * 2 // (vocab * BYTES[dtype])
    return dict(batch=batch, seq=_log_int(rng, 1, max(1, min(1024, most // batch))),
                vocab=vocab, dtype=dtype, temperature=rng.choice([1.0, 0.7]),
                fill=rng.choice([0.6, 0.75, 0.9]))


def draw(rng):
    kind = rng.choice(["logp", "logp", "policy", "loss", "loss", "loss", "dropout", "lora",
                       "lora"])
    if kind == "logp":
        return dict(kind=kind, train=rng.random() < 0.5, **_draw_logits(rng))
    if kind == "loss":
        return dict(kind=kind, beta=rng.choice([0.0, 0.04]),
                    normalizer=rng.choice(["tokens", "sequences"]), **_draw_logits(rng))
    if kind == "policy":
        batch = _log_int(rng, 1, 256)
        return dict(kind=kind, batch=batch, seq=_log_int(rng, 1, min(4096, MOST_TOKENS // batch)),
                    beta=rng.choice([0.0, 0.04]), normalizer=rng.choice(["tokens", "sequences"]),
                    fill=rng.choice([0.6, 0.75, 0.9]))
    if kind == "dropout":
        cols = _log_int(rng, 1, 18944)
        return dict(kind=kind, rows=_log_int(rng, 1, min(16384, MOST_DROPOUT // (2 * cols))),
                    cols=cols, dtype=rng.choice(["bf16", "f16", "f32"]),
                    p=rng.choice([0.05, 0.1, 0.5]))
    return dict(kind=kind, batch=rng.randint(1, 8), seq=_log_int(rng, 16, 523),
                inp=32 * rng.randint(16, 112), out=32 * rng.randint(8, 112),
                rank=rng.choice([8, 16, 32]), dtype=rng.choice(["bf16", "bf16", "f16"]),
                p=rng.choice([0.05, 0.1, 0.5]))


# ----------------------------------------------------------------- inputs --

NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453,
       -0.28444138169288635, -0.18477343022833234, -0.09105003625154495, 0.0,
       0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
       0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
QB = 64  # NF4 blocksize


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _mask(c, g):
    """Counted positions: the first U[2 fill - 1, 1] of each row (a response and its padding)."""
    b, s = c["batch"], c["seq"]
    u = torch.rand(b, 1, generator=g, device="cuda")
    n = ((2 * c["fill"] - 1 + 2 * (1 - c["fill"]) * u) * s).ceil().clamp(1, s)
    return torch.arange(s, device="cuda")[None, :] < n


def _logits_state(c, g):
    """Logits of a rollout's positions, each sampled token well above the noise, and the
    token ids (-100 where nothing is counted)."""
    b, s, v, dt = c["batch"], c["seq"], c["vocab"], DTYPES[c["dtype"]]
    mask = _mask(c, g)
    ids = torch.randint(0, v, (b, s), generator=g, device="cuda")
    logits = _randn(g, b, s, v, std=2.0, dtype=dt)
    up = torch.rand(b, s, 1, generator=g, device="cuda") * 12 + 4
    logits.scatter_add_(2, ids[..., None], up.to(dt))
    return logits, ids.masked_fill(~mask, -100), mask


def _old_logps(c, g, logits, ids, mask):
    """The log-probabilities under a policy a few updates older, and the reference's."""
    z = logits.float() / c["temperature"]
    logp = z.gather(2, ids.clamp(min=0)[..., None])[..., 0] - z.logsumexp(2)
    shape = logp.shape
    old = logp + _randn(g, *shape, std=0.1)
    ref = logp + _randn(g, *shape, std=0.2) if c["beta"] else None
    return old.masked_fill(~mask, 0.0), None if ref is None else ref.masked_fill(~mask, 0.0)


def _weight(g, n, k, std=0.02):
    """Packed bytes and float32 absmax of a random [n, k] weight, quantized to NF4."""
    blocks = _randn(g, n * k // QB, QB, std=std)
    absmax = blocks.abs().amax(1)
    code = torch.tensor(NF4, device="cuda")
    q = torch.bucketize(blocks / absmax[:, None], (code[1:] + code[:-1]) / 2).to(torch.uint8)
    q = q.view(-1)
    return ((q[0::2] << 4) | q[1::2]).view(-1, 1), absmax, code


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c=c)
    if c["kind"] in ("logp", "loss"):
        logits, ids, mask = _logits_state(c, g)
        s.update(logits=logits, ids=ids, mask=mask)
        if c["kind"] == "loss":
            s["old"], s["ref"] = _old_logps(c, g, logits, ids, mask)
            s["adv"] = _randn(g, c["batch"])
            logits.requires_grad_()
        elif c["train"]:
            s["grad"] = _randn(g, c["batch"], c["seq"])
            logits.requires_grad_()
    elif c["kind"] == "policy":
        shape = (c["batch"], c["seq"])
        s["logps"] = -2.0 * torch.rand(shape, generator=g, device="cuda") ** 2
        s["old"] = s["logps"] + _randn(g, *shape, std=0.2)
        s["ref"] = s["logps"] + _randn(g, *shape, std=0.3) if c["beta"] else None
        s["adv"], s["mask"] = _randn(g, c["batch"]), _mask(c, g)
        s["logps"].requires_grad_()
    elif c["kind"] == "dropout":
        dt = DTYPES[c["dtype"]]
        s["x"] = _randn(g, c["rows"], c["cols"], dtype=dt).requires_grad_()
        s["grad"] = _randn(g, c["rows"], c["cols"], std=0.1, dtype=dt)
        s["rng"] = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda")
    else:
        dt, k, n, r = DTYPES[c["dtype"]], c["inp"], c["out"], c["rank"]
        packed, absmax, code = _weight(g, n, k)
        packed.quant_state = SimpleNamespace(absmax=absmax, code=code, blocksize=QB,
                                             shape=(n, k), nested=False)
        s["base"] = SimpleNamespace(weight=packed, bias=None)
        s["a"] = _randn(g, r, k, std=0.02, dtype=dt).requires_grad_()
        s["b"] = _randn(g, n, r, std=0.02, dtype=dt).requires_grad_()
        s["x"] = _randn(g, c["batch"], c["seq"], k, dtype=dt).requires_grad_()
        s["grad"] = _randn(g, c["batch"], c["seq"], n, std=0.1, dtype=dt)
        s["rng"] = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda")
        s["dropout"] = torch.nn.Dropout(c["p"])
    return s


# ------------------------------------------------------------- plain forms --

def _softmax_parts(s):
    """exp(x/T - max), its float64 sum, and the float64 log-probability of each id."""
    t = s["c"]["temperature"]
    x = s["logits"].detach().float()
    top = x.amax(-1, keepdim=True)
    e = ((x - top) / t).exp()
    total = e.sum(-1, dtype=torch.float64)
    at = x.gather(-1, s["ids"].clamp(min=0)[..., None])[..., 0]
    logp = (at.double() - top[..., 0].double()) / t - total.log()
    return x, top, e, total, torch.where(s["mask"], logp, 0.0)


def _logits_grad(s, e, total, coef):
    """coef/T (1[v = id] - p_v), rounded to the logits' type."""
    k = torch.where(s["mask"], coef, 0.0) / s["c"]["temperature"]
    g = e * (-k / total).float()[..., None]
    g.scatter_add_(-1, s["ids"].clamp(min=0)[..., None], k.float()[..., None])
    return torch.where(s["mask"][..., None], g, 0.0).to(s["logits"].dtype)


def _plain_logp(s):
    x, top, e, total, logp = _softmax_parts(s)
    mean = (e * (x - top)).sum(-1, dtype=torch.float64) / total / s["c"]["temperature"]
    entropy = torch.where(s["mask"], total.log() - mean, 0.0)
    out = [logp.float(), entropy.float()]
    if s["c"]["train"]:
        out.append(_logits_grad(s, e, total, s["grad"].double()))
    return out


def _plain_policy(s, logp):
    """Loss, metrics (mean ratio, clipped share, mean KL, mean old - new) and the loss's
    derivative by each logp, in float64: the ratios stand next to the clip's borders."""
    c, mask = s["c"], s["mask"]
    diff = torch.where(mask, logp - s["old"].double(), 0.0)
    ratio, a = diff.exp(), s["adv"].double()[:, None]
    capped, clipped = ratio.clamp(max=DELTA), ratio.clamp(1 - EPS_LOW, 1 + EPS_HIGH)
    gain = torch.minimum(capped * a, clipped * a)
    free = (ratio * a <= clipped * a) & (ratio <= DELTA)
    free = free | (clipped == ratio)
    d = torch.where(free, -ratio * a, 0.0)
    kl = torch.zeros_like(gain)
    if s["ref"] is not None:
        lr = torch.where(mask, s["ref"].double() - logp, 0.0)
        kl = lr.exp() - lr - 1
        d = d + c["beta"] * (1 - lr.exp())
    n = mask.sum(1, keepdim=True).double()
    w = mask / n.sum() if c["normalizer"] == "tokens" else \
        mask / n.clamp(min=1) / (n > 0).sum()
    loss = ((c["beta"] * kl - gain) * w).sum()
    share = mask / n.sum()
    metrics = torch.stack([(v * share).sum() for v in (ratio, (~free).double(), kl, -diff)])
    return loss.float(), metrics.float(), d * w


def _plain_loss(s):
    _, _, e, total, logp = _softmax_parts(s)
    loss, metrics, coef = _plain_policy(s, logp)
    return [loss, logp.float(), metrics, _logits_grad(s, e, total, coef)]


def _philox(rng, count):
    """[count, 8] 16-bit draws: Philox4x32-10 (Salmon et al. 2011), counter (i, offset),
    key seed. 32-bit words in int64; a product's high word from 16-bit halves."""
    low = 0xFFFFFFFF
    i = torch.arange(count, device="cuda")
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    c0, c1 = i & low, i >> 32
    c2, c3 = (rng[1] & low).expand_as(i), ((rng[1] >> 32) & low).expand_as(i)
    for _ in range(10):
        h0 = (c0 * 0xD251 + (c0 * 0x1F53 >> 16)) >> 16
        h1 = (c2 * 0xCD9E + (c2 * 0x8D57 >> 16)) >> 16
        l0, l1 = (c0 * 0xD2511F53) & low, (c2 * 0xCD9E8D57) & low
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([w & 0xFFFF, w >> 16], 2).view(count, 8)


def _plain_drop(x, p, rng):
    """x where the draw of its place is kept, scaled, in float32."""
    n, t = x.numel(), round(p * 65536)
    keep = (_philox(rng, -(-n // 8)).view(-1)[:n] >= t).view(x.shape)
    return torch.where(keep, x.float() * (65536 / (65536 - t)), 0.0)


def _plain_dropout(s):
    x, p = s["x"].detach(), s["c"]["p"]
    return [_plain_drop(x, p, s["rng"]).to(x.dtype),
            _plain_drop(s["grad"], p, s["rng"]).to(x.dtype)]


def _plain_lora(s):
    c, w = s["c"], s["base"].weight
    q = torch.stack([w.view(-1) >> 4, w.view(-1) & 15], 1).view(-1, QB).long()
    st = w.quant_state
    x, a, b = (s[n].detach().float() for n in ("x", "a", "b"))
    # the weight's values are those of the 16-bit type
    weight = (st.code[q] * st.absmax[:, None]).to(s["x"].dtype).float().view(st.shape)
    x, g = x.view(-1, c["inp"]), s["grad"].float().view(-1, c["out"])
    scaling, t = 2.0, round(c["p"] * 65536)
    keep = (_philox(s["rng"], x.numel() // 8).view(x.shape) >= t).float()
    keep = keep * (65536 / (65536 - t))
    xd = x * keep
    xa, gb = xd @ a.T, (g * scaling) @ b
    y = x @ weight.T + scaling * (xa @ b.T)
    gx = g @ weight + (gb @ a) * keep
    out = [y.view(*s["x"].shape[:2], -1), gx.view(s["x"].shape), gb.T @ xd,
           scaling * (g.T @ xa)]
    return [v.to(s["x"].dtype) for v in out]


# --------------------------------------------------------- the framework's --

def _own(s):
    from grpo_mi355x import kernels

    c = s["c"]
    clip = dict(eps_low=EPS_LOW, eps_high=EPS_HIGH, delta=DELTA, beta=c.get("beta", 0.0),
                normalizer=c.get("normalizer", "tokens"))
    if c["kind"] == "logp":
        logp, entropy = kernels.token_logprobs(s["logits"], s["ids"], s["mask"],
                                               temperature=c["temperature"],
                                               return_entropy=True)
        if not c["train"]:
            return [logp, entropy]
        return [logp.detach(), entropy, *torch.autograd.grad(logp, s["logits"], s["grad"])]
    if c["kind"] == "policy":
        loss, metrics = kernels.grpo_policy_loss(s["logps"], s["old"], s["adv"], s["mask"],
                                                 ref_logps=s["ref"], **clip)
        return [loss.detach(), metrics, *torch.autograd.grad(loss, s["logps"])]
    if c["kind"] == "loss":
        loss, logp, metrics = kernels.fused_grpo_loss(
            s["logits"], s["ids"], s["old"], s["adv"], s["mask"], ref_logps=s["ref"],
            temperature=c["temperature"], **clip)
        return [loss.detach(), logp, metrics, *torch.autograd.grad(loss, s["logits"])]
    if c["kind"] == "dropout":
        y = kernels.counter_dropout(s["x"], c["p"], s["rng"])
        return [y.detach(), *torch.autograd.grad(y, s["x"], s["grad"])]
    y = kernels.lora_fused_forward(s["x"], base_layer=s["base"], lora_A=s["a"], lora_B=s["b"],
                                   scaling=2.0, dropout=s["dropout"], dropout_rng=s["rng"])
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["grad"])]


def run(state):
    if own:
        return _own(state)
    kind = state["c"]["kind"]
    if kind == "logp":
        return _plain_logp(state)
    if kind == "policy":
        loss, metrics, d = _plain_policy(state, state["logps"].detach().double())
        return [loss, metrics, d.float()]
    if kind == "loss":
        return _plain_loss(state)
    return _plain_dropout(state) if kind == "dropout" else _plain_lora(state)


# -------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] in ("logp", "loss"):
        rows = c["batch"] * c["seq"]
        read = c["fill"] * rows * c["vocab"]  # rows that are not counted are not read
        train = c["kind"] == "loss" or c["train"]
        size = BYTES[c["dtype"]]
        # x - max, exp, sum, entropy; then the softmax times its row's factor
        return dict(bytes=read * size + (rows * c["vocab"] * size if train else 0) + 24 * rows,
                    flops=read * (9 if train else 6))
    if c["kind"] == "policy":
        n = c["batch"] * c["seq"]
        return dict(bytes=n * (13 + (4 if c["beta"] else 0)), flops=20 * n)
    if c["kind"] == "dropout":
        n = c["rows"] * c["cols"]
        return dict(bytes=4 * n * BYTES[c["dtype"]], flops=2 * n)
    m, n, k, r = c["batch"] * c["seq"], c["out"], c["inp"], c["rank"]
    moved = n * k / 2 + n * k / QB * 4 + 2 * (2 * m * k + 2 * m * n + 2 * r * (n + k))
    return dict(bytes=moved, flops=2 * m * (2 * n * k + 3 * r * (n + k)))


# ------------------------------------------------- the definition, 64 bits --

def _draws(rng, count):
    """Philox4x32-10 in numpy's unsigned integers: [count * 8] 16-bit draws."""
    seed, offset = (int(v) & (2 ** 64 - 1) for v in rng.tolist())
    low = np.uint64(0xFFFFFFFF)
    i = np.arange(count, dtype=np.uint64)
    ctr = [i & low, i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF),
           np.full_like(i, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(q >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), q & low,
               (p >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(ctr, 1).astype(np.uint32)
    return torch.from_numpy(words.view(np.uint16).astype(np.int32).reshape(-1)).cuda()


def _exact_policy(s, logp):
    """Loss and metrics of float64 log-probabilities, differentiable."""
    c, mask, adv = s["c"], s["mask"], s["adv"].double().unsqueeze(1)
    count = mask.double().sum(1)
    total = logp.new_zeros(())
    sums = [0.0, 0.0, 0.0, 0.0]
    for row in range(c["batch"]):
        at = mask[row].nonzero()[:, 0]
        if not len(at):
            continue
        lp, a = logp[row, at], adv[row]
        r = torch.exp(lp - s["old"][row, at].double())
        bound = torch.where(a >= 0, torch.full_like(a, 1 + EPS_HIGH),
                            torch.full_like(a, 1 - EPS_LOW))
        # the pessimistic one of the two gains is r a up to the border on its side
        stopped = (r > bound) if a >= 0 else (r < bound)
        gain = torch.where(stopped, bound, r) * a
        capped = ~stopped & (r > DELTA)
        gain = torch.where(capped, torch.full_like(r, DELTA) * a, gain)
        term = -gain
        if s["ref"] is not None:
            q = s["ref"][row, at].double() - lp
            kl = torch.expm1(q) - q
            term = term + c["beta"] * kl
            sums[2] += float(kl.sum())
        sums[0] += float(r.sum())
        sums[1] += float((stopped | capped).sum())
        sums[3] += float((s["old"][row, at].double() - lp).sum())
        part = term.sum()
        total = total + (part if c["normalizer"] == "tokens" else part / count[row])
    total = total / (count.sum() if c["normalizer"] == "tokens" else (count > 0).sum())
    return total, torch.tensor(sums, dtype=torch.float64, device="cuda") / count.sum()


def exact(case, seed):
    s = prepare(case, seed)
    c, kind = case, case["kind"]
    if kind in ("logp", "loss"):
        z = s["logits"].detach().double().requires_grad_()
        logq = torch.log_softmax(z / c["temperature"], dim=-1)
        picked = logq.gather(-1, s["ids"].clamp(min=0).unsqueeze(-1)).squeeze(-1)
        picked = picked.masked_fill(~s["mask"], 0.0)
        if kind == "loss":
            loss, metrics = _exact_policy(s, picked)
            return [loss.detach(), picked.detach(), metrics, *torch.autograd.grad(loss, z)]
        entropy = -(logq.detach().exp() * logq.detach()).sum(-1).masked_fill(~s["mask"], 0.0)
        if not c["train"]:
            return [picked.detach(), entropy]
        return [picked.detach(), entropy,
                *torch.autograd.grad(picked, z, s["grad"].double())]
    if kind == "policy":
        logp = s["logps"].detach().double().requires_grad_()
        loss, metrics = _exact_policy(s, logp)
        return [loss.detach(), metrics, *torch.autograd.grad(loss, logp)]
    x = s["x"].detach().double()
    drops = round(c["p"] * 65536)
    u = _draws(s["rng"], -(-x.numel() // 8))[:x.numel()].view(x.shape)
    kept = (u >= drops).double() / (1 - drops / 65536)
    if kind == "dropout":
        return [x * kept, s["grad"].double() * kept]
    w = s["base"].weight
    code = w.quant_state.code
    table = torch.stack([code[w.long() >> 4], code[w.long() & 15]], -1).view(-1, QB)
    weight = (table * w.quant_state.absmax.view(-1, 1)).to(s["x"].dtype).double()
    weight = weight.view(c["out"], c["inp"])
    x = x.requires_grad_()
    a, b = (s[n].detach().double().requires_grad_() for n in ("a", "b"))
    y = x @ weight.t() + ((x * kept) @ a.t()) @ b.t() * 2.0
    return [y.detach(), *torch.autograd.grad(y, (x, a, b), s["grad"].double())]

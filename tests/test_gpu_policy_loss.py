"""The policy update's loss kernels against ``oracle.policy_loss`` in float64.

Bounds, with e = 2^-24 (half a float32 step), per counted row of V logits:

* every term exp2(x k - M) is off by at most 2 e (the exponential's ulp) and, from its
  argument a, by ln 2 |a| e relative, weighted by 2^a <= 1: 0.54 e; a sum of n terms in
  order adds at most n e of the whole, and a thread sums at most ceil(V / 512) + 8 terms
  before ten more levels; so S is off by (V / 512 + 24) e relative, logp by as much.
* k is off by e relative: logp by e times the distance of the token's logit from the
  distribution's mean, at most |logp| + H.
* logp's rounding: e |logp|.

The entropy adds t / S: sums of terms e^a a of one sign up to |a| <= 2 log2 V + 32, bounded
by (V / 512 + 26) e (H + 1) in the same way. A gradient c / T (1[v = id] - p_v) is off by p's
relative error (that of S, 2.6 e for its own exponential with |a| up to 150: 104 e) plus three
roundings, then half a step of its type.
"""

import math

import numpy as np
import pytest
import torch

from oracle import policy_loss as P

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def within(got, want, tol):
    """|got - want| <= tol everywhere (a NaN fails), with what is wrong in a few words."""
    if isinstance(got, torch.Tensor):
        got = got.detach().cpu().double().numpy()
    got = np.asarray(got).reshape(np.shape(want))
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol)
    at = tuple(int(i[0]) for i in np.nonzero(bad)) if bad.any() else None
    assert at is None, (f"{bad.sum()} of {bad.size} off, first {at}: {got[at]} for {want[at]}, "
                        f"bound {np.broadcast_to(tol, bad.shape)[at]}")


def _ops():
    from grpo_mi355x import kernels

    return kernels


def make(rows, vocab, dtype, seed, std=2.0, shift=0.0, counted=0.75):
    """CPU inputs: logits in the type, ids (-100 where not counted), mask."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * std + shift
    ids = torch.randint(0, vocab, (rows,), generator=g)
    x[torch.arange(rows), ids] += 6 * torch.rand(rows, generator=g)
    mask = torch.rand(rows, generator=g) < counted
    return x.to(DT[dtype]), torch.where(mask, ids, -100), mask


def bounds(x, ids, mask, t):
    """(logp, entropy, softmax) in float64 and the bounds on the first two."""
    logp, ent, p = P.token_logprobs(x.double().numpy(), ids.numpy(), mask.numpy(), t)
    n = x.shape[1] / 512 + 24
    return logp, ent, p, E * (n + 2 * np.abs(logp) + ent), E * (n + 2) * (2 * ent + 2)


def grad_bound(want, p, coef, t, dtype):
    c = np.abs(coef / t)[:, None]
    half = torch.finfo(DT[dtype]).eps / 2
    tiny = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}[dtype] + 2.0 ** -126
    return E * c * (p * (p.shape[1] / 512 + 130) + 3) * (p > 0) + half * np.abs(want) + tiny


VOCABS = [1, 2, 7, 8, 9, 511, 1000, 4097, 32003]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("t", [1.0, 0.7])
def test_token_logprobs_and_gradient(dev, dtype, vocab, t):
    rows = 5
    x, ids, mask = make(rows, vocab, dtype, seed=vocab + int(10 * t))
    logp, ent, p, tol, tol_ent = bounds(x, ids, mask, t)
    leaf = x.to(dev).requires_grad_()
    got, got_ent = _ops().token_logprobs(leaf, ids.to(dev), mask.to(dev), temperature=t,
                                         return_entropy=True)
    assert got.dtype == got_ent.dtype == torch.float32
    assert not got_ent.requires_grad
    within(got, logp, tol)
    within(got_ent, ent, tol_ent)
    coef = torch.randn(rows, generator=torch.Generator().manual_seed(1))
    grad, = torch.autograd.grad(got, leaf, coef.to(dev))
    want = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy(), t)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    within(grad, want, grad_bound(want, p, coef.double().numpy(), t, dtype))
    assert not grad[~mask.to(dev)].any()
    with torch.no_grad():  # the form without a gradient gives the same values
        again = _ops().token_logprobs(leaf, ids.to(dev), mask.to(dev), temperature=t)
    assert torch.equal(again, got.detach())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [151936, 152064, 262147, 2000003])
def test_whole_vocabularies(dev, dtype, vocab):
    x, ids, mask = make(3, vocab, dtype, seed=5, counted=1.1)
    logp, ent, p, tol, tol_ent = bounds(x, ids, mask, 1.0)
    leaf = x.to(dev).requires_grad_()
    got, got_ent = _ops().token_logprobs(leaf, ids.to(dev), return_entropy=True)
    within(got, logp, tol)
    within(got_ent, ent, tol_ent)
    coef = torch.tensor([1.0, -2.0, 0.5])
    grad, = torch.autograd.grad(got, leaf, coef.to(dev))
    want = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy())
    within(grad, want, grad_bound(want, p, coef.double().numpy(), 1.0, dtype))


def test_an_offset_of_all_logits_changes_nothing(dev):
    x, ids, mask = make(4, 5000, "f32", seed=2, counted=1.1)
    x = torch.round(x * 64) / 64  # so that the shifted logits are exact too
    for shift in (0.0, 1000.0, -4096.0, 65536.0):
        y = x + shift
        logp, _, _, tol, _ = bounds(x, ids, mask, 0.7)
        got = _ops().token_logprobs(y.to(dev), ids.to(dev), temperature=0.7)
        assert torch.equal(y - shift, x)
        # x k - M has one rounding at the size of its result: no shift in the bound
        within(got, logp, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [777, 50257])
def test_masked_vocabulary_and_lowest_values(dev, dtype, vocab):
    x, ids, _ = make(6, vocab, dtype, seed=9, counted=1.1)
    low = torch.finfo(x.dtype).min
    x[0, 100:] = -math.inf
    ids[0] = 3
    x[1, 100:] = low
    ids[1] = 5
    x[2] = low                      # the whole row at the lowest value: uniform
    x[3, ids[3]] = -math.inf        # the token itself is ruled out
    x[4, :] = -math.inf
    x[4, 9] = 2.0
    ids[4] = 9                      # only one token is left
    mask = torch.ones(6, dtype=torch.bool)
    logp, ent, p, tol, tol_ent = bounds(x, ids, mask, 1.0)
    leaf = x.to(dev).requires_grad_()
    got, got_ent = _ops().token_logprobs(leaf, ids.to(dev), return_entropy=True)
    g = got.detach().cpu().double().numpy()
    assert g[3] == -math.inf and logp[3] == -math.inf
    keep = np.array([0, 1, 2, 4, 5])
    within(g[keep], logp[keep], tol[keep])
    within(got_ent, ent, tol_ent)
    assert abs(g[4]) <= 3 * E  # one term: its own error, not a sum's
    coef = torch.ones(6)
    grad, = torch.autograd.grad(got, leaf, coef.to(dev))
    want = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy())
    within(grad, want, grad_bound(want, p, np.ones(6), 1.0, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1030, 70001])  # one workgroup a row, and several
def test_values_that_are_not_finite(dev, dtype, vocab):
    x, ids, mask = make(6, vocab, dtype, seed=4, counted=1.1)
    x[0] = -math.inf                # nothing left: NaN, as a log-softmax
    x[1, 7] = math.inf
    x[2, 900] = math.nan
    x[3] = math.nan                 # not counted: not read
    x[4, 0] = math.inf
    mask[3] = mask[4] = False
    ids[3], ids[4] = -100, 10 ** 12
    leaf = x.to(dev).requires_grad_()
    got, ent = _ops().token_logprobs(leaf, ids.to(dev), mask.to(dev), return_entropy=True)
    want = torch.log_softmax(x.double(), -1)[torch.arange(6), ids.clamp(0, vocab - 1)]
    g = got.detach().cpu()
    assert torch.isnan(g[:3]).all() and torch.isnan(want[:3]).all()
    assert g[3] == g[4] == 0 and ent[3] == ent[4] == 0
    assert abs(float(g[5]) - float(want[5])) <= 64 * E * (1 + abs(float(want[5])))
    grad, = torch.autograd.grad(got.sum(), leaf)
    assert torch.isnan(grad[:3]).any(1).all()
    assert not grad[3:5].any()
    assert torch.isfinite(grad[5]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [100.0, 900.0, 20000.0])
def test_gradients_of_large_logits(dev, dtype, size):
    """Whatever their size: below and beyond where 16-bit gradients go by vectors."""
    x, ids, mask = make(5, 4096, "f32", seed=7, counted=1.1)
    x = (x + size).to(DT[dtype])
    logp, ent, p, tol, _ = bounds(x, ids, mask, 0.7)
    coef = torch.tensor([1.0, -2.0, 0.5, 3.0, -0.25])
    leaf = x.to(dev).requires_grad_()
    got = _ops().token_logprobs(leaf, ids.to(dev), temperature=0.7)
    within(got, logp, tol)
    grad, = torch.autograd.grad(got, leaf, coef.to(dev))
    want = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy(), 0.7)
    # by vectors the exponent is off by 2^-13 of the value at most
    extra = 0.0 if dtype == "f32" else 2.0 ** -13 * np.abs(coef.numpy() / 0.7)[:, None] * p
    within(grad, want, grad_bound(want, p, coef.double().numpy(), 0.7, dtype) + extra)


def test_ids_outside_the_vocabulary_give_nan(dev):
    x, ids, mask = make(4, 100, "f32", seed=1, counted=1.1)
    ids[0], ids[1], ids[2] = -1, 100, 2 ** 40
    got = _ops().token_logprobs(x.to(dev), ids.to(dev))
    assert torch.isnan(got[:3]).all() and torch.isfinite(got[3])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strided_and_unaligned_logits(dev, dtype):
    """Rows at every alignment: slices of the vocabulary, of the positions, an expanded
    batch and a transposed one give what their contiguous copies give."""
    base, _, _ = make(6 * 5, 135, dtype, seed=8)
    base = base.view(6, 5, 135).to(dev)
    views = [base[:, :-1], base[:, 1:, 3:130], base[::2, :, 1:], base.transpose(0, 1),
             base[:1].expand(3, -1, -1), base[..., ::2], base[:, 2]]
    for v in views:
        ids = torch.randint(0, v.shape[-1], v.shape[:-1], device=dev)
        mask = torch.rand(ids.shape, device=dev) < 0.8
        out = []
        for x in (v, v.contiguous()):
            leaf = x.detach().requires_grad_()
            assert leaf.stride() == x.stride()
            got, ent = _ops().token_logprobs(leaf, ids, mask, return_entropy=True)
            grad, = torch.autograd.grad(got, leaf, torch.ones_like(got))
            out.append((got.detach(), ent, grad))
        # another split of the row over the threads: the sums' order differs
        assert torch.allclose(out[0][0], out[1][0], rtol=4 * E, atol=64 * E)
        assert torch.allclose(out[0][1], out[1][1], rtol=64 * E, atol=64 * E)
        assert torch.allclose(out[0][2].float(), out[1][2].float(),
                              rtol=2 * torch.finfo(v.dtype).eps, atol=64 * E)


def test_leading_shapes(dev):
    x, ids, _ = make(24, 50, "f32", seed=3)
    ids = ids.clamp(min=0).to(dev)
    flat = _ops().token_logprobs(x.to(dev), ids)
    four = _ops().token_logprobs(x.to(dev).view(2, 3, 4, 50), ids.view(2, 3, 4))
    assert torch.equal(four.reshape(-1), flat)
    for shape in ((0, 5, 50), (3, 0, 50), (0, 50)):
        leaf = torch.zeros(shape, device=dev, requires_grad=True)
        got = _ops().token_logprobs(leaf, torch.zeros(shape[:-1], dtype=torch.int64, device=dev))
        assert got.shape == shape[:-1]
        got.sum().backward()
        assert leaf.grad.shape == shape


def test_refusals_on_the_device(dev):
    x = torch.zeros(2, 3, 8, device=dev)
    ids = torch.zeros(2, 3, dtype=torch.int64, device=dev)
    ops = _ops()
    for bad, message in [((x.double(), ids), "bfloat16"), ((x, ids.int()), "int64"),
                         ((x, ids[:1]), "token_ids must be"), ((x, ids.cpu()), "must be on"),
                         ((x[..., :0], ids), "at least one"), ((x[0, 0], ids[0, 0]), "vocab"),
                         ((x, ids, ids[:, :2]), "mask must be")]:
        with pytest.raises(ValueError, match=message):
            ops.token_logprobs(*bad)
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_logprobs(x, ids, temperature=t)
    with pytest.raises(ValueError, match="batch, seq, vocab"):
        ops.fused_grpo_loss(x[0], ids[0], None, torch.zeros(3, device=dev))
    wide = x[:1, :1, :1].expand(1, 1, 2 ** 30 + 1)  # no memory of its own
    with pytest.raises(ValueError, match="vocabulary of at most"):
        ops.token_logprobs(wide, ids[:1, :1])
    for shape in ((1, 2 ** 31), (2 ** 23, 1)):
        with pytest.raises(ValueError, match="2.23 sequences"):
            ops.grpo_policy_loss(x[0, :1, :1].expand(shape), None, x[0, 0, :1].expand(shape[0]))
    leaf = x.clone().requires_grad_()
    got = ops.token_logprobs(leaf, ids)
    grad, = torch.autograd.grad(got.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        grad.sum().backward()


@pytest.mark.parametrize("t", [1e-20, 1e-10, 3e-9, 1e-8, 1e-7, 1e20])
def test_temperatures_at_the_ends(dev, t):
    """Ties share a row whatever the temperature; -inf and (below) anything less has none.
    Exponents reach 8 in size, with two roundings of 2^-24 each: 2^-20 of ln 2 and up."""
    x = torch.full((1, 4, 1001), -math.inf, device=dev)
    x[0, 0, :10], x[0, 1, 5:9], x[0, 2, 1000], x[0, 3, ::7] = 2.3, -3.1, 0.0, 29.7
    if t < 1.0:
        x[0, :, 501] = -4.0
    ids = torch.tensor([[3, 8, 1000, 7]], device=dev)
    n = torch.tensor([[10.0, 4.0, 1.0, 143.0]], dtype=torch.float64, device=dev)
    leaf = x.requires_grad_()
    got = _ops().token_logprobs(leaf, ids, temperature=t)
    assert torch.allclose(got.double(), -n.log(), rtol=2.0 ** -20, atol=0.0)
    # the gradient times T: 1 - 1 / n at the token, -1 / n at the ties, 0 elsewhere
    grad, = torch.autograd.grad(got.sum() * t, leaf)
    want = -(x.detach() == x.detach().amax(-1, keepdim=True)).double() / n[..., None]
    want.scatter_add_(2, ids[..., None], torch.ones_like(want[..., :1]))
    assert torch.allclose(grad.double(), want, rtol=2.0 ** -18, atol=1e-30)


# ------------------------------------------------------------- policy loss --

def tokens(b, s, seed, counted=0.75, spread=0.4):
    """Log-probabilities whose ratios keep 1e-3 from every border used below."""
    g = np.random.default_rng(seed)
    logp = (-3 * g.random((b, s))).astype(np.float32)
    diff = spread * g.standard_normal((b, s))
    for border in (math.log(0.8), math.log(1.2), math.log(1.28), math.log(1.5)):
        near = np.abs(diff - border) < 1e-3
        diff[near] = border + 2e-3
    old = (logp - diff).astype(np.float32)
    ref = (logp + 0.3 * g.standard_normal((b, s))).astype(np.float32)
    mask = g.random((b, s)) < counted
    if b > 2:
        mask[1] = False
    return logp, old, ref, g.standard_normal(b).astype(np.float32), mask


def close(got, want, scale, n):
    """float64 work on float32 inputs: one rounding of the result, sums of n terms of
    absolute sum ``scale`` in float64."""
    got = float(got.detach())
    return abs(got - want) <= 1.01 * E * abs(want) + (n + 64) * 2.0 ** -52 * scale + 1e-45


@pytest.mark.parametrize("b, s", [(1, 1), (3, 1), (1, 257), (5, 333), (64, 200), (700, 3),
                                  (1500, 2), (2, 40000)])
@pytest.mark.parametrize("normalizer", ["tokens", "sequences", 1234.5])
@pytest.mark.parametrize("beta, delta", [(0.0, None), (0.04, 1.5)])
def test_policy_loss_and_gradient(dev, b, s, normalizer, beta, delta):
    logp, old, ref, adv, mask = tokens(b, s, seed=b * 1000 + s)
    want, want_metrics, want_grad = P.policy_loss(
        logp, old, adv, mask, ref if beta else None, 0.2, 0.28, delta or math.inf, beta,
        normalizer)
    put = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    leaf = put(logp).requires_grad_()
    loss, metrics = _ops().grpo_policy_loss(
        leaf, put(old), put(adv), put(mask), ref_logps=put(ref) if beta else None, eps_low=0.2,
        eps_high=0.28, delta=delta, beta=beta, normalizer=normalizer)
    n = mask.sum()
    # exp is off by a step or two of float64; the terms' absolute sum is at most
    scale = float(np.abs(adv).max() * 4 + 1) * (1.0 if isinstance(normalizer, str)
                                                else n / normalizer)
    assert loss.shape == () and loss.dtype == torch.float32
    assert close(loss, want, scale, n)
    assert not metrics.requires_grad
    for j in range(4):
        assert close(metrics[j], want_metrics[j], 8.0, n), j
    factor = -0.75
    grad, = torch.autograd.grad(loss * factor, leaf)
    # the derivative, its product with the upstream gradient and one rounding
    within(grad, factor * want_grad, 1.01 * E * np.abs(factor * want_grad) + 2.0 ** -149)
    assert not grad[~put(mask)].any()


def test_policy_loss_by_differences(dev):
    """The gradient is the difference quotient of the loss itself."""
    logp, old, ref, adv, mask = tokens(3, 4, seed=11, counted=1.1)
    mask[:] = True
    put = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731

    def loss(lp):
        return _ops().grpo_policy_loss(lp, put(old), put(adv), put(mask), ref_logps=put(ref),
                                       beta=0.1, eps_high=0.28, normalizer=1.0)

    leaf = put(logp).requires_grad_()
    grad, = torch.autograd.grad(loss(leaf)[0], leaf)
    h = 2.0 ** -11
    for b in range(3):
        for s in range(4):
            d = torch.zeros_like(leaf)
            d[b, s] = h
            up, down = float(loss(leaf.detach() + d)[0]), float(loss(leaf.detach() - d)[0])
            # the loss's own rounding (12 terms of a size up to 4: 48 e each way) over 2 h,
            # and a third derivative of at most 16
            assert abs((up - down) / (2 * h) - float(grad[b, s])) <= 96 * E / h + 16 * h * h


def test_policy_loss_options(dev):
    logp, old, ref, adv, mask = tokens(6, 50, seed=21)
    put = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    ops = _ops()
    leaf = put(logp).requires_grad_()
    # on-policy: no old log-probabilities, every ratio 1
    loss, metrics = ops.grpo_policy_loss(leaf, None, put(adv), put(mask))
    want, _, want_grad = P.policy_loss(logp, None, adv, mask)
    assert close(loss, want, 8.0, mask.size)
    assert metrics[0] == 1 and metrics[1] == 0 and metrics[3] == 0
    grad, = torch.autograd.grad(loss, leaf)
    within(grad, want_grad, 1.01 * E * np.abs(want_grad))
    # an advantage for each token, masks of other types, no mask
    wide = np.ascontiguousarray(np.broadcast_to(adv[:, None], logp.shape))
    base = ops.grpo_policy_loss(put(logp), put(old), put(adv), put(mask))
    for m in (put(mask).long(), put(mask).float(), put(mask).to(torch.uint8)):
        got = ops.grpo_policy_loss(put(logp), put(old), put(wide), m)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    full = ops.grpo_policy_loss(put(logp), put(old), put(adv))
    ones = ops.grpo_policy_loss(put(logp), put(old), put(adv), torch.ones_like(put(mask)))
    assert torch.equal(full[0], ones[0]) and torch.equal(full[1], ones[1])
    # strided and 16-bit inputs are taken at their values
    t = put(logp).t().contiguous().t()
    got = ops.grpo_policy_loss(t, put(old).double(), put(adv), put(mask))
    assert torch.equal(got[0], base[0])


@pytest.mark.parametrize("normalizer", ["tokens", "sequences", 7.0])
def test_nothing_counted(dev, normalizer):
    b, s, v = 3, 4, 40
    nan = torch.full((b, s), math.nan, device=dev)
    mask = torch.zeros(b, s, dtype=torch.bool, device=dev)
    adv = torch.full((b,), math.nan, device=dev)
    leaf = nan.clone().requires_grad_()
    loss, metrics = _ops().grpo_policy_loss(leaf, nan, adv, mask, ref_logps=nan, beta=0.1,
                                            normalizer=normalizer)
    loss.backward()
    assert loss == 0 and not metrics.any() and not leaf.grad.any()
    logits = torch.full((b, s, v), math.nan, device=dev, requires_grad=True)
    ids = torch.full((b, s), -100, device=dev)
    loss, logp, metrics = _ops().fused_grpo_loss(logits, ids, nan, adv, mask, ref_logps=nan,
                                                 beta=0.1, normalizer=normalizer)
    loss.backward()
    assert loss == 0 and not metrics.any() and not logp.any() and not logits.grad.any()
    for shape in ((0, 4), (3, 0)):
        e = torch.zeros(shape, device=dev, requires_grad=True)
        loss, metrics = _ops().grpo_policy_loss(e, None, torch.zeros(shape[0], device=dev),
                                                normalizer=normalizer)
        loss.backward()
        assert loss == 0 and not metrics.any() and e.grad.shape == shape


# ------------------------------------------------------ loss from the logits --

def loss_inputs(b, s, vocab, dtype, seed, t=1.0, beta=0.04):
    x, ids, _ = make(b * s, vocab, dtype, seed, counted=1.1)
    _, _, _, adv, mask = tokens(b, s, seed)
    flat = torch.from_numpy(mask.reshape(-1))
    logp, _, p = P.token_logprobs(x.double().numpy(), ids.numpy(), np.ones(b * s, bool), t)
    diff = (tokens(b, s, seed + 1)[0] - tokens(b, s, seed + 1)[1]).reshape(-1).astype(np.float64)
    old = np.float32(logp - diff).reshape(b, s)
    ref = np.float32(logp + 0.1).reshape(b, s) if beta else None
    ids = torch.where(flat, ids, -100)
    return x.view(b, s, vocab), ids.view(b, s), old, ref, adv, mask, logp, p


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("b, s, vocab", [(1, 1, 9), (300, 30, 65), (1100, 1, 17), (3, 5, 1000), (4, 33, 4097), (2, 3, 151936),
                                         (1, 2, 262147), (40, 16, 300), (8, 16, 151936), (8, 16, 160003)])
@pytest.mark.parametrize("normalizer, t, beta", [("tokens", 1.0, 0.0), ("sequences", 0.7, 0.04)])
def test_fused_loss_and_gradient(dev, dtype, b, s, vocab, normalizer, t, beta):
    x, ids, old, ref, adv, mask, logp, p = loss_inputs(b, s, vocab, dtype, seed=vocab + b, t=t,
                                                       beta=beta)
    if not mask.any():
        mask[0, 0] = True
        ids[0, 0] = 3
        logp, _, p = P.token_logprobs(x.view(b * s, vocab).double().numpy(),
                                      ids.clamp(min=0).reshape(-1).numpy(),
                                      np.ones(b * s, bool), t)
    want, want_metrics, d = P.policy_loss(logp.reshape(b, s), old, adv, mask, ref, 0.2, 0.28,
                                          math.inf, beta, normalizer)
    put = lambda a: None if a is None else torch.as_tensor(a).to(dev)  # noqa: E731
    leaf = put(x).requires_grad_()
    loss, got_logp, metrics = _ops().fused_grpo_loss(
        leaf, put(ids), put(old), put(adv), put(mask), ref_logps=put(ref), temperature=t,
        eps_high=0.28, beta=beta, normalizer=normalizer)
    assert not got_logp.requires_grad and not metrics.requires_grad
    tol = E * (vocab / 512 + 24 + 2 * np.abs(logp.reshape(b, s)) + math.log(vocab))
    within(got_logp, np.where(mask, logp.reshape(b, s), 0), tol)
    top = float(tol.max())  # logp's error moves a ratio below 8 by at most 8 of it
    scale = float(np.abs(adv).max()) * 8 + 1
    assert abs(float(loss.detach()) - want) <= top * scale + E * abs(want)
    for j in range(4):
        assert abs(float(metrics[j]) - want_metrics[j]) <= 8 * top + E * abs(want_metrics[j]), j
    factor = 0.5
    grad, = torch.autograd.grad(loss * factor, leaf)
    coef = factor * d.reshape(-1)
    wantg = P.logits_grad(p, ids.clamp(min=0).reshape(-1).numpy(), mask.reshape(-1), coef, t)
    # the row's factor is off by 2 of logp's error relative (r, and the KL term's exp)
    slack = (np.abs(coef) * 4 + (0.1 if beta else 0.0)) * top
    tol = grad_bound(wantg, p, coef, t, dtype) + (slack / t)[:, None] * (
        p + (np.arange(vocab)[None] == ids.reshape(-1, 1).numpy()))
    within(grad, wantg, tol * mask.reshape(-1, 1))


def test_fused_loss_is_its_parts(dev):
    """One call equals token_logprobs then grpo_policy_loss, to logp's rounding."""
    x, ids, old, ref, adv, mask, logp, _ = loss_inputs(4, 20, 3001, "f32", seed=6)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    kw = dict(ref_logps=put(ref), beta=0.04, delta=3.0)
    one, two = put(x).requires_grad_(), put(x).requires_grad_()
    loss, lp, metrics = _ops().fused_grpo_loss(one, put(ids), put(old), put(adv), put(mask), **kw)
    parts = _ops().token_logprobs(two, put(ids), put(mask))
    assert torch.equal(parts.detach(), lp)
    loss2, metrics2 = _ops().grpo_policy_loss(parts, put(old), put(adv), put(mask), **kw)
    tol = 16 * E * float(np.abs(logp).max())
    assert abs(float(loss.detach()) - float(loss2.detach())) <= tol
    assert torch.allclose(metrics, metrics2, rtol=4 * E, atol=tol)
    loss.backward()
    loss2.backward()
    assert torch.allclose(one.grad, two.grad, rtol=64 * E, atol=tol / mask.sum())


def test_backward_twice_and_scaled(dev):
    """A second backward of a kept graph, and any upstream gradient, give the gradient."""
    x, ids, old, _, adv, mask, _, _ = loss_inputs(2, 9, 2000, "bf16", seed=3, beta=0.0)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    leaf = put(x).requires_grad_()
    loss, _, _ = _ops().fused_grpo_loss(leaf, put(ids), put(old), put(adv), put(mask))
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = one.clone()
    one.mul_(3.0)  # the caller owns what it was given
    two, = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(two, kept)
    half, = torch.autograd.grad(0.5 * loss, leaf, retain_graph=True)
    assert torch.equal(half, kept * 0.5)  # a power of two: the same roundings
    leaf.grad = None
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(leaf.grad, kept + kept)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vectors, rows", [(300, 7), (2600, 7), (5000, 7), (7200, 7), (9800, 7),
                                           (14400, 130), (19500, 130)])
def test_gradient_of_the_one_pass(dev, dtype, vectors, rows):
    """The gradient made with the loss is, to the bit, what the logits give again (which the
    test above holds to 64 bits), at every size of row and for rows of every kind."""
    from grpo_mi355x import _lib

    dt = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    vocab = vectors * 16 // dt.itemsize + 3
    assert _lib.library().grpo_policy_loss_logits_one_pass(
        ["bf16", "f16", "f32"].index(dtype), 1, rows, vocab)
    g = torch.Generator().manual_seed(vectors)
    x = torch.randn(1, rows, vocab, generator=g).mul_(3).to(dt)
    ids = torch.randint(0, vocab, (1, rows), generator=g)
    mask = torch.ones(1, rows, dtype=torch.bool)
    x[0, 0, 50:], ids[0, 0] = -math.inf, 7
    x[0, 1, 50:], ids[0, 1] = torch.finfo(dt).min, vocab - 1
    x[0, 2], x[0, 3, 9], x[0, 4, vocab - 1] = torch.finfo(dt).min, math.inf, math.nan
    x[0, 5] += 900.0
    x[0, 6], mask[0, 6], ids[0, 6] = math.nan, False, -100
    old = torch.randn(1, rows, generator=g) - 9.0
    put = lambda t: t.to(dev)  # noqa: E731
    leaf = put(x).requires_grad_()
    loss, _, _ = _ops().fused_grpo_loss(leaf, put(ids), put(old), torch.ones(1, device=dev),
                                        put(mask), temperature=0.9)
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    two, = torch.autograd.grad(loss, leaf)
    assert torch.allclose(one, two, rtol=0.0, atol=0.0, equal_nan=True)
    one = one[0].cpu()
    assert torch.isfinite(one[[0, 1, 2, 5]]).all() and not one[6].any()
    assert one[3].isnan().any() and one[4].isnan().all()
    # (a ratio above the clip leaves a row without a gradient)
    assert torch.isfinite(one[7:]).all() and one[:3].any() and (rows == 7 or one[7:].any())


def test_logits_changed_before_the_backward_are_refused(dev):
    x, ids, old, _, adv, mask, _, _ = loss_inputs(2, 3, 64, "f32", seed=3, beta=0.0)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    leaf = put(x).requires_grad_()
    logits = leaf * 1.0
    loss, _, _ = _ops().fused_grpo_loss(logits, put(ids), put(old), put(adv), put(mask))
    with torch.no_grad():
        logits.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_another_stream_and_many_calls(dev):
    """Calls on a side stream, two in flight, equal those on the default stream."""
    sets = [loss_inputs(3, 17, 5003, "bf16", seed=s) for s in (1, 2)]
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731

    def go(x, ids, old, ref, adv, mask, *_):
        leaf = put(x).requires_grad_()
        loss, lp, m = _ops().fused_grpo_loss(leaf, put(ids), put(old), put(adv), put(mask),
                                             ref_logps=put(ref), beta=0.04)
        return [loss.detach(), lp, m, *torch.autograd.grad(loss, leaf)]

    want = [go(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(go(*s))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_captured_and_replayed(dev):
    """Forward and backward in one graph, replayed with other inputs between eager work."""
    b, s, vocab = 3, 7, 4099
    sets = [loss_inputs(b, s, vocab, "bf16", seed=k) for k in (1, 2, 3)]
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731

    def eager(v):
        leaf = put(v[0]).requires_grad_()
        loss, lp, m = _ops().fused_grpo_loss(leaf, put(v[1]), put(v[2]), put(v[4]), put(v[5]),
                                             ref_logps=put(v[3]), beta=0.04)
        return [loss.detach(), lp, m, *torch.autograd.grad(loss, leaf)]

    want = [eager(v) for v in sets]
    held = [put(sets[0][i]).clone() for i in range(6)]
    held[0].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        loss, lp, m = _ops().fused_grpo_loss(held[0], held[1], held[2], held[4], held[5],
                                             ref_logps=held[3], beta=0.04)
        return [loss.detach(), lp, m, *torch.autograd.grad(loss, held[0])]

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in (0, 1, 2, 1):
        with torch.no_grad():
            for h, v in zip(held, sets[k]):
                h.copy_(put(v))
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, want[k]):
            assert torch.equal(u, v)
        eager(sets[k])  # eager work between the replays
        torch.cuda.synchronize()


def test_offsets_past_32_bits(dev):
    """16384 rows of 151936 values: 5 GB, rows past 2^31 values. The last rows' results are
    those of a call of their own (the weights do not depend on the batch: a number)."""
    rows, vocab = 16384, 151936
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(1, rows, vocab, generator=g, device=dev, dtype=torch.bfloat16)
    ids = torch.randint(0, vocab, (1, rows), generator=g, device=dev)
    old = torch.full((1, rows), -12.0, device=dev)
    adv = torch.randn(1, rows, generator=g, device=dev)
    x.requires_grad_()

    def go(x, ids, old, adv):
        loss, lp, _ = _ops().fused_grpo_loss(x, ids, old, adv, normalizer=100.0)
        grad, = torch.autograd.grad(loss, x)
        lp2 = _ops().token_logprobs(x, ids)
        grad2, = torch.autograd.grad(lp2, x, adv)
        return lp, grad, lp2.detach(), grad2

    lp, grad, lp2, grad2 = go(x, ids, old, adv)
    end = slice(rows - 5, rows)
    # 4096 rows and more are not cut over workgroups; these five are, and their sums' order
    # differs: to the roundings of logp, and a gradient's half step either way
    want = go(x.detach()[:, end].clone().requires_grad_(), ids[:, end], old[:, end], adv[:, end])
    for a, b in ((lp, want[0]), (lp2, want[2])):
        assert torch.allclose(a[:, end], b, rtol=4 * E, atol=16 * E)
    for a, b in ((grad, want[1]), (grad2, want[3])):
        assert torch.allclose(a[:, end].float(), b.float(), rtol=2.0 ** -7, atol=1e-30)


def test_shifted_view_of_a_models_logits(dev):
    """logits[:, :-1] as a trainer slices them: the gradient reaches the whole tensor."""
    x, ids, old, ref, adv, mask, _, _ = loss_inputs(3, 8, 2001, "bf16", seed=5)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    whole = torch.cat([put(x), torch.full((3, 1, 2001), math.nan, device=dev).bfloat16()], 1)
    leaf, part = whole.clone().requires_grad_(), put(x).requires_grad_()
    kw = dict(ref_logps=put(ref), beta=0.04)
    args = (put(ids), put(old), put(adv), put(mask))
    a, lp, _ = _ops().fused_grpo_loss(leaf[:, :-1], *args, **kw)
    b, lp2, _ = _ops().fused_grpo_loss(part, *args, **kw)
    a.backward()
    b.backward()
    # rows start at other addresses, so their sums' order differs
    assert torch.allclose(lp, lp2, rtol=4 * E, atol=16 * E)
    assert torch.allclose(leaf.grad[:, :-1].float(), part.grad.float(), rtol=2.0 ** -7, atol=1e-30)
    assert not leaf.grad[:, -1].any()


def test_saved_tensors_that_moved(dev):
    """Hooks that keep the saved logits elsewhere: the backward reads what it is given."""
    x, ids, old, _, adv, mask, _, _ = loss_inputs(2, 9, 2000, "bf16", seed=3, beta=0.0)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    grads = []
    for hooks in (False, True):
        leaf = put(x).requires_grad_()
        with torch.autograd.graph.save_on_cpu() if hooks else torch.enable_grad():
            loss, _, _ = _ops().fused_grpo_loss(leaf * 1.0, put(ids), put(old), put(adv),
                                                put(mask))
            lp = _ops().token_logprobs(leaf * 1.0, put(ids), put(mask))
        torch.full_like(leaf, math.nan)  # takes the place of what was given back
        grads.append(torch.autograd.grad(0.5 * loss, leaf) + torch.autograd.grad(lp.sum(), leaf))
    for u, v in zip(*grads):
        assert torch.equal(u, v)


@pytest.mark.parametrize("vocab", [600, 160001])  # a row in registers, and beyond
def test_fused_loss_options(dev, vocab):
    """On-policy, a cap below the clip's border, an advantage for each token, a number as
    normalizer, a strided mask and a mask of another type."""
    b, s = 3, 6
    x, ids, old, _, _, mask, logp, p = loss_inputs(b, s, vocab, "f32", seed=8, beta=0.0)
    adv = np.random.default_rng(3).standard_normal((b, s)).astype(np.float32)
    put = lambda a: None if a is None else torch.as_tensor(a).to(dev)  # noqa: E731
    wide = torch.zeros(b, s + 2, dtype=torch.int64, device=dev)
    wide[:, 1:-1] = put(mask)
    top = E * (vocab / 512 + 24 + 2 * np.abs(logp).max() + math.log(vocab))
    for o in (None, old):
        leaf = put(x).requires_grad_()
        loss, lp, metrics = _ops().fused_grpo_loss(leaf, put(ids), put(o), put(adv),
                                                   wide[:, 1:-1], delta=1.05, normalizer=77.0)
        want, want_metrics, d = P.policy_loss(logp.reshape(b, s), o, adv, mask, delta=1.05,
                                              normalizer=77.0)
        scale = (8 * np.abs(adv).max() + 1) * mask.sum() / 77
        assert abs(float(loss.detach()) - want) <= top * scale + E * abs(want)
        within(metrics, want_metrics, 8 * top + E * np.abs(want_metrics))
        grad, = torch.autograd.grad(loss, leaf)
        coef = d.reshape(-1)
        wantg = P.logits_grad(p, ids.clamp(min=0).reshape(-1).numpy(), mask.reshape(-1), coef)
        tol = grad_bound(wantg, p, coef, 1.0, "f32") + (np.abs(coef) * 4 * top)[:, None] * (
            p + (np.arange(vocab)[None] == ids.reshape(-1, 1).numpy()))
        within(grad.reshape(b * s, vocab), wantg, tol * mask.reshape(-1, 1))
    # without a gradient: the same loss
    with torch.no_grad():
        again = _ops().fused_grpo_loss(put(x), put(ids), put(old), put(adv), put(mask),
                                       delta=1.05, normalizer=77.0)
    assert abs(float(again[0]) - float(loss.detach())) <= 2 * top * scale
    assert torch.allclose(again[1], lp, rtol=4 * E, atol=16 * E)


def test_policy_loss_of_16_bit_log_probabilities(dev):
    logp, old, _, adv, mask = tokens(3, 9, seed=2)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    leaf = put(logp).bfloat16().requires_grad_()
    loss, _ = _ops().grpo_policy_loss(leaf, put(old), put(adv), put(mask))
    loss.backward()
    want, _, grad = P.policy_loss(leaf.detach().cpu().double().numpy(), old, adv, mask)
    assert close(loss, want, 8.0 * float(np.abs(adv).max()), mask.size)
    assert leaf.grad.dtype == torch.bfloat16
    within(leaf.grad, grad, (2.0 ** -8 + E) * np.abs(grad))


@pytest.mark.parametrize("rows", [4, 700])  # cut over workgroups, and not
def test_the_parts_captured_and_replayed(dev, rows):
    """token_logprobs, grpo_policy_loss and their gradients in one graph, replayed with
    other inputs between eager work."""
    vocab = 20001
    g = torch.Generator(device=dev).manual_seed(4)

    def inputs():
        x = torch.randn(2, rows // 2, vocab, generator=g, device=dev).bfloat16()
        ids = torch.randint(0, vocab, (2, rows // 2), generator=g, device=dev)
        old = -10 + torch.randn(2, rows // 2, generator=g, device=dev)
        mask = torch.rand(2, rows // 2, generator=g, device=dev) < 0.7
        return [x, ids, old, torch.randn(2, generator=g, device=dev), mask]

    def step(v):
        lp, ent = _ops().token_logprobs(v[0], v[1], v[4], return_entropy=True)
        loss, m = _ops().grpo_policy_loss(lp, v[2], v[3], v[4], normalizer="sequences")
        return [lp.detach(), ent, loss.detach(), m, *torch.autograd.grad(loss, v[0])]

    sets = [inputs() for _ in range(3)]
    want = []
    for v in sets:
        want.append(step([v[0].clone().requires_grad_(), *v[1:]]))
    held = [t.clone() for t in sets[0]]
    held[0].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for k in (0, 1, 2, 1):
        with torch.no_grad():
            for h, v in zip(held, sets[k]):
                h.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, want[k]):
            assert torch.equal(u, v)
        step([sets[k][0].clone().requires_grad_(), *sets[k][1:]])
        torch.cuda.synchronize()


@pytest.mark.parametrize("b", [0, 7, 1024, 1025, 5000])
def test_c_entries_with_a_mask_and_no_tokens(dev, b):
    """Sequences of length 0 and a mask pointer all the same: nothing counted, whatever the
    number of sequences."""
    import ctypes

    from grpo_mi355x import _lib

    lib = _lib.device_library()
    policy = ctypes.byref(_lib.Policy(0.2, 0.2, math.inf, 0.0, 1.0, 1))
    buf, out = torch.ones(64, dtype=torch.uint8, device=dev), torch.full((5,), 7.0, device=dev)
    need = max(lib.grpo_policy_loss_workspace_bytes(b, 0),
               lib.grpo_policy_loss_logits_workspace_bytes(0, b, 0, 8))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    at, loss, metrics = buf.data_ptr(), out.data_ptr(), out[1:].data_ptr()
    rest = (ws.data_ptr(), need, _lib.stream_handle(dev))
    assert lib.grpo_policy_loss(at, None, None, at, 0, at, b, 0, policy, loss, metrics, None,
                                *rest) == 0
    assert not out.any()
    out.fill_(7.0)
    assert lib.grpo_policy_loss_logits(at, 0, 8, 8, b, 0, 8, at, at, 1.0, None, None, at, 0,
                                       policy, loss, at, metrics, None, None, None, 0, 0,
                                       *rest) == 0
    assert not out.any()


@pytest.mark.parametrize("dtype, vocab", [("bf16", 1000), ("f32", 160001)])  # one pass, and not
def test_a_reference_without_a_weight_is_a_metric_alone(dev, dtype, vocab):
    """beta = 0 with ref_logps: loss and gradients are those without it to the bit, also where
    exp(ref - logp) is not finite."""
    x, ids, old, _, adv, mask, logp, _ = loss_inputs(3, 6, vocab, dtype, seed=8, beta=0.0)
    mask[:] = True
    ids = ids.clamp(min=0)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    kw = dict(eps_high=0.28, normalizer="sequences")

    def run(x, ref):
        leaf = put(x).requires_grad_()
        loss, lp, m = _ops().fused_grpo_loss(leaf, put(ids), put(old), put(adv), put(mask),
                                             ref_logps=ref, **kw)
        lp2 = lp.clone().requires_grad_()
        loss2, m2 = _ops().grpo_policy_loss(lp2, put(old), put(adv), put(mask), ref_logps=ref,
                                            **kw)
        grads = [*torch.autograd.grad(loss, leaf), *torch.autograd.grad(loss2, lp2)]
        return [loss.detach(), loss2.detach(), lp, *grads], [m, m2]

    ref = put(np.float32(logp + 0.1).reshape(3, 6))
    plain, with_ref = run(x, None), run(x, ref)
    assert all(torch.equal(u, v) for u, v in zip(plain[0], with_ref[0]))
    at = P.token_logprobs(x.view(18, vocab).double().numpy(), ids.reshape(-1).numpy(),
                          np.ones(18, bool))[0]
    q = ref.cpu().double().numpy() - at.reshape(3, 6)
    want = float((np.exp(q) - q - 1).mean())
    for m, m0 in zip(with_ref[1], plain[1]):
        # logp is off by less than 2^-15 here, and each term's slope is e^q - 1
        assert abs(float(m[2]) - want) <= 2.0 ** -15 * np.abs(np.expm1(q)).mean() + E * want
        assert m0[2] == 0 and torch.equal(m[[0, 1, 3]], m0[[0, 1, 3]])
    x[0, 1, ids[0, 1]] = -math.inf  # a token that the mask of the vocabulary forbids
    x[1, 2, ids[1, 2]] = -3000.0    # ref - logp past the exponential's range
    plain, with_ref = run(x, None), run(x, ref)
    assert all(torch.isfinite(u).all() for u in (*plain[0][:2], *plain[0][3:]))
    assert all(torch.equal(u, v) for u, v in zip(plain[0], with_ref[0]))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gradients_just_inside_the_vector_path(dev, dtype):
    """|M| just below 1024, where 16-bit gradients by vectors are least exact."""
    x, ids, mask = make(5, 4096, "f32", seed=7, counted=1.1)
    x = (x + 478.0).to(DT[dtype])
    top = x.double().amax(1) / (0.7 * math.log(2.0)) + 4
    assert 1000 < top.min() and top.max() < 1023
    logp, ent, p, tol, _ = bounds(x, ids, mask, 0.7)
    coef = torch.tensor([1.0, -2.0, 0.5, 3.0, -0.25])
    leaf = x.to(dev).requires_grad_()
    got = _ops().token_logprobs(leaf, ids.to(dev), temperature=0.7)
    within(got, logp, tol)
    grad, = torch.autograd.grad(got, leaf, coef.to(dev))
    want = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy(), 0.7)
    extra = 2.0 ** -13 * np.abs(coef.numpy() / 0.7)[:, None] * p
    within(grad, want, grad_bound(want, p, coef.double().numpy(), 0.7, dtype) + extra)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fused", [True, False])
def test_the_scale_is_more_than_one_float(dev, dtype, fused):
    """log2(e) / 0.7 rounded to float32 is off by 2.0e-8, and every logp with it: a loss whose
    advantages cancel shows it. Each row has one logit of 0, its token's between -60 and -28
    and -inf elsewhere, so S is exact to e^(-28 / 0.7) = 4e-18 and logp is x / T to float64's
    roundings. The tokens of the positive advantages lie 16 below the others in the mean: one
    float32 would move the loss by 2.0e-8 * 16 / 0.7 / 2 = 2.3e-7."""
    b, s, vocab = 8, 8, 1000
    g = torch.Generator().manual_seed(12)
    tok = -(torch.arange(64) % 16).float() - 28.0
    tok[:32] -= 16.0
    x = torch.full((64, vocab), -math.inf)
    ids = torch.randint(1, vocab, (64,), generator=g)
    x[:, 0], x[torch.arange(64), ids] = 0.0, tok
    logp = tok.double().numpy() / 0.7
    adv = torch.tensor([1.0] * 4 + [-1.0] * 4)
    old = torch.from_numpy(np.float32(logp)).view(b, s)
    want, _, _ = P.policy_loss(logp.reshape(b, s), old.numpy(), adv.numpy(), np.ones((b, s), bool))
    leaf = x.view(b, s, vocab).to(DT[dtype]).to(dev).requires_grad_(fused)
    loss, got, _ = _ops().fused_grpo_loss(leaf, ids.view(b, s).to(dev), old.to(dev), adv.to(dev),
                                          temperature=0.7)
    assert abs(want) < 1e-5  # what old's rounding leaves
    # float32's rounding of the loss, S, and float64's of logp (86 * 2^-52) and of the sums
    assert abs(float(loss.detach()) - want) <= E * abs(want) + 1e-13
    within(got, logp.reshape(b, s), 1.01 * E * np.abs(logp.reshape(b, s)))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab, t", [(2403, 1.0), (20803, 0.7), (40003, 1.0), (57003, 0.9)])
def test_gradient_of_the_one_pass_in_64_bits(dev, dtype, vocab, t):
    """The gradient that the forward makes, for an upstream gradient of 1, against the oracle."""
    b, s = 2, 4
    x, ids, old, ref, adv, mask, logp, p = loss_inputs(b, s, vocab, dtype, seed=vocab, t=t)
    _, _, d = P.policy_loss(logp.reshape(b, s), old, adv, mask, ref, 0.2, 0.28, math.inf, 0.04,
                            "tokens")
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    leaf = put(x).requires_grad_()
    loss, _, _ = _ops().fused_grpo_loss(leaf, put(ids), put(old), put(adv), put(mask),
                                        ref_logps=put(ref), temperature=t, eps_high=0.28, beta=0.04)
    grad, = torch.autograd.grad(loss, leaf)
    coef = d.reshape(-1)
    at = ids.clamp(min=0).reshape(-1).numpy()
    want = P.logits_grad(p, at, mask.reshape(-1), coef, t)
    # the row's factor as in test_fused_loss_and_gradient; 16-bit gradients by vectors 2^-13
    top = float((E * (vocab / 512 + 24 + 2 * np.abs(logp) + math.log(vocab))).max())
    slack = (np.abs(coef) * 4 + 0.1) * top
    tol = grad_bound(want, p, coef, t, dtype) + (slack / t)[:, None] * (
        p + (np.arange(vocab)[None] == at[:, None]))
    extra = 0.0 if dtype == "f32" else 2.0 ** -13 * np.abs(coef / t)[:, None] * p
    within(grad, want, (tol + extra) * mask.reshape(-1, 1))


def test_tokens_without_an_advantage(dev):
    """A = 0: no gain and no gradient at any ratio; the token counts as moving up to delta, on
    either side of the clip, and as stopped beyond it."""
    r = torch.tensor([[0.5, 1.0, 1.1, 1.9, 3.0, 7.0]], dtype=torch.float64)
    logp = torch.full_like(r, -2.0)
    old = (logp - r.log()).float()
    adv = torch.zeros(1)
    for delta, stopped in ((None, 0), (4.0, 1)):
        want, metrics, grad = P.policy_loss(logp.numpy(), old.numpy(), adv.numpy(),
                                            np.ones((1, 6), bool), delta=delta or math.inf)
        leaf = logp.float().to(dev).requires_grad_()
        loss, m = _ops().grpo_policy_loss(leaf, old.to(dev), adv.to(dev), delta=delta)
        loss.backward()
        assert loss == want == 0 and not leaf.grad.any() and not grad.any()
        assert float(m[1]) == np.float32(stopped / 6) == np.float32(metrics[1])


def test_log_probabilities_are_read_as_float32(dev):
    """float64 log-probabilities are taken to float32 first, and their gradient is float32's."""
    logp, old, _, adv, mask = tokens(3, 9, seed=4)
    put = lambda a: torch.as_tensor(a).to(dev)  # noqa: E731
    wide = (put(logp).double() + 2.0 ** -40).requires_grad_()
    leaf = put(logp).requires_grad_()
    one = _ops().grpo_policy_loss(wide, put(old).double(), put(adv).double(), put(mask))[0]
    two = _ops().grpo_policy_loss(leaf, put(old), put(adv), put(mask))[0]
    one.backward()
    two.backward()
    assert torch.equal(one, two) and wide.grad.dtype == torch.float64
    assert torch.equal(wide.grad, leaf.grad.double())


@pytest.mark.parametrize("shape", [(0, 4, 33), (3, 0, 33), (1500, 0, 33), (0, 0, 1)])
@pytest.mark.parametrize("masked", [True, False])
def test_logits_of_no_positions(dev, shape, masked):
    x = torch.zeros(shape, dtype=torch.bfloat16, device=dev, requires_grad=True)
    ids = torch.zeros(shape[:2], dtype=torch.int64, device=dev)
    mask = torch.ones(shape[:2], dtype=torch.bool, device=dev) if masked else None
    adv = torch.ones(shape[0], device=dev)
    for normalizer in ("tokens", "sequences", 3.0):
        loss, logp, metrics = _ops().fused_grpo_loss(x, ids, None, adv, mask, normalizer=normalizer)
        grad, = torch.autograd.grad(loss, x)
        assert loss == 0 and not metrics.any() and logp.shape == shape[:2] and grad.shape == shape
    logp, ent = _ops().token_logprobs(x, ids, mask, return_entropy=True)
    grad, = torch.autograd.grad(logp.sum(), x)
    assert logp.shape == ent.shape == shape[:2] and grad.shape == shape


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_an_expanded_leaf_gets_the_sum(dev, dtype):
    """One row of logits for every position (stride 0): the gradient is the sum over them."""
    vocab = 777
    row, ids, _ = make(6, vocab, dtype, seed=3, counted=1.1)
    row = row[:1]
    leaf = row.to(dev).requires_grad_()
    coef = torch.tensor([1.0, 0.5, -0.25, 2.0, -1.0, 0.125])
    for view in (leaf.expand(6, vocab), leaf[None].expand(2, 3, vocab)):
        got = _ops().token_logprobs(view, ids.view(view.shape[:-1]).to(dev))
        grad, = torch.autograd.grad(got, leaf, coef.view(got.shape).to(dev))
        x = row.expand(6, vocab)
        mask = torch.ones(6, dtype=torch.bool)
        logp, _, p, tol, _ = bounds(x, ids, mask, 1.0)
        within(got.reshape(-1), logp, tol)
        each = P.logits_grad(p, ids.numpy(), mask.numpy(), coef.double().numpy())
        # each row rounded to the type, then five additions in it
        size = np.abs(each).sum(0)
        half = torch.finfo(DT[dtype]).eps / 2
        bound = grad_bound(each, p, coef.double().numpy(), 1.0, dtype).sum(0)
        within(grad[0], each.sum(0), bound + 5 * half * size + 5 * 2.0 ** -25)

"""CPU pins of ``oracle.policy_loss``: torch's float64 autograd, differences, known answers."""

import math

import numpy as np
import pytest
import torch

from oracle import policy_loss as P


def test_philox_known_answers():
    # the generator's published vectors: all zeros, all ones, digits of pi
    got = P.philox(np.zeros((1, 4), np.uint32), (0, 0))[0]
    assert [hex(v) for v in got] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    got = P.philox(np.full((1, 4), 0xFFFFFFFF, np.uint32), (0xFFFFFFFF, 0xFFFFFFFF))[0]
    assert [hex(v) for v in got] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]
    got = P.philox(np.array([[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], np.uint32),
                   (0xA4093822, 0x299F31D0))[0]
    assert [hex(v) for v in got] == ["0xd16cfe09", "0x94fdcceb", "0x5001e420", "0x24126ea1"]


@pytest.mark.parametrize("p", [0.0, 0.05, 0.5, 0.99])
def test_dropout_factors_keep_the_mean(p):
    f = P.dropout_factors(400_003, p, 7, 2 ** 40 + 3)
    t = math.floor(p * 65536 + 0.5)
    assert f.shape == (400_003,)
    assert set(np.unique(f)) <= {0.0, 65536 / (65536 - t)}
    sd = math.sqrt(p * (1 - p) / f.size)
    assert abs((f == 0).mean() - t / 65536) <= 6 * sd
    other = P.dropout_factors(400_003, p, 7, 2 ** 40 + 4)
    assert p == 0 or (f != other).any()


def _tokens(seed=0, b=5, s=7):
    g = np.random.default_rng(seed)
    logp = -3 * g.random((b, s))
    old, ref = logp + 0.5 * g.standard_normal((b, s)), logp + 0.3 * g.standard_normal((b, s))
    mask = g.random((b, s)) < 0.7
    mask[1] = False  # a sequence of which nothing counts
    return logp, old, ref, g.standard_normal(b), mask


@pytest.mark.parametrize("normalizer", ["tokens", "sequences", 40.0])
@pytest.mark.parametrize("delta", [math.inf, 1.5, 1.05])
@pytest.mark.parametrize("beta", [0.0, 0.3])
def test_policy_loss_is_torch_autograds(normalizer, delta, beta):
    logp, old, ref, adv, mask = _tokens()
    loss, metrics, grad = P.policy_loss(logp, old, adv, mask, ref if beta else None, 0.2, 0.28,
                                        delta, beta, normalizer)
    x = torch.tensor(logp, requires_grad=True)
    r, a, m = (x - torch.tensor(old)).exp(), torch.tensor(adv)[:, None], torch.tensor(mask)
    term = -torch.minimum(r.clamp(max=delta) * a, r.clamp(0.8, 1.28) * a)
    if beta:
        q = torch.tensor(ref) - x
        term = term + beta * (q.exp() - q - 1)
    n = m.double().sum(1, keepdim=True)
    if normalizer == "sequences":
        w = m / n.clamp(min=1) / (n > 0).sum()
    else:
        w = m.double() / (n.sum() if normalizer == "tokens" else normalizer)
    want = (term * w).sum()
    want.backward()
    assert loss == pytest.approx(want.item(), rel=1e-12)
    np.testing.assert_allclose(grad, x.grad.numpy(), rtol=1e-12, atol=1e-15)
    assert metrics[0] == pytest.approx(r[m].mean().item(), rel=1e-12)


def test_logits_grad_is_the_difference_quotient():
    g = np.random.default_rng(3)
    x, ids, mask = g.standard_normal((4, 9)), np.array([0, 8, 3, 2]), np.array([1, 1, 0, 1], bool)
    coef, t = g.standard_normal(4), 0.7
    logp, ent, p = P.token_logprobs(x, ids, mask, t)
    want = torch.log_softmax(torch.tensor(x) / t, -1)
    at = want[torch.arange(4), torch.tensor(ids)].numpy() * mask
    np.testing.assert_allclose(logp, at, rtol=1e-12)
    np.testing.assert_allclose(ent, -(want.exp() * want).sum(-1).numpy() * mask, rtol=1e-12)
    grad, h = P.logits_grad(p, ids, mask, coef, t), 1e-6
    for r in range(4):
        for v in range(9):
            up, down = x.copy(), x.copy()
            up[r, v] += h
            down[r, v] -= h
            d = (P.token_logprobs(up, ids, mask, t)[0] - P.token_logprobs(down, ids, mask, t)[0])
            assert grad[r, v] == pytest.approx((d * coef).sum() / (2 * h), abs=1e-8)

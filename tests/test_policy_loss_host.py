"""Refusals of the policy update's operators, made on the host before any launch."""

import ctypes
import math

import pytest
import torch

from grpo_mi355x import _lib
from grpo_mi355x.kernels import dropout, policy_loss


def test_tensors_off_the_device_are_refused():
    x, ids = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="ROCm/HIP device"):
        policy_loss.token_logprobs(x, ids)
    with pytest.raises(ValueError, match="ROCm/HIP device"):
        policy_loss.fused_grpo_loss(x, ids, None, torch.zeros(2))
    with pytest.raises(ValueError, match="ROCm/HIP device"):
        policy_loss.grpo_policy_loss(torch.zeros(2, 3), None, torch.zeros(2))
    with pytest.raises(ValueError, match="ROCm/HIP device"):
        dropout.counter_dropout(torch.zeros(4), 0.1, torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("kw, message", [
    (dict(eps_low=-0.1), "eps_low"), (dict(eps_high=math.nan), "eps_low and eps_high"),
    (dict(delta=0.0), "delta"), (dict(beta=-1.0), "beta"), (dict(beta=math.inf), "beta"),
    (dict(beta=0.1), "ref_logps"), (dict(normalizer="rows"), "normalizer"),
    (dict(normalizer=0.0), "normalizer"), (dict(normalizer=math.nan), "normalizer"),
])
def test_policy_parameters_are_refused(kw, message):
    with pytest.raises(ValueError, match=message):
        policy_loss.grpo_policy_loss(torch.zeros(2, 3), None, torch.zeros(2), **kw)
    with pytest.raises(ValueError, match=message):
        policy_loss.fused_grpo_loss(torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64),
                                    None, torch.zeros(2), **kw)


def test_shapes_of_the_tokens_are_refused():
    dev, shape = torch.device("cpu"), (2, 3)
    make = policy_loss._Tokens
    good = torch.zeros(2)
    with pytest.raises(ValueError, match="positions"):
        make(dev, (2, 3, 4), None, None, good, None)
    with pytest.raises(ValueError, match="old_logps must be"):
        make(dev, shape, torch.zeros(2, 4), None, good, None)
    with pytest.raises(ValueError, match="ref_logps must be a floating"):
        make(dev, shape, None, torch.zeros(2, 3, dtype=torch.int64), good, None)
    with pytest.raises(ValueError, match="advantages must be"):
        make(dev, shape, None, None, torch.zeros(3), None)
    with pytest.raises(ValueError, match="advantages must be"):
        make(dev, shape, None, None, torch.zeros(3, 2), None)
    with pytest.raises(ValueError, match="mask must be"):
        make(dev, shape, None, None, good, torch.ones(3, 2, dtype=torch.bool))
    with pytest.raises(ValueError, match="must be on cpu"):
        make(dev, shape, None, None, torch.zeros(2, device="meta"), None)


@pytest.mark.parametrize("p", [-0.1, 1.0, math.nan, 1 - 2 ** -18])
def test_dropout_probability_is_refused(p):
    with pytest.raises(ValueError, match="dropout p"):
        dropout.check_dropout(p, torch.zeros(2, dtype=torch.int64), torch.device("cpu"))


def test_dropout_state_is_refused():
    cpu = torch.device("cpu")
    for rng in (torch.zeros(2), torch.zeros(3, dtype=torch.int64),
                torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="two values"):
            dropout.check_dropout(0.1, rng, cpu)
    with pytest.raises(ValueError, match="must be on"):
        dropout.check_dropout(0.1, torch.zeros(2, dtype=torch.int64), torch.device("meta"))


# The addresses below are never read: every call is refused, or has nothing to do.
FAKE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.library()


def _rows(lib, dtype=0, sb=8, ss=8, b=2, s=3, v=8, ids=FAKE, t=1.0, x=FAKE, logp=FAKE, stat=FAKE):
    return lib.grpo_token_logprobs(x, dtype, sb, ss, b, s, v, ids, None, t, logp, None, stat, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(sb=-1), dict(b=-1), dict(v=0), dict(ids=None), dict(t=0.0),
    dict(t=math.inf), dict(t=math.nan), dict(t=1e-36), dict(x=None), dict(x=FAKE + 1),
    dict(logp=None), dict(stat=FAKE + 4), dict(b=1 << 20, s=4),
])
def test_c_entry_refuses_logits(lib, kw):
    assert _rows(lib, **kw) == -1, lib.grpo_last_error()


def test_c_entry_with_no_rows_does_nothing(lib):
    assert _rows(lib, b=0, x=None, ids=None, logp=None) == 0
    assert lib.grpo_token_logprobs_backward(None, 0, 0, 0, 0, 5, 8, None, None, 1.0, None, None,
                                            None, None, None) == 0
    assert lib.grpo_dropout(None, None, 0, 0, 0.1, FAKE, None) == 0


def _policy(**kw):
    p = dict(eps_low=0.2, eps_high=0.2, delta=math.inf, beta=0.0, denom=1.0, normalizer=0)
    p.update(kw)
    return _lib.Policy(**p)


def _loss(lib, policy, logp=FAKE, adv=FAKE, b=2, s=3, ws=FAKE, nbytes=1 << 20):
    return lib.grpo_policy_loss(logp, None, None, adv, 0, None, b, s,
                                None if policy is None else ctypes.byref(policy), FAKE, FAKE, ws,
                                nbytes, None)


@pytest.mark.parametrize("kw", [
    dict(eps_low=-1.0), dict(eps_high=math.nan), dict(delta=0.0), dict(delta=math.nan),
    dict(beta=-1.0), dict(beta=math.inf), dict(normalizer=3), dict(normalizer=2, denom=0.0),
])
def test_c_entry_refuses_policies(lib, kw):
    assert _loss(lib, _policy(**kw)) == -1, lib.grpo_last_error()


def test_c_entry_refuses_buffers(lib):
    assert _loss(lib, None) == -1
    assert _loss(lib, _policy(), logp=None) == -1
    assert _loss(lib, _policy(), adv=None) == -1
    assert _loss(lib, _policy(), ws=None) == -1
    assert _loss(lib, _policy(), ws=FAKE + 8) == -1
    need = lib.grpo_policy_loss_workspace_bytes(2, 3, 0)
    assert 0 < need <= lib.grpo_policy_loss_workspace_bytes(2, 3, 1)
    assert _loss(lib, _policy(), nbytes=need - 1) == -3
    assert _loss(lib, _policy(), b=1 << 16, s=1 << 16) == -1


@pytest.mark.parametrize("kw", [dict(p=1.0), dict(p=-0.5), dict(p=math.nan), dict(dtype=3),
                                dict(n=-1), dict(x=None), dict(rng=None), dict(rng=FAKE + 4),
                                dict(p=1 - 2 ** -18)])
def test_c_entry_refuses_dropout(lib, kw):
    a = dict(x=FAKE, y=FAKE, n=8, dtype=0, p=0.1, rng=FAKE)
    a.update(kw)
    assert lib.grpo_dropout(a["x"], a["y"], a["n"], a["dtype"], a["p"], a["rng"], None) == -1

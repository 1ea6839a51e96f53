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
    dev, shape = torch.device("cpu"), torch.Size((2, 3))

    def make(old=None, ref=None, adv=torch.zeros(2), shape=shape):
        return policy_loss._check_tokens(shape, dev, old, ref, adv)

    with pytest.raises(ValueError, match="positions"):
        make(shape=torch.Size((2, 3, 4)))
    with pytest.raises(ValueError, match="old_logps must be"):
        make(old=torch.zeros(2, 4))
    with pytest.raises(ValueError, match="ref_logps must be a floating"):
        make(ref=torch.zeros(2, 3, dtype=torch.int64))
    for adv in (torch.zeros(3), torch.zeros(3, 2), torch.zeros(2, 3, 1), torch.zeros(())):
        with pytest.raises(ValueError, match="advantages must be"):
            make(adv=adv)
    with pytest.raises(ValueError, match="mask must be"):
        policy_loss._mask_rows(torch.ones(3, 2, dtype=torch.bool), shape, dev)
    for name in ("old", "ref", "adv"):
        with pytest.raises(ValueError, match="must be on cpu"):
            make(**{name: torch.zeros(2 if name == "adv" else shape, device="meta")})


def test_policy_parameters_are_read_at_every_call():
    """The parameters kept for equal arguments are those of the values, not of a tensor."""
    n = torch.tensor(4.0)
    args = (0.2, 0.2, None, 0.0)
    four = policy_loss._policy(*args, n, None)._obj
    n.fill_(8.0)
    eight = policy_loss._policy(*args, n, None)._obj
    assert (four.denom, eight.denom) == (4.0, 8.0)
    assert policy_loss._policy(*args, 8, None)._obj.normalizer == 2
    assert policy_loss._policy(*args, "sequences", None)._obj.normalizer == 1


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
    return lib.grpo_token_logprobs(x, dtype, sb, ss, b, s, v, ids, None, t, logp, None, stat, None,
                                   0, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(sb=-1), dict(b=-1), dict(v=0), dict(ids=None), dict(t=0.0),
    dict(t=math.inf), dict(t=math.nan), dict(t=1e-36), dict(x=None), dict(x=FAKE + 1),
    dict(logp=None), dict(stat=FAKE + 4), dict(b=1 << 20, s=4), dict(v=(1 << 30) + 1),
    dict(t=1e21),
])
def test_c_entry_refuses_logits(lib, kw):
    assert _rows(lib, **kw) == -1, lib.grpo_last_error()


def test_c_entry_wants_a_workspace_where_rows_are_cut(lib):
    need = lib.grpo_token_logprobs_workspace_bytes(0, 8, 1, 151936)
    assert need > 0
    for rows, vocab in ((4096, 151936), (8, 2000)):  # enough rows; short ones
        assert lib.grpo_token_logprobs_workspace_bytes(0, rows, 1, vocab) == 0
    args = (FAKE, 0, 151936, 0, 8, 1, 151936, FAKE, None, 1.0, FAKE, None, None)
    assert lib.grpo_token_logprobs(*args, None, need, None) == -1
    assert lib.grpo_token_logprobs(*args, FAKE + 8, need, None) == -1
    assert lib.grpo_token_logprobs(*args, FAKE, need - 1, None) == -3


def test_rows_that_are_made_in_one_pass(lib):
    one = lib.grpo_policy_loss_logits_one_pass
    assert [one(0, 2, 3, v) for v in (1, 114688, 114689, 0)] == [1, 1, 0, 0]
    assert [one(2, 2, 3, v) for v in (50257, 57344, 57345)] == [1, 1, 0] and one(3, 2, 3, 8) == 0
    assert [one(2, 8, s, 151936) for s in (15, 16)] == [0, 1]


def test_c_entry_refuses_a_gradient_it_cannot_make(lib):
    need = 1 << 30

    def go(v, stat, coef, grad, sb=24):
        return lib.grpo_policy_loss_logits(
            FAKE, 0, v, v, 2, 3, v, FAKE, None, 1.0, None, None, FAKE, 0, ctypes.byref(_policy()),
            FAKE, FAKE, FAKE, stat, coef, grad, sb, 8, FAKE, need, None)

    assert go(8, FAKE, None, None) == -1 and go(8, FAKE + 4, FAKE, None) == -1
    assert go(8, None, None, FAKE) == -1  # no place for the statistics
    assert go(160000, FAKE, FAKE, FAKE) == -1 and go(8, FAKE, FAKE, FAKE + 1) == -1
    assert go(8, FAKE, FAKE, FAKE, sb=-1) == -1


def test_c_entry_with_no_rows_does_nothing(lib):
    assert _rows(lib, b=0, x=None, ids=None, logp=None) == 0
    assert lib.grpo_token_logprobs_backward(None, 0, 0, 0, 0, 5, 8, None, None, 1.0, None, None,
                                            None, None, 0, 0, None) == 0
    assert lib.grpo_dropout(None, None, 0, 0, 0.1, FAKE, None) == 0


def _policy(**kw):
    p = dict(eps_low=0.2, eps_high=0.2, delta=math.inf, beta=0.0, denom=1.0, normalizer=0)
    p.update(kw)
    return _lib.Policy(**p)


def _loss(lib, policy, logp=FAKE, adv=FAKE, b=2, s=3, ws=FAKE, nbytes=1 << 20):
    return lib.grpo_policy_loss(logp, None, None, adv, 0, None, b, s,
                                None if policy is None else ctypes.byref(policy), FAKE, FAKE, None,
                                ws, nbytes, None)


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
    need = lib.grpo_policy_loss_workspace_bytes(2, 3)
    assert 0 < need <= lib.grpo_policy_loss_logits_workspace_bytes(0, 2, 3, 8)
    assert _loss(lib, _policy(), nbytes=need - 1) == -3
    assert _loss(lib, _policy(), b=1 << 16, s=1 << 16) == -1


@pytest.mark.parametrize("kw", [dict(p=1.0), dict(p=-0.5), dict(p=math.nan), dict(dtype=3),
                                dict(n=-1), dict(x=None), dict(rng=None), dict(rng=FAKE + 4),
                                dict(x=FAKE + 1), dict(y=FAKE + 2, dtype=2),
                                dict(p=1 - 2 ** -18)])
def test_c_entry_refuses_dropout(lib, kw):
    a = dict(x=FAKE, y=FAKE, n=8, dtype=0, p=0.1, rng=FAKE)
    a.update(kw)
    assert lib.grpo_dropout(a["x"], a["y"], a["n"], a["dtype"], a["p"], a["rng"], None) == -1


@pytest.mark.parametrize("make, kept", [
    (lambda x: x, False),                       # contiguous and aligned: as it is
    (lambda x: x[:, :-1], True), (lambda x: x[:, 1:], True),
    (lambda x: x[..., 3:], False),              # a fifth of each row unused would be too much
    (lambda x: x[..., 1:], True),
    (lambda x: x[::2], False), (lambda x: x[:1].expand(4, -1, -1), False),
    (lambda x: x.transpose(0, 1), True), (lambda x: x[..., ::2], False),
    (lambda x: x[:, 1], False), (lambda x: x[1:2], True), (lambda x: x.view(-1, 9)[1:], True),
])
def test_the_gradients_rows_stand_as_the_logits_do(make, kept):
    """Rows of the gradient never overlap, and keep the logits' offsets where they can."""
    base = torch.zeros(5, 6, 9, dtype=torch.bfloat16)
    v = make(base)
    ids = torch.zeros(v.shape[:-1], dtype=torch.int64)
    x, _ = policy_loss._rows(v, ids, None, 1.0)
    g, sb, ss = policy_loss._empty_grad(v, x)
    assert g.shape == v.shape and g.dtype == v.dtype
    size = g.untyped_storage().nbytes() // 2
    at = [(g.data_ptr() - g.untyped_storage().data_ptr()) // 2 + b * sb + s * ss
          for b in range(x.shape[0]) for s in range(x.shape[1])]
    cells = torch.zeros(size, dtype=torch.int32)
    for a in at:
        assert a + 9 - (9 - v.shape[-1]) <= size
        cells[a:a + v.shape[-1]] += 1
    assert int(cells.max()) == 1 and int(cells.sum()) == v.numel()
    if kept:
        assert g.stride() == v.stride()
        rows = [x.data_ptr() + 2 * (b * x.stride(0) + s * x.stride(1))
                for b in range(x.shape[0]) for s in range(x.shape[1])]
        for a, r in zip(at, rows):
            assert (g.untyped_storage().data_ptr() + 2 * a - r) % 16 == 0
    else:
        assert g.is_contiguous()


def test_layers_with_counter_dropout():
    """Injected layers carry the dropout asked for; eval mode and p = 0 drop nothing."""
    from grpo_mi355x.core.lora import inject_lora_layers
    from grpo_mi355x.core.nf4 import Linear4bitNF4

    def model():
        m = torch.nn.Module()
        m.q_proj = Linear4bitNF4.from_weight(torch.randn(32, 64) * 0.02, None)
        return m

    for kw, kind in ((dict(), torch.nn.Identity), (dict(dropout=0.1), torch.nn.Dropout),
                     (dict(dropout=0.1, counter_dropout=True), dropout.CounterDropout),
                     (dict(counter_dropout=True), torch.nn.Identity)):
        m = model()
        assert inject_lora_layers(m, ["q_proj"], rank=4, verbose=False, **kw) == 1
        assert type(m.q_proj.lora_dropout) is kind
    d = dropout.CounterDropout(0.1)
    x = torch.ones(3)
    assert d.active() and not d.eval().active() and d(x) is x
    assert dropout.CounterDropout(0.0)(x) is x and "p=0.1" in repr(d)
    with pytest.raises(ValueError, match="dropout p"):
        dropout.CounterDropout(1.0)
    with pytest.raises(ValueError, match="dropout p"):
        dropout.CounterDropout(1 - 2 ** -18)  # rounds to 1 in steps of 1/65536
    torch.manual_seed(3)
    a = dropout.CounterDropout.draw(torch.device("cpu"))
    torch.manual_seed(3)
    assert torch.equal(a, dropout.CounterDropout.draw(torch.device("cpu")))
    assert a.dtype == torch.int64 and a.shape == (2,)

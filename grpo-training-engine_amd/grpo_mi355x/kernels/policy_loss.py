"""The policy update's loss on the HIP kernels (``csrc/policy_loss.hip``).

* ``token_logprobs``: log-probabilities of given tokens under a vocabulary of logits,
  with their gradient (the old, reference and current policy's log-probabilities,
  ``src/grpo/trainer.py:486-839``);
* ``grpo_policy_loss``: the two-sided clipped policy loss with a cap on the ratio and a
  KL term (``src/grpo/algorithm.py:115-254``) from per-token log-probabilities;
* ``fused_grpo_loss``: the loss straight from the logits (``src/triton_kernels/
  grpo_loss.py:571-625``), the vocabulary read once forward.

Positions are ``[batch, seq]``; ``logits[b, s]`` scores ``token_ids[b, s]`` (shifting
logits against tokens is the caller's slice: ``logits[:, :-1]`` is taken as it is, without
a copy).  ``mask`` says which positions count; the others are not read, whatever stands
there, and get logp 0 and gradient 0.  Softmax statistics, losses and gradients are
float32 or float64; the logits' gradient is rounded once, to the logits' type.
Arguments that do not fit raise ``ValueError``, a missing device ``ImportError``.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NORMALIZERS = {"tokens": 0, "sequences": 1}


def _on(device: torch.device):
    """The device's context where it is not the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}.")


def _float_rows(t: Optional[torch.Tensor], name: str, shape) -> Optional[torch.Tensor]:
    """A float32 contiguous tensor of ``shape`` (any float type is taken)."""
    if t is None:
        return None
    if not t.dtype.is_floating_point:
        raise ValueError(f"{name} must be a floating-point tensor, got {t.dtype}.")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}.")
    t = t.detach()
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _mask_rows(mask: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
    """The mask as contiguous bool (any type: nonzero counts)."""
    if mask is None:
        return None
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"mask must be {list(shape)}, got {list(mask.shape)}.")
    if mask.dtype != torch.bool:
        mask = mask != 0
    return mask if mask.is_contiguous() else mask.contiguous()


class _Rows:
    """Checked logits with their ids and mask, and the C arguments that describe them."""

    def __init__(self, logits, token_ids, mask, temperature):
        if logits.ndim < 2:
            raise ValueError(f"logits must be [..., vocab], got {list(logits.shape)}.")
        if not logits.is_cuda:
            raise ValueError("logits must be on the ROCm/HIP device.")
        if logits.dtype not in _DTYPES:
            raise ValueError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}.")
        lead = logits.shape[:-1]
        if tuple(token_ids.shape) != tuple(lead):
            raise ValueError(f"token_ids must be {list(lead)}, got {list(token_ids.shape)}.")
        if token_ids.dtype != torch.int64:
            raise ValueError(f"token_ids must be int64, got {token_ids.dtype}.")
        if logits.shape[-1] < 1:
            raise ValueError("logits must have a vocabulary of at least one token.")
        t = float(temperature)
        if not (0.0 < t < math.inf):
            raise ValueError(f"temperature must be positive and finite, got {temperature}.")
        _same_device(logits.device, token_ids=token_ids, mask=mask)
        x = logits.detach()
        if x.stride(-1) != 1 and x.shape[-1] > 1 or any(v < 0 for v in x.stride()):
            x = x.contiguous()
        if x.ndim > 3:
            x = x.reshape(-1, x.shape[-2], x.shape[-1])
        self.shape, self.t = tuple(lead), t
        self.x, self.ids = x, token_ids.contiguous()
        self.mask = _mask_rows(mask, lead)
        self.vocab = x.shape[-1]
        if x.ndim == 3:
            self.b, self.s, self.sb, self.ss = x.shape[0], x.shape[1], x.stride(0), x.stride(1)
        else:
            self.b, self.s, self.sb, self.ss = x.shape[0], 1, x.stride(0), 0
        if self.b * self.s >= 1 << 22:
            raise ValueError("at most 2**22 - 1 rows of logits in a call.")

    def args(self):
        return (self.x.data_ptr(), _DTYPES[self.x.dtype], self.sb, self.ss, self.b, self.s,
                self.vocab, self.ids.data_ptr(), _lib.ptr(self.mask), self.t)


def _grad_of(rows: _Rows, stat, coef, scale) -> torch.Tensor:
    """The logits' gradient, of the logits' shape."""
    out = torch.empty((*rows.shape, rows.vocab), dtype=rows.x.dtype, device=rows.x.device)
    with _on(out.device):
        rc = _lib.device_library().grpo_token_logprobs_backward(
            *rows.args(), stat.data_ptr(), coef.data_ptr(), _lib.ptr(scale), out.data_ptr(),
            _lib.stream_handle(out.device))
    if rc:
        _lib.check(rc, "grpo_token_logprobs_backward")
    return out


def _logprobs(rows: _Rows, entropy: bool, train: bool):
    dev, n = rows.x.device, rows.b * rows.s
    logp = torch.empty(rows.shape, dtype=torch.float32, device=dev)
    ent = torch.empty(rows.shape, dtype=torch.float32, device=dev) if entropy else None
    stat = torch.empty((n, 4), dtype=torch.float32, device=dev) if train else None
    with _on(dev):
        rc = _lib.device_library().grpo_token_logprobs(
            *rows.args(), logp.data_ptr(), _lib.ptr(ent), _lib.ptr(stat),
            _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, "grpo_token_logprobs")
    return logp, ent, stat


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, token_ids, mask, temperature, entropy):
        rows = _Rows(logits, token_ids, mask, temperature)
        logp, ent, stat = _logprobs(rows, entropy, True)
        ctx.save_for_backward(logits, rows.ids, rows.mask, stat)
        ctx.temperature = rows.t
        if ent is not None:
            ctx.mark_non_differentiable(ent)
        return logp, ent

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logp, _):
        logits, ids, mask, stat = ctx.saved_tensors
        rows = _Rows(logits, ids, mask, ctx.temperature)
        grad = _float_rows(grad_logp, "grad", rows.shape)
        return _grad_of(rows, stat, grad, None), None, None, None, None


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                   return_entropy: bool = False):
    """``log softmax(logits / temperature)`` at ``token_ids``, float32.

    ``logits [..., V]`` (bfloat16, float16 or float32; any row strides), ``token_ids``
    int64 of the leading shape, ``mask`` of that shape (None: every position counts).
    Differentiable by ``logits``.  With ``return_entropy`` also the entropy of each
    position's distribution, which carries no gradient.  An id outside the vocabulary at a
    counted position gives NaN there."""
    if torch.is_grad_enabled() and logits.requires_grad:
        logp, ent = _TokenLogprobs.apply(logits, token_ids, mask, temperature, return_entropy)
    else:
        logp, ent, _ = _logprobs(_Rows(logits, token_ids, mask, temperature), return_entropy,
                                 False)
    return (logp, ent) if return_entropy else logp


# ------------------------------------------------------------ policy loss --

def _policy(eps_low, eps_high, delta, beta, normalizer) -> _lib.Policy:
    eps_low, eps_high, beta = float(eps_low), float(eps_high), float(beta)
    cap = math.inf if delta is None else float(delta)
    if not (0.0 <= eps_low < math.inf and 0.0 <= eps_high < math.inf):
        raise ValueError("eps_low and eps_high must be >= 0 and finite.")
    if not cap > 0.0:
        raise ValueError(f"delta must be positive, got {delta}.")
    if not 0.0 <= beta < math.inf:
        raise ValueError(f"beta must be >= 0 and finite, got {beta}.")
    if isinstance(normalizer, str):
        if normalizer not in _NORMALIZERS:
            raise ValueError(f"normalizer must be 'tokens', 'sequences' or a number, got "
                             f"{normalizer!r}.")
        return _lib.Policy(eps_low, eps_high, cap, beta, 1.0, _NORMALIZERS[normalizer])
    denom = float(normalizer)
    if not 0.0 < denom < math.inf:
        raise ValueError(f"the normalizer must be positive and finite, got {normalizer}.")
    return _lib.Policy(eps_low, eps_high, cap, beta, denom, 2)


class _Tokens:
    """Checked per-token inputs of the policy loss, and the C arguments they make."""

    def __init__(self, device, shape, old_logps, ref_logps, advantages, mask):
        if len(shape) != 2:
            raise ValueError(f"positions must be [batch, seq], got {list(shape)}.")
        _same_device(device, old_logps=old_logps, ref_logps=ref_logps, advantages=advantages,
                     mask=mask)
        self.old = _float_rows(old_logps, "old_logps", shape)
        self.ref = _float_rows(ref_logps, "ref_logps", shape)
        self.per_token = advantages.ndim == 2
        self.adv = _float_rows(advantages, "advantages",
                               shape if self.per_token else shape[:1])
        self.mask = _mask_rows(mask, shape)
        self.shape = tuple(shape)

    def args(self):
        return (_lib.ptr(self.old), _lib.ptr(self.ref), self.adv.data_ptr(), self.per_token)


def _need_ref(beta: float, ref_logps) -> None:
    if beta and ref_logps is None:
        raise ValueError("beta > 0 needs ref_logps.")


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, tokens, policy):
        lp = _float_rows(logps, "logps", tokens.shape)
        loss, metrics, ws = _policy_loss(lp, tokens, policy)
        ctx.save_for_backward(logps, tokens.old, tokens.ref, tokens.adv, tokens.mask, ws)
        ctx.per_token, ctx.policy = tokens.per_token, policy
        ctx.mark_non_differentiable(metrics)
        return loss, metrics

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        logps, old, ref, adv, mask, ws = ctx.saved_tensors
        lp = _float_rows(logps, "logps", logps.shape)
        g = grad_loss.to(torch.float32).contiguous()
        out = torch.empty_like(lp)
        b, s = lp.shape
        with _on(lp.device):
            rc = _lib.device_library().grpo_policy_loss_backward(
                lp.data_ptr(), _lib.ptr(old), _lib.ptr(ref), adv.data_ptr(), ctx.per_token,
                _lib.ptr(mask), b, s, ctypes.byref(ctx.policy), g.data_ptr(), out.data_ptr(),
                ws.data_ptr(), ws.numel(), _lib.stream_handle(lp.device))
        if rc:
            _lib.check(rc, "grpo_policy_loss_backward")
        return (out if out.dtype == logps.dtype else out.to(logps.dtype)), None, None


def _policy_loss(lp, tokens, policy):
    lib, dev, (b, s) = _lib.device_library(), lp.device, tokens.shape
    loss = torch.empty((), dtype=torch.float32, device=dev)
    metrics = torch.empty(4, dtype=torch.float32, device=dev)
    nbytes = lib.grpo_policy_loss_workspace_bytes(b, s, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = lib.grpo_policy_loss(
            lp.data_ptr(), *tokens.args(), _lib.ptr(tokens.mask), b, s, ctypes.byref(policy),
            loss.data_ptr(), metrics.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, "grpo_policy_loss")
    return loss, metrics, ws


def grpo_policy_loss(logps: torch.Tensor, old_logps: Optional[torch.Tensor],
                     advantages: torch.Tensor, mask: Optional[torch.Tensor] = None, *,
                     ref_logps: Optional[torch.Tensor] = None, eps_low: float = 0.2,
                     eps_high: float = 0.2, delta: Optional[float] = None, beta: float = 0.0,
                     normalizer="tokens"):
    """The two-sided clipped policy loss with a KL term; ``(loss, metrics)``.

    Per counted token, with ``r = exp(logps - old_logps)``, ``q = ref_logps - logps`` and
    its advantage ``A``::

        l = beta (exp(q) - q - 1) - min(min(r, delta) A, clip(r, 1 - eps_low, 1 + eps_high) A)

    ``loss`` is the sum of ``l`` over the counted tokens divided by their number
    (``normalizer="tokens"``), the mean over sequences of each one's mean
    (``"sequences"``; sequences without a counted token are left out), or the sum divided
    by a number.  ``logps``, ``old_logps`` (None: the policy's own, r = 1) and
    ``ref_logps`` are ``[batch, seq]``, ``advantages`` ``[batch]`` or ``[batch, seq]``;
    computed in float64, differentiable by ``logps`` alone.  ``metrics`` (float32 [4], no
    gradient) are means over the counted tokens: r, the share whose gain no longer moves
    with r (clipped or capped), ``exp(q) - q - 1`` and ``old_logps - logps``.  With nothing
    counted, loss and metrics are 0."""
    policy = _policy(eps_low, eps_high, delta, beta, normalizer)
    _need_ref(policy.beta, ref_logps)
    if not logps.is_cuda:
        raise ValueError("logps must be on the ROCm/HIP device.")
    tokens = _Tokens(logps.device, logps.shape, old_logps, ref_logps, advantages, mask)
    if torch.is_grad_enabled() and logps.requires_grad:
        return _PolicyLoss.apply(logps, tokens, policy)
    loss, metrics, _ = _policy_loss(_float_rows(logps, "logps", logps.shape), tokens, policy)
    return loss, metrics


class _LogitsLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, tokens, policy):
        loss, logp, metrics, stat, coef = _logits_loss(rows, tokens, policy, True)
        ctx.save_for_backward(logits, rows.ids, rows.mask, stat, coef)
        ctx.temperature = rows.t
        ctx.mark_non_differentiable(logp, metrics)
        return loss, logp, metrics

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        logits, ids, mask, stat, coef = ctx.saved_tensors
        rows = _Rows(logits, ids, mask, ctx.temperature)
        g = grad_loss.to(torch.float32).contiguous()
        return _grad_of(rows, stat, coef, g), None, None, None


def _logits_loss(rows: _Rows, tokens: _Tokens, policy, train: bool):
    lib, dev, n = _lib.device_library(), rows.x.device, rows.b * rows.s
    loss = torch.empty((), dtype=torch.float32, device=dev)
    metrics = torch.empty(4, dtype=torch.float32, device=dev)
    logp = torch.empty(rows.shape, dtype=torch.float32, device=dev)
    stat = torch.empty((n, 4), dtype=torch.float32, device=dev) if train else None
    coef = torch.empty(n, dtype=torch.float32, device=dev) if train else None
    nbytes = lib.grpo_policy_loss_workspace_bytes(rows.b, rows.s, 1)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = lib.grpo_policy_loss_logits(
            *rows.args(), *tokens.args(), ctypes.byref(policy), loss.data_ptr(), logp.data_ptr(),
            metrics.data_ptr(), _lib.ptr(stat), _lib.ptr(coef), ws.data_ptr(), nbytes,
            _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, "grpo_policy_loss_logits")
    return loss, logp, metrics, stat, coef


def fused_grpo_loss(logits: torch.Tensor, token_ids: torch.Tensor,
                    old_logps: Optional[torch.Tensor], advantages: torch.Tensor,
                    mask: Optional[torch.Tensor] = None, *,
                    ref_logps: Optional[torch.Tensor] = None, temperature: float = 1.0,
                    eps_low: float = 0.2, eps_high: float = 0.2, delta: Optional[float] = None,
                    beta: float = 0.0, normalizer="tokens"):
    """``grpo_policy_loss`` of ``token_logprobs(logits, token_ids)``, the log-probabilities
    never leaving the call's precision; ``(loss, logps, metrics)``.

    ``logits [batch, seq, V]``; the other arguments are those of the two operators.
    Differentiable by ``logits`` alone; ``logps`` (float32, 0 where not counted) and
    ``metrics`` carry no gradient."""
    policy = _policy(eps_low, eps_high, delta, beta, normalizer)
    _need_ref(policy.beta, ref_logps)
    if logits.ndim != 3:
        raise ValueError(f"logits must be [batch, seq, vocab], got {list(logits.shape)}.")
    rows = _Rows(logits, token_ids, mask, temperature)
    tokens = _Tokens(logits.device, rows.shape, old_logps, ref_logps, advantages, rows.mask)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _LogitsLoss.apply(logits, rows, tokens, policy)
    loss, logp, metrics, _, _ = _logits_loss(rows, tokens, policy, False)
    return loss, logp, metrics


__all__ = ["token_logprobs", "grpo_policy_loss", "fused_grpo_loss"]

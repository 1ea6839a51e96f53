"""The policy update's loss on the HIP kernels (``csrc/policy_loss.hip``).

* ``token_logprobs``: log-probabilities of given tokens under a vocabulary of logits,
  with their gradient (the old, reference and current policy's log-probabilities,
  ``src/grpo/trainer.py:486-839``);
* ``grpo_policy_loss``: the two-sided clipped policy loss with a cap on the ratio and a
  KL term (``src/grpo/algorithm.py:115-254``) from per-token log-probabilities;
* ``fused_grpo_loss``: the loss straight from the logits (``src/triton_kernels/
  grpo_loss.py:571-625``), the vocabulary read once for the loss and its gradient.

Positions are ``[batch, seq]``; ``logits[b, s]`` scores ``token_ids[b, s]`` (shifting
logits against tokens is the caller's slice: ``logits[:, :-1]`` is taken as it is, without
a copy).  ``mask`` says which positions count; the others are not read, whatever stands
there, and get logp 0 and gradient 0.  Softmax statistics, losses and gradients are
float32 or float64; the logits' gradient is rounded once, to the logits' type.
Arguments that do not fit raise ``ValueError``, a missing device ``ImportError``; forward-mode
derivatives raise (``RuntimeError``), as they do from any function that has none.  Nothing is
kept between calls: every buffer is the call's own.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .ops import derivative_recorded

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NORMALIZERS = {"tokens": 0, "sequences": 1}
_MAX_ROWS = 1 << 22
_MAX_VOCAB = 1 << 30


def _run(device: torch.device, name: str, *args) -> None:
    """The C entry point on the device's current stream."""
    fn = getattr(_lib.device_library(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _lib.stream_handle(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, name)


def _once(backward):
    """``once_differentiable``, its bookkeeping left out where no graph is being made."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


# ------------------------------------------------------- argument checks --

def _float_rows(t: Optional[torch.Tensor], name: str, shape,
                device: torch.device) -> Optional[torch.Tensor]:
    """``t`` as a contiguous float32 tensor of ``shape`` without a graph."""
    if t is None:
        return None
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}.")
    if not t.dtype.is_floating_point:
        raise ValueError(f"{name} must be a floating-point tensor, got {t.dtype}.")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}.")
    if t.requires_grad:
        t = t.detach()
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _mask_rows(mask: Optional[torch.Tensor], shape,
               device: torch.device) -> Optional[torch.Tensor]:
    """The mask as contiguous bool (any type: nonzero counts)."""
    if mask is None:
        return None
    if mask.device != device:
        raise ValueError(f"mask must be on {device}, got {mask.device}.")
    if mask.shape != shape:
        raise ValueError(f"mask must be {list(shape)}, got {list(mask.shape)}.")
    if mask.dtype != torch.bool:
        mask = mask != 0
    return mask if mask.is_contiguous() else mask.contiguous()


def _check_logits(logits, token_ids, mask, temperature):
    """(contiguous ids, mask, temperature) that fit the logits."""
    if logits.ndim < 2:
        raise ValueError(f"logits must be [..., vocab], got {list(logits.shape)}.")
    if not logits.is_cuda:
        raise ValueError("logits must be on the ROCm/HIP device.")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}.")
    *lead, vocab = logits.shape
    lead = torch.Size(lead)
    if token_ids.shape != lead:
        raise ValueError(f"token_ids must be {list(lead)}, got {list(token_ids.shape)}.")
    if token_ids.dtype != torch.int64:
        raise ValueError(f"token_ids must be int64, got {token_ids.dtype}.")
    if token_ids.device != logits.device:
        raise ValueError(f"token_ids must be on {logits.device}, got {token_ids.device}.")
    if not vocab:
        raise ValueError("logits must have a vocabulary of at least one token.")
    if vocab > _MAX_VOCAB:
        raise ValueError(f"a vocabulary of at most {_MAX_VOCAB} tokens, got {vocab}.")
    if lead.numel() >= _MAX_ROWS:
        raise ValueError(f"at most {_MAX_ROWS - 1} rows of logits in a call.")
    t = float(temperature)
    if not 0.0 < t < math.inf:
        raise ValueError(f"temperature must be positive and finite, got {temperature}.")
    if not token_ids.is_contiguous():
        token_ids = token_ids.contiguous()
    return token_ids, _mask_rows(mask, lead, logits.device), t


def _rows(logits, ids, mask, t):
    """(the tensor read, the C arguments that describe its rows)."""
    x = logits.detach()
    if x.ndim == 2:
        x = x.unsqueeze(1)
    elif x.ndim > 3:
        x = x.reshape(-1, x.shape[-2], x.shape[-1])
    b, s, v = x.shape
    sb, ss, sv = x.stride()
    if sv != 1 and v > 1:
        x = x.contiguous()
        sb, ss, sv = x.stride()
    return x, (x.data_ptr(), _DTYPES[x.dtype], sb, ss, b, s, v, ids.data_ptr(), _lib.ptr(mask), t)


def _empty_grad(logits, x):
    """(a tensor for the logits' gradient, its row strides): rows as far from a 16-byte
    boundary as the logits' own, by their strides where those leave little unused."""
    b, s, v = x.shape
    shape, dev = logits.shape, x.device
    off = x.data_ptr() % 16 // x.element_size()
    if (off or not x.is_contiguous()) and x.data_ptr() == logits.data_ptr() and logits.ndim <= 3:
        sb, ss, _ = x.stride()
        rows = sorted((n, d) for n, d in ((ss, s), (sb, b)) if d > 1)
        extent, apart = v, True
        for stride, n in rows:  # the inner rows end before the next outer one begins
            apart = apart and stride >= extent
            extent += stride * (n - 1)
        if apart and extent <= 1.25 * b * s * v:
            buf = torch.empty(off + extent, dtype=x.dtype, device=dev)
            return buf.as_strided(shape, logits.stride(), off), sb, ss
    return torch.empty(shape, dtype=x.dtype, device=dev), s * v, v


# ---------------------------------------------------- log-probabilities --

@functools.lru_cache(maxsize=256)
def _logp_bytes(dtype: int, b: int, s: int, v: int) -> int:
    return _lib.library().grpo_token_logprobs_workspace_bytes(dtype, b, s, v)


def _grad_of(logits, ids, mask, t, stat: int, coef: int, scale) -> torch.Tensor:
    """The logits' gradient, of the logits' shape (stat, coef: addresses)."""
    x, rows = _rows(logits, ids, mask, t)
    out, sb, ss = _empty_grad(logits, x)
    _run(x.device, "grpo_token_logprobs_backward", *rows, stat, coef, _lib.ptr(scale),
         out.data_ptr(), sb, ss)
    return out


def _logprobs(logits, ids, mask, t, entropy: bool, train: bool):
    x, rows = _rows(logits, ids, mask, t)
    dev, (b, s, v) = x.device, x.shape
    logp = torch.empty(ids.shape, dtype=torch.float32, device=dev)
    ent = torch.empty_like(logp) if entropy else None
    stat = torch.empty((b * s, 4), dtype=torch.float32, device=dev) if train else None
    nbytes = _logp_bytes(rows[1], b, s, v)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _run(dev, "grpo_token_logprobs", *rows, logp.data_ptr(), _lib.ptr(ent), _lib.ptr(stat),
         _lib.ptr(ws), nbytes)
    return logp, ent, stat


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, t, entropy):
        logp, ent, stat = _logprobs(logits, ids, mask, t, entropy, True)
        ctx.save_for_backward(logits, ids, mask, stat)
        ctx.t = t
        ctx.set_materialize_grads(False)
        if ent is not None:
            ctx.mark_non_differentiable(ent)
        return logp, ent

    @staticmethod
    @_once
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None, None, None
        logits, ids, mask, stat = ctx.saved_tensors
        grad = _float_rows(grad, "grad", ids.shape, ids.device)
        return (_grad_of(logits, ids, mask, ctx.t, stat.data_ptr(), grad.data_ptr(), None), None,
                None, None, None)


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                   return_entropy: bool = False):
    """``log softmax(logits / temperature)`` at ``token_ids``, float32.

    ``logits [..., V]`` (bfloat16, float16 or float32; any row strides), ``token_ids``
    int64 of the leading shape, ``mask`` of that shape (None: every position counts).
    Differentiable by ``logits``.  With ``return_entropy`` also the entropy of each
    position's distribution, which carries no gradient.  An id outside the vocabulary at a
    counted position gives NaN there."""
    ids, mask, t = _check_logits(logits, token_ids, mask, temperature)
    if derivative_recorded(logits):
        logp, ent = _TokenLogprobs.apply(logits, ids, mask, t, return_entropy)
    else:
        logp, ent, _ = _logprobs(logits, ids, mask, t, return_entropy, False)
    return (logp, ent) if return_entropy else logp


# ------------------------------------------------------------ policy loss --

@functools.lru_cache(maxsize=64)
def _policy_of(eps_low: float, eps_high: float, cap: float, beta: float, normalizer):
    if not (0.0 <= eps_low < math.inf and 0.0 <= eps_high < math.inf):
        raise ValueError("eps_low and eps_high must be >= 0 and finite.")
    if not cap > 0.0:
        raise ValueError(f"delta must be positive, got {cap}.")
    if not 0.0 <= beta < math.inf:
        raise ValueError(f"beta must be >= 0 and finite, got {beta}.")
    if isinstance(normalizer, str):
        if normalizer not in _NORMALIZERS:
            raise ValueError(f"normalizer must be 'tokens', 'sequences' or a number, got "
                             f"{normalizer!r}.")
        return ctypes.byref(_lib.Policy(eps_low, eps_high, cap, beta, 1.0,
                                        _NORMALIZERS[normalizer]))
    if not 0.0 < normalizer < math.inf:
        raise ValueError(f"the normalizer must be positive and finite, got {normalizer}.")
    return ctypes.byref(_lib.Policy(eps_low, eps_high, cap, beta, normalizer, 2))


def _policy(eps_low, eps_high, delta, beta, normalizer, ref_logps):
    beta = float(beta)
    policy = _policy_of(float(eps_low), float(eps_high),
                        math.inf if delta is None else float(delta), beta,
                        normalizer if isinstance(normalizer, str) else float(normalizer))
    if beta and ref_logps is None:
        raise ValueError("beta > 0 needs ref_logps.")
    return policy


def _check_tokens(shape, device, old_logps, ref_logps, advantages):
    """(old, ref, advantages as float32, whether these are per token) that fit ``shape``."""
    if len(shape) != 2:
        raise ValueError(f"positions must be [batch, seq], got {list(shape)}.")
    if shape[0] >= 1 << 23 or shape.numel() >= 1 << 31:
        raise ValueError(f"fewer than 2^23 sequences and 2^31 tokens, got {list(shape)}.")
    per_token = advantages.ndim == 2
    return (_float_rows(old_logps, "old_logps", shape, device),
            _float_rows(ref_logps, "ref_logps", shape, device),
            _float_rows(advantages, "advantages", shape if per_token else shape[:1], device),
            per_token)


@functools.lru_cache(maxsize=256)
def _policy_bytes(b: int, s: int) -> int:
    return _lib.library().grpo_policy_loss_workspace_bytes(b, s)


def _policy_loss(lp, tokens, mask, policy, train: bool):
    old, ref, adv, per_token = tokens
    dev, (b, s) = lp.device, lp.shape
    loss = torch.empty((), dtype=torch.float32, device=dev)
    metrics = torch.empty(4, dtype=torch.float32, device=dev)
    # the float64 derivatives, where the backward wants them, then the workspace
    keep = -(-8 * b * s // 256) * 256 if train else 0
    nbytes = _policy_bytes(b, s)
    buf = torch.empty(keep + nbytes, dtype=torch.uint8, device=dev)
    at = buf.data_ptr()
    _run(dev, "grpo_policy_loss", lp.data_ptr(), _lib.ptr(old), _lib.ptr(ref), adv.data_ptr(),
         per_token, _lib.ptr(mask), b, s, policy, loss.data_ptr(), metrics.data_ptr(),
         at if train else None, at + keep, nbytes)
    return loss, metrics, buf


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, lp, tokens, mask, policy):
        loss, metrics, ctx.coef = _policy_loss(lp, tokens, mask, policy, True)
        ctx.shape, ctx.dtype = logps.shape, logps.dtype
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(metrics)
        return loss, metrics

    @staticmethod
    @_once
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None
        if grad_loss.dtype != torch.float32:
            grad_loss = grad_loss.float()
        dev = grad_loss.device
        out = torch.empty(ctx.shape, dtype=torch.float32, device=dev)
        _run(dev, "grpo_policy_loss_backward", ctx.coef.data_ptr(), grad_loss.data_ptr(),
             out.numel(), out.data_ptr())
        return out if ctx.dtype == torch.float32 else out.to(ctx.dtype), None, None, None, None


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
    ``ref_logps`` are ``[batch, seq]``, ``advantages`` ``[batch]`` or ``[batch, seq]``; all of
    them are read as float32 (other types are converted, float64 included) and computed with
    in float64; differentiable by ``logps`` alone.  ``metrics`` (float32 [4], no
    gradient) are means over the counted tokens: r, the share whose gain no longer moves
    with r (clipped or capped; with advantage 0 only past both ``delta`` and the clip),
    ``exp(q) - q - 1`` and ``old_logps - logps``.  ``ref_logps`` with
    ``beta`` 0 changes the third metric alone.  With nothing counted, loss and metrics are 0."""
    policy = _policy(eps_low, eps_high, delta, beta, normalizer, ref_logps)
    if not logps.is_cuda:
        raise ValueError("logps must be on the ROCm/HIP device.")
    shape, dev = logps.shape, logps.device
    tokens = _check_tokens(shape, dev, old_logps, ref_logps, advantages)
    mask = _mask_rows(mask, shape, dev)
    lp = _float_rows(logps, "logps", shape, dev)
    if derivative_recorded(logps):
        return _PolicyLoss.apply(logps, lp, tokens, mask, policy)
    return _policy_loss(lp, tokens, mask, policy, False)[:2]


# ------------------------------------------------- the loss from logits --

@functools.lru_cache(maxsize=256)
def _logits_plan(dtype: int, b: int, s: int, v: int):
    """(workspace bytes, whether the gradient is made with the loss)."""
    lib = _lib.library()
    return (lib.grpo_policy_loss_logits_workspace_bytes(dtype, b, s, v),
            bool(lib.grpo_policy_loss_logits_one_pass(dtype, b, s, v)))


def _logits_loss(logits, ids, mask, t, tokens, policy, train: bool):
    old, ref, adv, per_token = tokens
    x, rows = _rows(logits, ids, mask, t)
    dev, (b, s, v) = x.device, x.shape
    nbytes, one_pass = _logits_plan(rows[1], b, s, v)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    metrics = torch.empty(4, dtype=torch.float32, device=dev)
    logp = torch.empty(ids.shape, dtype=torch.float32, device=dev)
    grad, sb, ss = _empty_grad(logits, x) if train and one_pass else (None, 0, 0)
    # what the backward needs of each row (16 bytes of statistics, 4 of its derivative), then
    # the workspace
    keep = -(-20 * b * s // 256) * 256 if train else 0
    buf = torch.empty(keep + nbytes, dtype=torch.uint8, device=dev)
    at = buf.data_ptr()
    _run(dev, "grpo_policy_loss_logits", *rows, _lib.ptr(old), _lib.ptr(ref), adv.data_ptr(),
         per_token, policy, loss.data_ptr(), logp.data_ptr(), metrics.data_ptr(),
         at if train else None, at + 16 * b * s if train else None, _lib.ptr(grad), sb, ss,
         at + keep, nbytes)
    return loss, logp, metrics, buf, (grad, sb, ss)


class _LogitsLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, t, tokens, policy):
        loss, logp, metrics, ctx.buf, ctx.grad = _logits_loss(logits, ids, mask, t, tokens,
                                                              policy, True)
        ctx.save_for_backward(logits, ids, mask)
        ctx.t = t
        ctx.mark_non_differentiable(logp, metrics)
        ctx.set_materialize_grads(False)
        return loss, logp, metrics

    @staticmethod
    @_once
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return None, None, None, None, None, None
        logits, ids, mask = ctx.saved_tensors
        if grad_loss.dtype != torch.float32:
            grad_loss = grad_loss.float()
        stat = ctx.buf.data_ptr()
        coef = stat + 16 * ids.numel()
        # handed out once: it is the caller's from here on
        (grad, sb, ss), ctx.grad = ctx.grad, (None, 0, 0)
        if grad is None:
            grad = _grad_of(logits, ids, mask, ctx.t, stat, coef, grad_loss)
        else:
            x, rows = _rows(logits, ids, mask, ctx.t)
            _run(x.device, "grpo_policy_loss_logits_rescale", *rows, stat, coef,
                 grad_loss.data_ptr(), grad.data_ptr(), sb, ss)
        return grad, None, None, None, None, None


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
    ``metrics`` carry no gradient.  The logits' gradient is made with the loss, for an
    upstream gradient of 1, and the backward hands it out (or computes it again where the
    upstream gradient is another, and for a second backward); fewer than 128 rows of more than
    229376 bytes get theirs in the backward."""
    policy = _policy(eps_low, eps_high, delta, beta, normalizer, ref_logps)
    if logits.ndim != 3:
        raise ValueError(f"logits must be [batch, seq, vocab], got {list(logits.shape)}.")
    ids, mask, t = _check_logits(logits, token_ids, mask, temperature)
    tokens = _check_tokens(ids.shape, logits.device, old_logps, ref_logps, advantages)
    if derivative_recorded(logits):
        return _LogitsLoss.apply(logits, ids, mask, t, tokens, policy)
    return _logits_loss(logits, ids, mask, t, tokens, policy, False)[:3]


__all__ = ["token_logprobs", "grpo_policy_loss", "fused_grpo_loss"]

"""``counter_dropout`` -- dropout whose mask is never stored (``csrc/dropout.hip``).

The mask is a function of the element's index and of ``rng``, two int64 on the device
(seed and offset): the backward, and every kernel that needs it, makes it again.  ``rng`` is
read on the device, so a captured graph draws new masks when the tensor changes.
"""

from __future__ import annotations

import torch

from .. import _lib
from .ops import derivative_recorded

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check_p(p: float) -> float:
    p = float(p)
    if not (0.0 <= p and p * 65536.0 + 0.5 < 65536.0):
        raise ValueError(f"dropout p must be in [0, 1) (in steps of 1/65536), got {p}.")
    return p


def check_dropout(p: float, rng: torch.Tensor, device: torch.device) -> float:
    """``p`` as a float, after the checks that every dropout entry point makes."""
    p = _check_p(p)
    if rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous():
        raise ValueError("rng must be a contiguous int64 tensor of two values, seed and offset.")
    if rng.device != device:
        raise ValueError(f"rng must be on {device}, got {rng.device}.")
    return p


def _dropout(x: torch.Tensor, p: float, rng: torch.Tensor) -> torch.Tensor:
    if not x.is_contiguous():
        x = x.contiguous()
    y, dev = torch.empty_like(x), x.device
    args = (x.data_ptr(), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p, rng.data_ptr())
    fn = _lib.device_library().grpo_dropout
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, _lib.stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream_handle(dev))
    if rc:
        _lib.check(rc, "grpo_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng):
        ctx.p = p
        ctx.save_for_backward(rng)
        ctx.save_for_forward(rng)
        return _dropout(x, p, rng)

    @staticmethod
    def backward(ctx, grad):
        # the mask again; its own gradient is the same call, so it differentiates twice
        rng, = ctx.saved_tensors
        run = _Dropout.apply if torch.is_grad_enabled() and grad.requires_grad else _dropout
        return run(grad, ctx.p, rng), None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        # linear in x: the tangent under the same mask
        return counter_dropout(tangent, ctx.p, ctx.saved_tensors[0])


def counter_dropout(x: torch.Tensor, p: float, rng: torch.Tensor) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p``, the others scaled.

    Element ``e`` of ``x`` (row-major) is dropped iff ``u(e) < t``, ``t = round(65536 p)``,
    where ``u(e)`` are 16 bits of the Philox4x32-10 block with counter ``(e // 8, offset)``
    and key ``seed``, ``rng = [seed, offset]``; the rest is multiplied by
    ``65536 / (65536 - t)`` and rounded once.  A dropped element gives 0, also where x is
    not finite.  The same ``rng`` gives the same mask; the caller changes the offset from
    call to call (``CounterDropout`` does), and leaves ``rng`` unchanged until the backward
    has run.  Differentiable by ``x``, in forward mode too.  bfloat16, float16 or float32,
    any shape."""
    if not x.is_cuda:
        raise ValueError("x must be on the ROCm/HIP device.")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}.")
    p = check_dropout(p, rng, x.device)
    if derivative_recorded(x):
        return _Dropout.apply(x, p, rng)
    return _dropout(x, p, rng)


class CounterDropout(torch.nn.Module):
    """``nn.Dropout`` on ``counter_dropout``: seed and offset of each call are drawn on the
    device from torch's generator, so ``torch.manual_seed``, activation checkpointing and
    graph capture govern the mask as they do any of torch's random numbers."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        self.p = _check_p(p)

    @staticmethod
    def draw(device: torch.device) -> torch.Tensor:
        """Seed and offset of one mask."""
        return torch.randint(0, 2 ** 63 - 1, (2,), dtype=torch.int64, device=device)

    def active(self) -> bool:
        return self.training and self.p > 0.0

    def forward(self, x: torch.Tensor, rng: torch.Tensor | None = None) -> torch.Tensor:
        if not self.active():
            return x
        return counter_dropout(x, self.p, self.draw(x.device) if rng is None else rng)

    def extra_repr(self) -> str:
        return f"p={self.p}"


__all__ = ["CounterDropout", "counter_dropout", "check_dropout"]

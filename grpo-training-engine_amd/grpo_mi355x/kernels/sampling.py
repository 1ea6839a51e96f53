"""``sample_tokens`` -- a token from each row of logits, from given uniform numbers
(``csrc/sample_tokens.hip``), with temperature, top-k, top-p and min-p, for any vocabulary, type
and row.

Its top-p is not that of ``src/triton_kernels/paged_kv.py:418-450``, which the framework's sampled
decode keeps (``paged_kv_decode_model``, ``grpo_sample_top_p``): the token at which the mass passes
``top_p`` is kept here (the shortest head that holds ``top_p`` of the mass) and cut there. Of .5,
.3, .15 and .05 at .9 three are kept here, two there.
"""

from __future__ import annotations

import ctypes
import math
from typing import Union

import torch

from .. import _lib
from .policy_loss import _run

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MAX_VOCAB = 1 << 20
_MAX_ROWS = 1 << 31
Setting = Union[float, torch.Tensor]


def _row_setting(t: torch.Tensor, name: str, lead, device, dtype) -> torch.Tensor:
    """One setting per row, contiguous, of the kernel's type."""
    if t.shape != lead:
        raise ValueError(f"{name} must be a number or {list(lead)}, got {list(t.shape)}.")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}.")
    if t.dtype.is_complex or (dtype == torch.int32 and t.dtype.is_floating_point):
        raise ValueError(f"{name} cannot be {t.dtype}.")
    if dtype == torch.int32 and t.dtype in (torch.int64, torch.uint32, torch.uint64):
        t = t.long().clamp(0, _MAX_VOCAB)
    return t.to(dtype).contiguous()


def sample_tokens(logits: torch.Tensor, draws: torch.Tensor, *, temperature: Setting = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0, return_kept: bool = False):
    """One token id (int64) per row of ``logits [..., V]`` (bfloat16, float16 or float32; any
    row stride), from ``draws [...]``, uniform numbers in [0, 1) (float32 or float64).

    With ``w = exp((x - max) / temperature)`` and the tokens in descending order of their logits
    (ties by index), a token is kept while fewer than ``top_k`` stand before it, the mass before
    it is below ``top_p`` times the mass of those ``top_k``, and ``w >= min_p``; the first
    always is. The token is the first kept one at which the running mass passes ``draws`` times
    the kept mass. (The sampled decode's ``top_p`` also cuts the token that passes it.)

    Masses are integers (units of 2^-44 of the largest weight; 2^-(62 - log2 V) for more than 2^18
    tokens), so the same inputs give the same token, whatever runs beside. A weight in them is
    rounded to a unit for most bf16 rows, else off by 3e-11 of itself at most (2e-9 for 2^20
    tokens): a draw or a border closer than that to a sum may go to its other side.

    Each setting is a number or a tensor of the leading shape (float32; ``top_k`` integers).
    ``temperature`` 0 (or below):
    the lowest index of the maximum; ``top_k`` 0 (or below), ``top_p`` 1, ``min_p`` 0: no such
    filter. NaN and -inf logits are never drawn; beside +inf only +inf is. A row with nothing to
    draw gives -1. With ``return_kept`` also the number of kept tokens (int32)."""
    if logits.ndim < 1 or not logits.shape[-1]:
        raise ValueError(f"logits must be [..., vocab], got {list(logits.shape)}.")
    if not logits.is_cuda:
        raise ValueError("logits must be on the ROCm/HIP device.")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}.")
    lead, v, dev = logits.shape[:-1], logits.shape[-1], logits.device
    if v > _MAX_VOCAB:
        raise ValueError(f"a vocabulary of at most {_MAX_VOCAB} tokens, got {v}.")
    if draws.shape != lead or draws.device != dev:
        raise ValueError(f"draws must be {list(lead)} on {dev}, got {list(draws.shape)} on "
                         f"{draws.device}.")
    if draws.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"draws must be float32 or float64, got {draws.dtype}.")
    x = logits.detach()
    if x.ndim != 2:
        x = x.reshape(-1, v)
    m = x.shape[0]
    if (v > 1 and x.stride(1) != 1) or (m > 1 and 0 < x.stride(0) < v):  # (rows that overlap)
        x = x.contiguous()
    if m >= _MAX_ROWS:
        raise ValueError(f"at most {_MAX_ROWS - 1} rows of logits in a call.")
    draws = draws.contiguous()
    s, held = _lib.Sampler(), []
    for name, value, dtype in (("temperature", temperature, torch.float32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                               ("top_k", top_k, torch.int32)):
        if isinstance(value, torch.Tensor):
            held.append(_row_setting(value, name, lead, dev, dtype))
            setattr(s, name + "_rows", held[-1].data_ptr())
            continue
        number = value if name == "top_k" and isinstance(value, int) else float(value)
        if number != number or number in (math.inf, -math.inf):
            raise ValueError(f"{name} must be a finite number, got {value}.")
        if name == "top_k":
            number = min(max(int(number), 0), _MAX_VOCAB)
        setattr(s, name, number)
    tokens = torch.empty(lead, dtype=torch.int64, device=dev)
    kept = torch.empty(lead, dtype=torch.int32, device=dev) if return_kept else None
    _run(dev, "grpo_sample_tokens", x.data_ptr(), _DTYPES[x.dtype], x.stride(0), m, v,
         draws.data_ptr(), draws.dtype == torch.float64, ctypes.byref(s), tokens.data_ptr(),
         _lib.ptr(kept))
    return (tokens, kept) if return_kept else tokens


__all__ = ["sample_tokens"]

"""Checking a tree of drafted tokens in one pass (``csrc/draft_tree.hip``,
``csrc/tree_attention.hip``): the decode step's cache and attention operators
(``src/triton_kernels/paged_kv.py:63-319``) for several tokens per sequence.

Sequence ``b`` has ``context_lens[b]`` tokens in the paged cache. Its tree's nodes
``0 .. counts[b] - 1`` stand after them: node ``i``'s keys and values at slot
``context_lens[b] + i``, its parent ``parents[b, i]`` an earlier node (-1, or anything else
that is not an earlier node: none). Node 0 is the pending token, the newest one, whose keys and
values are not cached yet; the drafted tokens hang off it. One pass over the model calls, in
every layer,

* ``paged_rope_append``: queries and keys rotated, keys and values stored;
* ``paged_tree_attention``: every node over the cached tokens, its ancestors and itself;

then ``sample_tokens`` draws each node's next token, and

* ``accept_draft_tree`` follows the drafted tokens that were drawn and closes up the cache.

``context_lens`` is then ``context_lens + accepted``. Queries, keys, values and caches are
bfloat16 or float16, all of one type. Arguments that do not fit raise ``ValueError``, a missing
device ``ImportError``. No gradients. Nothing is kept between calls.
"""

from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from .. import _lib
from .policy_loss import _run

MAX_NODES = 64  # of a tree: one per lane of a wave
_HALF = (torch.bfloat16, torch.float16)
_I32 = torch.int32


def _check_cache(k_cache, v_cache, layered: bool):
    """(layers, num_blocks, Hkv, block_size, D), type and device of checked caches."""
    shape, dtype, device = k_cache.shape, k_cache.dtype, k_cache.device
    if len(shape) != 4 and not (layered and len(shape) == 5):
        raise ValueError("k_cache/v_cache must be [num_blocks, heads, block, head_dim]"
                         + (" or [layers, ...]." if layered else "."))
    if v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must have identical shapes.")
    if dtype not in _HALF or v_cache.dtype is not dtype:
        raise ValueError("k_cache/v_cache must be bfloat16 or float16, both the same.")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous.")
    if not k_cache.is_cuda or v_cache.get_device() != device.index:
        raise ValueError("k_cache/v_cache must be on the ROCm/HIP device, both on one.")
    if not k_cache.numel():
        raise ValueError("k_cache/v_cache must not be empty.")
    return shape if len(shape) == 5 else (1, *shape), dtype, device


def _check_ints(t: torch.Tensor, name: str, shape, device, dtype=_I32) -> None:
    if t.dtype is not dtype or t.get_device() != device.index or t.shape != shape:
        raise ValueError(f"{name} must be {str(dtype)[6:]} {list(shape)} on {device}, got "
                         f"{str(t.dtype)[6:]} {list(t.shape)} on {t.device}.")


def _check_tables(block_tables, context_lens, counts, b: int, device):
    """(context_lens, address of counts or None, the tables, their row stride and width), and
    counts, which has to live as long."""
    if block_tables.ndim != 2 or not block_tables.shape[1]:
        raise ValueError("block_tables must be [batch, max_blocks].")
    rows, width = block_tables.shape
    at, index = None, device.index
    # (one look at what is right; what is not is found below)
    if not (rows == b and block_tables.dtype is _I32 and block_tables.get_device() == index
            and context_lens.dtype is _I32 and context_lens.get_device() == index
            and context_lens.ndim == 1 and context_lens.shape[0] == b):
        _check_ints(block_tables, "block_tables", (b, width), device)
        _check_ints(context_lens, "context_lens", (b,), device)
    if counts is not None:
        _check_ints(counts, "counts", (b,), device)
        counts = counts.contiguous()
        at = counts.data_ptr()
    stride, step = block_tables.stride()
    if step != 1 and width > 1:
        block_tables = block_tables.contiguous()
        stride = width
    return context_lens.contiguous(), at, block_tables, stride, width, counts


def _rows(t: Optional[torch.Tensor], name: str, shape, device, dtype=_I32):
    """``t`` [B, T] with contiguous rows (an expanded row stays one), its address and row
    stride."""
    if t is None:
        return None, None, 0
    _check_ints(t, name, shape, device, dtype)
    if t.stride(1) != 1 and shape[1] > 1:
        t = t.contiguous()
    return t, t.data_ptr(), t.stride(0)


def _heads(t: torch.Tensor, name: str, shape, dtype, device):
    """``t`` [B, T, H, D] of the cache's type, its last dim contiguous, and three strides."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}.")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype} like the caches, got {t.dtype}.")
    if t.get_device() != device.index:
        raise ValueError(f"{name} must be on {device}, got {t.device}.")
    sb, st, sh, sd = t.stride()
    if sd != 1 and shape[3] > 1:
        t = t.contiguous()
        sb, st, sh, _ = t.stride()
    return t, sb, st, sh


def _grouped(hq: int, hkv: int) -> None:
    if hq < 1 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be a multiple of KV heads ({hkv}).")


def paged_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                      sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                      counts: Optional[torch.Tensor] = None,
                      positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate ``q [B, T, Hq, D]`` and ``k [B, T, Hkv, D]`` to their positions and store the
    rotated ``k`` and ``v`` at slots ``context_lens[b] + i``; returns the rotated ``q``.

    Any number of tokens ``T`` (a tree's nodes, or a chunk of a prompt; fewer than 2^24 in all),
    any strides.
    ``cos``/``sin`` ``[max_pos, D]`` in float32 or q's type (``rotary_emb.tables``); position of
    token ``i``: ``positions[b, i]`` (int32; clamped to the table), else ``context_lens[b] + i``.
    The rotation is float32, rounded once (the decode step's rounds three times in bf16, so its
    cached keys differ in last bits). Rows past ``counts[b]`` are not stored and their
    ``q`` is 0; slots past the block table, or in blocks outside the cache, are skipped."""
    (_, nb, hkv, bs, d), dtype, dev = _check_cache(k_cache, v_cache, False)
    if q.ndim != 4:
        raise ValueError(f"q must be [B, T, heads, {d}], got {list(q.shape)}.")
    b, t, hq, _ = q.shape
    q, qb, qt, qh = _heads(q, "q", (b, t, hq, d), dtype, dev)
    k, kb, kt, kh = _heads(k, "k", (b, t, hkv, d), dtype, dev)
    v, vb, vt, vh = _heads(v, "v", (b, t, hkv, d), dtype, dev)
    _grouped(hq, hkv)
    if d % 2:
        raise ValueError(f"head_dim must be even, got {d}.")
    if cos.ndim != 2 or cos.shape[1] != d or not cos.shape[0] or sin.shape != cos.shape:
        raise ValueError(f"cos/sin must be [max_pos, {d}], both the same.")
    wide = cos.dtype is torch.float32
    if not (wide or cos.dtype is dtype) or sin.dtype is not cos.dtype:
        raise ValueError("cos/sin must be float32 or of q's type, both the same.")
    if cos.get_device() != dev.index or sin.get_device() != dev.index:
        raise ValueError(f"cos/sin must be on {dev}.")
    cos, sin = cos.contiguous(), sin.contiguous()
    lens, n_at, tables, bt_stride, width, counts = _check_tables(block_tables, context_lens,
                                                                 counts, b, dev)
    positions, p_at, p_stride = _rows(positions, "positions", (b, t), dev)
    out = q.new_empty((b, t, hq, d))
    _run(dev, "grpo_paged_rope_append", q.data_ptr(), qb, qt, qh, k.data_ptr(), kb, kt, kh,
         v.data_ptr(), vb, vt, vh, dtype is torch.float16, cos.data_ptr(), sin.data_ptr(), wide,
         cos.shape[0], p_at, p_stride, lens.data_ptr(), n_at, out.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), nb, tables.data_ptr(), bt_stride, bs, width, b, t, hq, hkv, d)
    return out


@functools.lru_cache(maxsize=256)
def _attn_bytes(b: int, t: int, hq: int, hkv: int, d: int) -> int:
    return _lib.library().grpo_paged_tree_attn_workspace_bytes(b, t, hq, hkv, d)


def _check_nodes(t: int) -> None:
    if not 1 <= t <= MAX_NODES:
        raise ValueError(f"a drafted tree has 1 to {MAX_NODES} nodes, got {t}.")


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         block_tables: torch.Tensor, context_lens: torch.Tensor,
                         parents: Optional[torch.Tensor] = None, *,
                         counts: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the nodes' (rotated) ``q [B, T, Hq, D]``, ``T <= 64`` (fewer than 2^24 nodes in
    all), each over its sequence's ``context_lens[b]`` cached tokens, its ancestors and itself;
    ``[B, T, Hq, D]`` in q's type.

    ``parents`` int32 ``[B, T]`` (one tree for all: ``parents.expand(B, -1)``), None: a chain,
    node ``i - 1`` being the parent of ``i``. ``scale``: 1 / sqrt(D) unless given. Nodes past
    ``counts[b]``, and nodes that attend nothing, get 0. Tokens that a node does not attend do
    not reach it, whatever stands in their slots."""
    (_, nb, hkv, bs, d), dtype, dev = _check_cache(k_cache, v_cache, False)
    if q.ndim != 4:
        raise ValueError(f"q must be [B, T, heads, {d}], got {list(q.shape)}.")
    b, t, hq, _ = q.shape
    q, qb, qt, qh = _heads(q, "q", (b, t, hq, d), dtype, dev)
    _grouped(hq, hkv)
    _check_nodes(t)
    if d > 512:
        raise ValueError(f"head_dim at most 512, got {d}.")
    lens, n_at, tables, bt_stride, width, counts = _check_tables(block_tables, context_lens,
                                                                 counts, b, dev)
    parents, p_at, p_stride = _rows(parents, "parents", (b, t), dev)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    out = q.new_empty((b, t, hq, d))
    nbytes = _attn_bytes(b, t, hq, hkv, d)
    ws = q.new_empty(nbytes // 2) if nbytes else None
    _run(dev, "grpo_paged_tree_attn", q.data_ptr(), qb, qt, qh, dtype is torch.float16,
         k_cache.data_ptr(), v_cache.data_ptr(), nb, tables.data_ptr(), bt_stride, bs, width,
         lens.data_ptr(), p_at, p_stride, n_at, scale, out.data_ptr(), b, t, hq, hkv, d,
         _lib.ptr(ws), nbytes)
    return out


def accept_draft_tree(draft_tokens: torch.Tensor, parents: torch.Tensor, sampled: torch.Tensor,
                      context_lens: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      block_tables: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
                      eos_token_id: Optional[int] = None, pad_token_id: int = 0):
    """The drafted tokens that the model drew itself, and the cache without the others.

    ``draft_tokens``, ``sampled`` int64 ``[B, T]``: each node's token, and the token drawn from
    the logits at that node. Node 0 is accepted; after node ``i`` comes its first child whose
    drafted token is ``sampled[b, i]``. The path ends where no child has it, after
    ``eos_token_id`` and at a negative token. The accepted nodes' keys and values move to the
    slots ``context_lens[b] + 0, 1, ...``, in every layer where the caches are ``[layers,
    num_blocks, Hkv, block, D]`` (``PagedKVPool.k``, ``.v``); no two sequences' tables may share
    a block that holds these slots.

    Returns ``(tokens, accepted, path)``: the new tokens ``[B, T]`` int64 (``sampled`` along the
    path, the last of them pending; ``pad_token_id`` behind them), how many they are ``[B]``
    int32, and the accepted nodes ``[B, T]`` int32 (-1 behind them). The tokens
    have the distribution of drawing one at a time in the way ``sampled`` was drawn, whatever was
    drafted."""
    (layers, nb, hkv, bs, d), _, dev = _check_cache(k_cache, v_cache, True)
    shape = draft_tokens.shape
    if len(shape) != 2:
        raise ValueError(f"draft_tokens must be [B, T], got {list(shape)}.")
    b, t = shape
    _check_nodes(t)
    drafted, d_at, d_stride = _rows(draft_tokens, "draft_tokens", shape, dev, torch.int64)
    sampled, s_at, s_stride = _rows(sampled, "sampled", shape, dev, torch.int64)
    parents, p_at, p_stride = _rows(parents, "parents", shape, dev)
    if b > 65535:
        raise ValueError(f"at most 65535 sequences, got {b}.")
    lens, n_at, tables, bt_stride, width, counts = _check_tables(block_tables, context_lens,
                                                                 counts, b, dev)
    tokens = drafted.new_empty(shape)
    path = lens.new_empty(shape)
    accepted = lens.new_empty(b)
    _run(dev, "grpo_draft_tree_accept", d_at, d_stride, p_at, p_stride, s_at, s_stride,
         lens.data_ptr(), n_at, k_cache.data_ptr(), v_cache.data_ptr(), layers, nb,
         tables.data_ptr(), bt_stride, bs, width, b, t, hkv, d,
         -1 if eos_token_id is None else int(eos_token_id), int(pad_token_id), tokens.data_ptr(),
         accepted.data_ptr(), path.data_ptr())
    return tokens, accepted, path


__all__ = ["paged_rope_append", "paged_tree_attention", "accept_draft_tree", "MAX_NODES"]

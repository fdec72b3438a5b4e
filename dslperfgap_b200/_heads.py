"""Argument checks of the per-head operators (``rope``, ``qk_norm_rope``) and
their layout as the C ABI's ``dslpg_heads``."""
from __future__ import annotations

import torch

from . import _lib

MAX_HEAD_DIM = 1024
MAX_ROWS = 1 << 30


def dense_last(x: torch.Tensor) -> torch.Tensor:
    """x itself, or a contiguous copy when its last axis is not dense."""
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def check_like(x, like, name: str, what: str) -> None:
    if x.shape != like.shape or x.dtype != like.dtype:
        raise ValueError(f"{what}: {name} must have shape {tuple(like.shape)} and dtype {like.dtype}, "
                         f"got {tuple(x.shape)} and {x.dtype}")


def _strides(x: torch.Tensor) -> tuple:
    """Batch, sequence and head strides of [tokens, heads, D] or [batch, seq, heads, D]."""
    s = x.stride()
    return (0, s[0], s[1]) if x.dim() == 3 else (s[0], s[1], s[2])


def check_layout(q, k, positions, inv_freq, sections, what: str) -> None:
    """Raise for shapes and types that the operators do not take."""
    _lib.float_code(q, what)
    if q.dim() not in (3, 4):
        raise ValueError(f"{what}: q must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim], "
                         f"got shape {tuple(q.shape)}")
    if k.dtype != q.dtype:
        raise TypeError(f"{what}: q and k must have one dtype, got {q.dtype} and {k.dtype}")
    if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: k shape {tuple(k.shape)} does not match q {tuple(q.shape)} (heads may differ)")
    d = q.shape[-1]
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"{what}: head_dim must be in 1..{MAX_HEAD_DIM}, got {d}")
    if q.shape[:-2].numel() * (q.shape[-2] + k.shape[-2]) > MAX_ROWS:
        raise ValueError(f"{what}: more than {MAX_ROWS} rows (tokens times heads)")
    if positions.dtype not in _lib.LABEL_CODES:
        raise TypeError(f"{what}: positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.dtype != torch.float32:
        raise TypeError(f"{what}: inv_freq must be float32, got {inv_freq.dtype}")
    if inv_freq.dim() != 1 or not 2 <= 2 * inv_freq.shape[0] <= d:
        raise ValueError(f"{what}: inv_freq must be 1-D with 1 to head_dim / 2 = {d // 2} frequencies, "
                         f"got shape {tuple(inv_freq.shape)}")
    if sections is not None:
        n = inv_freq.shape[0]
        if not 1 <= len(sections) <= 4 or any(s < 0 for s in sections) or sum(sections) != n:
            raise ValueError(f"{what}: sections must be 1 to 4 counts that add up to the {n} frequencies, "
                             f"got {tuple(sections)}")


def layout(q, k, positions, inv_freq, sections, interleaved, what: str, dq=None, dk=None, weight=None):
    """(positions, inv_freq, dslpg_heads) of a checked call; q, k (dq, dk) are dense in their last axis."""
    tokens = tuple(q.shape[:-2])
    want = tokens if sections is None else (len(sections),) + tokens
    try:
        pos = positions.expand(want)
    except RuntimeError:
        raise ValueError(f"{what}: positions of shape {tuple(positions.shape)} do not broadcast to {want}") from None
    ps = pos.stride()
    if sections is None:
        ps = (0,) + ps
    if q.dim() == 3:
        ps = (ps[0], 0, ps[1])
    inv_freq = inv_freq.contiguous()
    h = _lib.Heads()
    h.batch, h.seq = (1, tokens[0]) if q.dim() == 3 else tokens
    h.q_heads, h.k_heads, h.head_dim, h.rotary_dim = q.shape[-2], k.shape[-2], q.shape[-1], 2 * inv_freq.shape[0]
    h.q_strides[:], h.k_strides[:], h.position_strides[:] = _strides(q), _strides(k), ps
    if dq is not None:
        h.dq_strides[:], h.dk_strides[:] = _strides(dq), _strides(dk)
    each = (inv_freq.shape[0],) if sections is None else tuple(int(s) for s in sections)
    h.axes, h.interleaved = len(each), 1 if interleaved else 0
    h.sections[:] = each + (0,) * (4 - len(each))
    h.dtype, h.positions_dtype = _lib.FLOAT_CODES[q.dtype], _lib.LABEL_CODES[positions.dtype]
    if weight is not None:
        h.weight_dtype = _lib.FLOAT_CODES[weight.dtype]
    return pos, inv_freq, h


def empty_rows(x: torch.Tensor) -> torch.Tensor:
    """A dense output of x's shape and type."""
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)

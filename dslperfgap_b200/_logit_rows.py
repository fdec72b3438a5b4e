"""Argument checks that the losses on rows of logits share (``policy_loss``,
``preference_loss``), and the rows as the C ABI's ``dslpg_logit_rows``."""
from __future__ import annotations

import torch

from . import _lib

MAX_COLS = 1 << 30
MIN_SCALE, MAX_SCALE = 1e-30, 1e30  # the exponents' constant is held in float32


def check_rows(logits, labels, logit_scale, what: str) -> None:
    _lib.float_code(logits, f"{what} logits")
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= MAX_COLS:
        raise ValueError(f"{what}: logits must be 2-D with 1 to {MAX_COLS} columns, got shape {tuple(logits.shape)}")
    if labels.dtype not in _lib.LABEL_CODES:
        raise TypeError(f"{what}: labels must be int32 or int64, got {labels.dtype}")
    if labels.dim() != 1 or labels.shape[0] != logits.shape[0]:
        raise ValueError(f"{what}: labels shape {tuple(labels.shape)} != ({logits.shape[0]},)")
    if logit_scale != 0 and not MIN_SCALE <= abs(logit_scale) <= MAX_SCALE:
        raise ValueError(f"{what}: logit_scale must be 0 or {MIN_SCALE} to {MAX_SCALE} in size, got {logit_scale}")


def check_vector(x, n: int, name: str, what: str) -> None:
    """x is a float32 vector of n values (any stride: an expanded scalar is one value for all)."""
    if x.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be float32, got {x.dtype}")
    if x.dim() != 1 or x.shape[0] != n:
        raise ValueError(f"{what}: {name} must have shape ({n},), got {tuple(x.shape)}")


def rows(logits, labels, logit_scale, ignored_index):
    """(dslpg_logit_rows, the tensors it points into)."""
    if logits.shape[1] > 1 and logits.stride(1) != 1 or logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]:
        logits = logits.contiguous()
    labels = labels.contiguous()
    r = _lib.LogitRows()
    r.logits, r.labels = logits.data_ptr(), labels.data_ptr()
    r.n_rows, r.n_cols = logits.shape
    r.row_stride = logits.stride(0) if logits.shape[0] > 1 else logits.shape[1]
    r.ignored_index, r.logit_scale = int(ignored_index), float(logit_scale)
    r.logits_dtype, r.labels_dtype = _lib.FLOAT_CODES[logits.dtype], _lib.LABEL_CODES[labels.dtype]
    return r, (logits, labels)


def empty_f32(n: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(n, dtype=torch.float32, device=like.device)


def empty_grad(logits: torch.Tensor) -> torch.Tensor:
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)

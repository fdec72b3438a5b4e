"""CUDA (sm_100a) preference loss on pairs of sequences, from rows of logits.

The rows of 2 n_pairs sequences lie one behind another: sequence s is rows
``seq_starts[s]`` to ``seq_starts[s + 1]`` (2 n_pairs + 1 ascending bounds, int32
or int64, on the GPU), the chosen ones first; pair k is sequences k and
n_pairs + k. With logp as in ``policy_loss``::

    log_ratio[s] = sum of logp - ref_logp over the rows of s
    m = beta (log_ratio[k] - log_ratio[n_pairs + k])
    loss[k] = (1 - smoothing) softplus(-m) + smoothing softplus(m)

``preference_loss_fwd`` returns ``(loss, log_ratio, logp, lse)``: float32
``[n_pairs]``, ``[2 n_pairs]`` and ``[n_rows]`` twice; ``preference_loss_bwd``
returns dlogits from the forward's ``lse`` and ``log_ratio`` and the pairs'
``dloss``. (The gradient of a row depends on whole sequences, so there is no form
that does both in one reading.) The suite has no kernel of this kind; the
calling convention is cross_entropy's.

A row is left out when its label is ``ignored_index`` or no column, or when it
lies before the first bound or behind the last: nothing of it is read, and its
logp, lse and gradient are 0. Bounds that do not ascend give wrong sums, but
nothing outside the rows is read or written.
"""
import ctypes
import math

from .. import _lib, _logit_rows as _rows

_fast_preference_loss_fwd = _lib.fast_op("preference_loss_fwd")
_fast_preference_loss_bwd = _lib.fast_op("preference_loss_bwd")


def _check(logits, labels, seq_starts, beta, smoothing, logit_scale, what):
    """The number of pairs."""
    _rows.check_rows(logits, labels, logit_scale, what)
    if seq_starts.dtype not in _lib.LABEL_CODES:
        raise TypeError(f"{what}: seq_starts must be int32 or int64, got {seq_starts.dtype}")
    if seq_starts.dim() != 1 or seq_starts.shape[0] < 3 or seq_starts.shape[0] % 2 == 0:
        raise ValueError(f"{what}: seq_starts must have 2 n_pairs + 1 bounds (n_pairs >= 1), "
                         f"got shape {tuple(seq_starts.shape)}")
    if not math.isfinite(beta):
        raise ValueError(f"{what}: beta must be finite, got {beta}")
    if not 0 <= smoothing <= 1:
        raise ValueError(f"{what}: smoothing must be in [0, 1], got {smoothing}")
    return seq_starts.shape[0] // 2


def _terms(seq_starts, ref_logp, n_pairs, beta, smoothing):
    t = _lib.PairTerms()
    t.seq_starts, t.starts_dtype, t.n_pairs = seq_starts.data_ptr(), _lib.LABEL_CODES[seq_starts.dtype], n_pairs
    if ref_logp is not None:
        t.ref_logp, t.ref_stride = ref_logp.data_ptr(), ref_logp.stride(0)
    t.beta, t.smoothing = beta, smoothing
    return t


def preference_loss_fwd(logits, labels, seq_starts, ref_logp, beta=0.1, smoothing=0.0, logit_scale=1.0,
                        ignored_index=-100):
    out = _fast_preference_loss_fwd(logits, labels, seq_starts, ref_logp, beta, smoothing, logit_scale, ignored_index)
    if out is not None:  # the C++ fast path took the common case
        return out
    what = "preference_loss_fwd"
    dev = _lib.require_cuda(logits, labels, seq_starts, ref_logp, what=what)
    pairs = _check(logits, labels, seq_starts, beta, smoothing, logit_scale, what)
    n = logits.shape[0]
    _rows.check_vector(ref_logp, n, "ref_logp", what)
    loss, log_ratio = _rows.empty_f32(pairs, logits), _rows.empty_f32(2 * pairs, logits)
    logp, lse = _rows.empty_f32(n, logits), _rows.empty_f32(n, logits)
    rows, keep = _rows.rows(logits, labels, logit_scale, ignored_index)
    starts = seq_starts.contiguous()
    terms = _terms(starts, ref_logp, pairs, beta, smoothing)
    _lib.launch(dev, "dslpg_preference_loss_fwd", ctypes.addressof(rows), ctypes.addressof(terms), loss.data_ptr(),
                log_ratio.data_ptr(), logp.data_ptr(), lse.data_ptr())
    return loss, log_ratio, logp, lse


def preference_loss_bwd(dloss, logits, lse, labels, seq_starts, log_ratio, beta=0.1, smoothing=0.0, logit_scale=1.0,
                        ignored_index=-100):
    out = _fast_preference_loss_bwd(dloss, logits, lse, labels, seq_starts, log_ratio, beta, smoothing, logit_scale,
                                    ignored_index)
    if out is not None:
        return out
    what = "preference_loss_bwd"
    dev = _lib.require_cuda(dloss, logits, lse, labels, seq_starts, log_ratio, what=what)
    pairs = _check(logits, labels, seq_starts, beta, smoothing, logit_scale, what)
    n = logits.shape[0]
    _rows.check_vector(dloss, pairs, "dloss", what)
    _rows.check_vector(lse, n, "lse", what)
    _rows.check_vector(log_ratio, 2 * pairs, "log_ratio", what)
    dlogits = _rows.empty_grad(logits)
    if n == 0:
        return dlogits
    lse, log_ratio, starts = lse.contiguous(), log_ratio.contiguous(), seq_starts.contiguous()
    rows, keep = _rows.rows(logits, labels, logit_scale, ignored_index)
    terms = _terms(starts, None, pairs, beta, smoothing)
    _lib.launch(dev, "dslpg_preference_loss_bwd", ctypes.addressof(rows), ctypes.addressof(terms), dloss.data_ptr(),
                dloss.stride(0), lse.data_ptr(), log_ratio.data_ptr(), dlogits.data_ptr(), logits.shape[1])
    return dlogits

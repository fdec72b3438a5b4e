"""CUDA (sm_100a) clipped policy loss with a KL term, on rows of logits.

Per row, with z = logit_scale * logits and logp = z[label] - logsumexp(z)::

    r = exp(logp - old_logp);  d = ref_logp - logp;  kl = exp(d) - d - 1
    loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef kl

``policy_loss_fwd`` returns ``(loss, logp, lse, kl)``, float32 ``[n_rows]``
each; ``policy_loss_bwd`` returns dlogits (the logits' shape and type) from the
forward's ``lse`` and the losses' gradients ``dloss``; ``policy_loss_fwd_bwd``
does both in one call, with one reading of the logits where their length allows
it, for a ``dloss`` known beforehand (the weights of a mean over tokens, for
instance), and returns ``(loss, logp, lse, kl, dlogits)``. The suite has no kernel of this kind; the calling convention is
cross_entropy's.

``old_logp``, ``advantages``, ``ref_logp`` and ``dloss`` are float32 ``[n_rows]``
of any stride. Without ``ref_logp`` the KL term is 0; with ``kl_coef`` 0 it is
only reported. A row whose label is ``ignored_index``, or no column, is left out:
nothing of it is read, and its loss, logp, lse, kl and gradient are 0.
"""
import ctypes
import math

from .. import _lib, _logit_rows as _rows

_fast_policy_loss_fwd = _lib.fast_op("policy_loss_fwd")
_fast_policy_loss_bwd = _lib.fast_op("policy_loss_bwd")
_fast_policy_loss_fwd_bwd = _lib.fast_op("policy_loss_fwd_bwd")


def _check(logits, labels, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, logit_scale, what):
    _rows.check_rows(logits, labels, logit_scale, what)
    n = logits.shape[0]
    _rows.check_vector(old_logp, n, "old_logp", what)
    _rows.check_vector(advantages, n, "advantages", what)
    if ref_logp is not None:
        _rows.check_vector(ref_logp, n, "ref_logp", what)
    if not 0 <= clip_low <= 1 or not clip_high >= 0:
        raise ValueError(f"{what}: needs 0 <= clip_low <= 1 and clip_high >= 0, got {clip_low} and {clip_high}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"{what}: kl_coef must be finite, got {kl_coef}")


def _terms(old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef):
    t = _lib.PolicyTerms()
    t.old_logp, t.advantages = old_logp.data_ptr(), advantages.data_ptr()
    t.old_stride, t.advantages_stride = old_logp.stride(0), advantages.stride(0)
    if ref_logp is not None:
        t.ref_logp, t.ref_stride = ref_logp.data_ptr(), ref_logp.stride(0)
    t.clip_low, t.clip_high, t.kl_coef = clip_low, clip_high, kl_coef
    return t


def policy_loss_fwd(logits, labels, old_logp, advantages, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                    logit_scale=1.0, ignored_index=-100):
    out = _fast_policy_loss_fwd(logits, labels, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef,
                                logit_scale, ignored_index)
    if out is not None:  # the C++ fast path took the common case
        return out
    what = "policy_loss_fwd"
    dev = _lib.require_cuda(logits, labels, old_logp, advantages, ref_logp, what=what)
    _check(logits, labels, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, logit_scale, what)
    n = logits.shape[0]
    loss, logp, lse, kl = (_rows.empty_f32(n, logits) for _ in range(4))
    if n == 0:
        return loss, logp, lse, kl
    rows, keep = _rows.rows(logits, labels, logit_scale, ignored_index)
    terms = _terms(old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef)
    _lib.launch(dev, "dslpg_policy_loss_fwd", ctypes.addressof(rows), ctypes.addressof(terms), loss.data_ptr(),
                logp.data_ptr(), lse.data_ptr(), kl.data_ptr())
    return loss, logp, lse, kl


def policy_loss_bwd(dloss, logits, lse, labels, old_logp, advantages, ref_logp=None, clip_low=0.2, clip_high=0.2,
                    kl_coef=0.0, logit_scale=1.0, ignored_index=-100):
    out = _fast_policy_loss_bwd(dloss, logits, lse, labels, old_logp, advantages, ref_logp, clip_low, clip_high,
                                kl_coef, logit_scale, ignored_index)
    if out is not None:
        return out
    what = "policy_loss_bwd"
    dev = _lib.require_cuda(dloss, logits, lse, labels, old_logp, advantages, ref_logp, what=what)
    _check(logits, labels, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, logit_scale, what)
    n = logits.shape[0]
    _rows.check_vector(dloss, n, "dloss", what)
    _rows.check_vector(lse, n, "lse", what)
    dlogits = _rows.empty_grad(logits)
    if n == 0:
        return dlogits
    lse = lse.contiguous()
    rows, keep = _rows.rows(logits, labels, logit_scale, ignored_index)
    terms = _terms(old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef)
    _lib.launch(dev, "dslpg_policy_loss_bwd", ctypes.addressof(rows), ctypes.addressof(terms), dloss.data_ptr(),
                dloss.stride(0), lse.data_ptr(), dlogits.data_ptr(), logits.shape[1])
    return dlogits


def policy_loss_fwd_bwd(logits, labels, old_logp, advantages, dloss, ref_logp=None, clip_low=0.2, clip_high=0.2,
                        kl_coef=0.0, logit_scale=1.0, ignored_index=-100):
    out = _fast_policy_loss_fwd_bwd(logits, labels, old_logp, advantages, dloss, ref_logp, clip_low, clip_high,
                                    kl_coef, logit_scale, ignored_index)
    if out is not None:
        return out
    what = "policy_loss_fwd_bwd"
    dev = _lib.require_cuda(logits, labels, old_logp, advantages, dloss, ref_logp, what=what)
    _check(logits, labels, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, logit_scale, what)
    n = logits.shape[0]
    _rows.check_vector(dloss, n, "dloss", what)
    loss, logp, lse, kl = (_rows.empty_f32(n, logits) for _ in range(4))
    dlogits = _rows.empty_grad(logits)
    if n == 0:
        return loss, logp, lse, kl, dlogits
    rows, keep = _rows.rows(logits, labels, logit_scale, ignored_index)
    terms = _terms(old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef)
    _lib.launch(dev, "dslpg_policy_loss_fwd_bwd", ctypes.addressof(rows), ctypes.addressof(terms), dloss.data_ptr(),
                dloss.stride(0), loss.data_ptr(), logp.data_ptr(), lse.data_ptr(), kl.data_ptr(), dlogits.data_ptr(),
                logits.shape[1])
    return loss, logp, lse, kl, dlogits

"""CUDA (sm_100a) RMSNorm of each query and key head with the rotary position
rotation in the same pass.

``qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6,
sections=None, interleaved=False)`` returns ``(q_out, k_out)``: each head
normalised over its features as ``rms_norm`` does (weights ``[head_dim]``),
then rotated as ``rope`` does, in fp32 with one rounding at the end.

``qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions,
inv_freq, eps=1e-6, sections=None, interleaved=False)`` returns ``(dq, dk,
dq_weight, dk_weight)``; the weights' gradients are float32 sums over all tokens
and heads, in a fixed order. Layouts are those of ``rope``.
"""
import ctypes

import torch

from .. import _heads, _lib

_fast_qk_norm_rope = _lib.fast_op("qk_norm_rope")
_fast_qk_norm_rope_bwd = _lib.fast_op("qk_norm_rope_bwd")


def _check_weights(q_weight, k_weight, d, what):
    code = _lib.float_code(q_weight, f"{what} q_weight")
    if _lib.float_code(k_weight, f"{what} k_weight") != code:
        raise TypeError(f"{what}: q_weight and k_weight must have one dtype, got {q_weight.dtype} and {k_weight.dtype}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(w.shape) != (d,):
            raise ValueError(f"{what}: {name} must have shape ({d},), got {tuple(w.shape)}")


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None, interleaved=False):
    out = _fast_qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, interleaved)
    if out is not None:  # the C++ fast path took the common case
        return out
    what = "qk_norm_rope"
    dev = _lib.require_cuda(q, k, q_weight, k_weight, positions, inv_freq, what=what)
    _heads.check_layout(q, k, positions, inv_freq, sections, what)
    _check_weights(q_weight, k_weight, q.shape[-1], what)
    q, k = _heads.dense_last(q), _heads.dense_last(k)
    qw, kw = q_weight.contiguous(), k_weight.contiguous()
    pos, freq, heads = _heads.layout(q, k, positions, inv_freq, sections, interleaved, what, weight=qw)
    q_out, k_out = _heads.empty_rows(q), _heads.empty_rows(k)
    if q.numel() + k.numel() == 0:
        return q_out, k_out
    _lib.launch(dev, "dslpg_qk_norm_rope_fwd", q.data_ptr(), k.data_ptr(), qw.data_ptr(), kw.data_ptr(),
                pos.data_ptr(), freq.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), ctypes.addressof(heads),
                float(eps))
    return q_out, k_out


def qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None,
                     interleaved=False):
    out = _fast_qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps, sections,
                                 interleaved)
    if out is not None:
        return out
    what = "qk_norm_rope_bwd"
    dev = _lib.require_cuda(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, what=what)
    _heads.check_layout(q, k, positions, inv_freq, sections, what)
    _check_weights(q_weight, k_weight, q.shape[-1], what)
    _heads.check_like(dq_out, q, "dq_out", what)
    _heads.check_like(dk_out, k, "dk_out", what)
    q, k, dq_out, dk_out = (_heads.dense_last(t) for t in (q, k, dq_out, dk_out))
    qw, kw = q_weight.contiguous(), k_weight.contiguous()
    pos, freq, heads = _heads.layout(q, k, positions, inv_freq, sections, interleaved, what, dq_out, dk_out, qw)
    dq, dk = _heads.empty_rows(q), _heads.empty_rows(k)
    if q.numel() + k.numel() == 0:
        return dq, dk, *(torch.zeros(w.shape, dtype=torch.float32, device=w.device) for w in (qw, kw))
    dqw, dkw = (torch.empty(w.shape, dtype=torch.float32, device=w.device) for w in (qw, kw))
    need = ctypes.c_int64(0)
    _lib.check(_lib.load().dslpg_qk_norm_rope_bwd_workspace_bytes(q.shape[-1], ctypes.byref(need)), what)
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
    _lib.launch(dev, "dslpg_qk_norm_rope_bwd", dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(),
                qw.data_ptr(), kw.data_ptr(), pos.data_ptr(), freq.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                dqw.data_ptr(), dkw.data_ptr(), ctypes.addressof(heads), float(eps), ws.data_ptr(), need.value)
    return dq, dk, dqw, dkw

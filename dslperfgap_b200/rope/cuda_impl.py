"""CUDA (sm_100a) rotary position rotation of query and key heads.

``rope(q, k, positions, inv_freq, sections=None, interleaved=False)`` returns
``(q_out, k_out)``; ``rope_bwd(dq_out, dk_out, positions, inv_freq, ...)`` the
gradients ``(dq, dk)``. The suite has no kernel of this kind; the calling
convention is the other operators'.

q and k are ``[tokens, heads, head_dim]`` or ``[batch, seq, heads, head_dim]``
(any strides with a dense last axis, so views into one projection output are
read in place); outputs are dense. ``inv_freq`` (float32, n values) rotates the
first 2n features: pairs (i, i + n), or (2i, 2i + 1) when ``interleaved``; the
others pass through; it has to be finite. Angles are right to fp32 for positions up to 2^38 in size
(and |inv_freq| up to 2^18). ``positions`` (int32 or int64) has q's token axes, or broadcasts to them. With ``sections`` (one to four counts that add up to n) it
has one more leading axis, and frequency i turns by the axis whose section
holds i: time, height and width of video patches, for instance.
"""
import ctypes

from .. import _heads, _lib

_fast_rope = _lib.fast_op("rope")
_fast_rope_bwd = _lib.fast_op("rope_bwd")


def rope(q, k, positions, inv_freq, sections=None, interleaved=False):
    out = _fast_rope(q, k, positions, inv_freq, sections, interleaved)
    if out is not None:  # the C++ fast path took the common case
        return out
    return _rotate(q, k, positions, inv_freq, sections, interleaved, "rope", "dslpg_rope_fwd")


def rope_bwd(dq_out, dk_out, positions, inv_freq, sections=None, interleaved=False):
    out = _fast_rope_bwd(dq_out, dk_out, positions, inv_freq, sections, interleaved)
    if out is not None:
        return out
    return _rotate(dq_out, dk_out, positions, inv_freq, sections, interleaved, "rope_bwd", "dslpg_rope_bwd")


def _rotate(q, k, positions, inv_freq, sections, interleaved, what, entry):
    dev = _lib.require_cuda(q, k, positions, inv_freq, what=what)
    _heads.check_layout(q, k, positions, inv_freq, sections, what)
    q, k = _heads.dense_last(q), _heads.dense_last(k)
    pos, freq, heads = _heads.layout(q, k, positions, inv_freq, sections, interleaved, what)
    q_out, k_out = _heads.empty_rows(q), _heads.empty_rows(k)
    if q.numel() + k.numel() == 0:
        return q_out, k_out
    _lib.launch(dev, entry, q.data_ptr(), k.data_ptr(), pos.data_ptr(), freq.data_ptr(), q_out.data_ptr(),
                k_out.data_ptr(), ctypes.addressof(heads))
    return q_out, k_out

"""Refusals of rope and qk_norm_rope that need no GPU: the argument checks on
host tensors, the C entry points' own, and host tensors at the public calls."""
import ctypes

import pytest
import torch

import dslperfgap_b200 as B
from dslperfgap_b200 import _heads, _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def good():
    return dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), positions=torch.zeros(3, dtype=torch.long),
                inv_freq=torch.ones(32), sections=None)


def test_good_layouts():
    a = good()
    _heads.check_layout(**a, what="t")
    pos, freq, h = _heads.layout(**a, interleaved=True, what="t")
    assert (h.batch, h.seq, h.q_heads, h.k_heads, h.head_dim, h.rotary_dim) == (1, 3, 4, 2, 64, 64)
    assert list(h.q_strides) == [0, 256, 64] and list(h.position_strides) == [0, 0, 1] and h.interleaved == 1
    a.update(q=torch.zeros(5, 3, 4, 64), k=torch.zeros(5, 3, 2, 64), positions=torch.zeros(2, 1, 3, dtype=torch.int32),
             sections=(20, 12))
    _heads.check_layout(**a, what="t")
    pos, freq, h = _heads.layout(**a, interleaved=False, what="t")
    assert (h.batch, h.seq, h.axes) == (5, 3, 2) and list(h.sections) == [20, 12, 0, 0]
    assert list(h.position_strides) == [3, 0, 1] and h.positions_dtype == _lib.I32


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), TypeError),
    (dict(q=torch.zeros(4, 64), k=torch.zeros(2, 64)), ValueError),
    (dict(q=torch.zeros(1, 1, 3, 4, 64), k=torch.zeros(1, 1, 3, 4, 64)), ValueError),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros(4, 2, 64)), ValueError),
    (dict(k=torch.zeros(3, 2, 32)), ValueError),
    (dict(k=torch.zeros(1, 3, 2, 64)), ValueError),
    (dict(q=torch.zeros(3, 4, 1026), k=torch.zeros(3, 2, 1026)), ValueError),
    (dict(q=torch.zeros(3, 4, 0), k=torch.zeros(3, 2, 0)), ValueError),
    (dict(q=torch.zeros(1, 1, 2).expand(1 << 20, 1 << 10, 2), k=torch.zeros(1, 1, 2).expand(1 << 20, 1, 2),
          inv_freq=torch.ones(1)), ValueError),
    (dict(positions=torch.zeros(3)), TypeError),
    (dict(positions=torch.zeros(3, dtype=torch.int16)), TypeError),
    (dict(inv_freq=torch.ones(32, dtype=torch.float64)), TypeError),
    (dict(inv_freq=torch.ones(33)), ValueError),
    (dict(inv_freq=torch.ones(0)), ValueError),
    (dict(inv_freq=torch.ones(1, 32)), ValueError),
    (dict(sections=(16, 15)), ValueError),
    (dict(sections=(40, -8)), ValueError),
    (dict(sections=()), ValueError),
    (dict(sections=(8, 8, 8, 4, 4)), ValueError),
])
def test_check_layout_refuses(change, error):
    with pytest.raises(error):
        _heads.check_layout(**{**good(), **change}, what="t")


@pytest.mark.parametrize("positions,sections", [(torch.zeros(4, dtype=torch.long), None),
                                                (torch.zeros(2, 3, dtype=torch.long), None),
                                                (torch.zeros(3, 3, dtype=torch.long), (16, 16))])
def test_positions_that_do_not_broadcast(positions, sections):
    with pytest.raises(ValueError, match="broadcast"):
        _heads.layout(**{**good(), "positions": positions, "sections": sections}, interleaved=False, what="t")


def test_host_tensors_are_refused():
    a = good()
    w = torch.ones(64)
    with pytest.raises(ValueError, match="CUDA"):
        B.rope(a["q"], a["k"], a["positions"], a["inv_freq"])
    with pytest.raises(ValueError, match="CUDA"):
        B.rope_bwd(a["q"], a["k"], a["positions"], a["inv_freq"])
    with pytest.raises(ValueError, match="CUDA"):
        B.qk_norm_rope(a["q"], a["k"], w, w, a["positions"], a["inv_freq"])
    with pytest.raises(ValueError, match="CUDA"):
        B.qk_norm_rope_bwd(a["q"], a["k"], a["q"], a["k"], w, w, a["positions"], a["inv_freq"])
    with pytest.raises(TypeError):
        B.rope([1.0], a["k"], a["positions"], a["inv_freq"])


def heads(**change):
    h = _lib.Heads()
    h.batch, h.seq, h.q_heads, h.k_heads, h.head_dim, h.rotary_dim = 1, 4, 2, 1, 64, 64
    h.q_strides[:] = (0, 128, 64)
    h.k_strides[:] = (0, 64, 64)
    h.position_strides[:] = (0, 0, 1)
    h.sections[:] = (32, 0, 0, 0)
    h.axes, h.dtype, h.weight_dtype, h.positions_dtype = 1, _lib.BF16, _lib.BF16, _lib.I64
    for name, v in change.items():
        if isinstance(v, tuple):
            getattr(h, name)[:] = v
        else:
            setattr(h, name, v)
    return h


@pytest.mark.parametrize("change,rc", [
    (dict(dtype=3), -3), (dict(positions_dtype=0), -3), (dict(batch=-1), -2), (dict(seq=-2), -2),
    (dict(q_heads=-1), -2), (dict(head_dim=0), -2), (dict(head_dim=1026, rotary_dim=64), -2), (dict(rotary_dim=0), -2),
    (dict(rotary_dim=66), -2), (dict(rotary_dim=31), -2), (dict(batch=1 << 20, seq=1 << 20), -2),
    (dict(batch=1 << 40, seq=1 << 40), -2), (dict(q_heads=1 << 29), -2), (dict(axes=0), -5), (dict(axes=5), -5),
    (dict(sections=(31, 0, 0, 0)), -5), (dict(axes=2, sections=(33, -1, 0, 0)), -5)])
def test_c_entries_refuse_layouts(lib, change, rc):
    h = heads(**change)
    at = ctypes.addressof(h)
    assert lib.dslpg_rope_fwd(16, 16, 16, 16, 16, 16, at, None) == rc
    assert lib.dslpg_rope_bwd(16, 16, 16, 16, 16, 16, at, None) == rc
    assert lib.dslpg_qk_norm_rope_fwd(16, 16, 16, 16, 16, 16, 16, 16, at, 1e-6, None) == rc
    assert lib.dslpg_qk_norm_rope_bwd(*[16] * 12, at, 1e-6, 16, 1 << 30, None) == rc


def test_c_entries_refuse_pointers_eps_and_workspace(lib):
    h = heads()
    at = ctypes.addressof(h)
    for i in range(7):
        args = [16] * 6 + [at]
        args[i] = None
        assert lib.dslpg_rope_fwd(*args, None) == -1, i
        assert lib.dslpg_rope_bwd(*args, None) == -1, i
    for i in range(9):
        args = [16] * 8 + [at]
        args[i] = None
        assert lib.dslpg_qk_norm_rope_fwd(*args, 1e-6, None) == -1, i
    for i in range(13):
        args = [16] * 12 + [at]
        args[i] = None
        assert lib.dslpg_qk_norm_rope_bwd(*args, 1e-6, 16, 1 << 30, None) == -1, i
    assert lib.dslpg_qk_norm_rope_bwd(*[16] * 12, at, 1e-6, None, 1 << 30, None) == -1
    need = ctypes.c_int64(0)
    assert lib.dslpg_qk_norm_rope_bwd_workspace_bytes(64, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.dslpg_qk_norm_rope_bwd_workspace_bytes(0, ctypes.byref(need)) == -2
    assert lib.dslpg_qk_norm_rope_bwd_workspace_bytes(64, None) == -1
    assert lib.dslpg_qk_norm_rope_bwd(*[16] * 12, at, 1e-6, 16, need.value - 1, None) == -5
    for eps in (-1.0, float("nan"), float("inf")):
        assert lib.dslpg_qk_norm_rope_fwd(*[16] * 8, at, eps, None) == -4
        assert lib.dslpg_qk_norm_rope_bwd(*[16] * 12, at, eps, 16, 1 << 30, None) == -4
    bad = heads(weight_dtype=4)
    assert lib.dslpg_qk_norm_rope_fwd(*[16] * 8, ctypes.addressof(bad), 1e-6, None) == -3


def test_empty_is_a_no_op(lib):
    for change in (dict(batch=0), dict(seq=0), dict(q_heads=0, k_heads=0)):
        h = heads(**change)
        assert lib.dslpg_rope_fwd(None, None, 16, 16, None, None, ctypes.addressof(h), None) == 0
        assert lib.dslpg_qk_norm_rope_fwd(None, None, 16, 16, 16, 16, None, None, ctypes.addressof(h), 1e-6, None) == 0

"""Refusals of policy_loss and preference_loss that need no GPU: the argument
checks on host tensors, the C entry points' own, and host tensors at the public
calls."""
import ctypes
import inspect

import pytest
import torch

import dslperfgap_b200 as B
from dslperfgap_b200 import _lib, _logit_rows, build
from dslperfgap_b200.policy_loss import cuda_impl as policy
from dslperfgap_b200.preference_loss import cuda_impl as preference


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def good_policy():
    return dict(logits=torch.zeros(4, 10), labels=torch.zeros(4, dtype=torch.long), old_logp=torch.zeros(4),
                advantages=torch.zeros(4), ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, logit_scale=1.0)


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(4, 10, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(4)), ValueError),
    (dict(logits=torch.zeros(4, 0)), ValueError),
    (dict(logits=torch.zeros(1, 1).expand(4, (1 << 30) + 1)), ValueError),
    (dict(labels=torch.zeros(4)), TypeError),
    (dict(labels=torch.zeros(5, dtype=torch.long)), ValueError),
    (dict(labels=torch.zeros(4, 1, dtype=torch.long)), ValueError),
    (dict(old_logp=torch.zeros(4, dtype=torch.bfloat16)), TypeError),
    (dict(old_logp=torch.zeros(3)), ValueError),
    (dict(advantages=torch.zeros(1)), ValueError),
    (dict(advantages=torch.tensor(1.0)), ValueError),
    (dict(ref_logp=torch.zeros(4, 1)), ValueError),
    (dict(ref_logp=torch.zeros(4).double()), TypeError),
    (dict(clip_low=-0.1), ValueError), (dict(clip_low=1.5), ValueError), (dict(clip_low=float("nan")), ValueError),
    (dict(clip_high=-0.1), ValueError), (dict(clip_high=float("nan")), ValueError),
    (dict(kl_coef=float("inf")), ValueError), (dict(logit_scale=float("nan")), ValueError),
])
def test_policy_check_refuses(change, error):
    policy._check(**good_policy(), what="t")
    with pytest.raises(error):
        policy._check(**{**good_policy(), **change}, what="t")


def good_pairs():
    return dict(logits=torch.zeros(4, 10), labels=torch.zeros(4, dtype=torch.long),
                seq_starts=torch.tensor([0, 2, 4]), beta=0.1, smoothing=0.0, logit_scale=1.0)


@pytest.mark.parametrize("change,error", [
    (dict(seq_starts=torch.zeros(3)), TypeError),
    (dict(seq_starts=torch.tensor([0])), ValueError),
    (dict(seq_starts=torch.tensor([0, 2])), ValueError),
    (dict(seq_starts=torch.tensor([0, 1, 2, 4])), ValueError),
    (dict(seq_starts=torch.tensor([[0, 1, 2]])), ValueError),
    (dict(beta=float("inf")), ValueError), (dict(smoothing=-0.1), ValueError), (dict(smoothing=1.1), ValueError),
    (dict(smoothing=float("nan")), ValueError), (dict(logit_scale=float("inf")), ValueError),
])
def test_preference_check_refuses(change, error):
    assert preference._check(**good_pairs(), what="t") == 1
    with pytest.raises(error):
        preference._check(**{**good_pairs(), **change}, what="t")


def test_host_tensors_are_refused():
    a, v, y = torch.zeros(4, 10), torch.zeros(4), torch.zeros(4, dtype=torch.long)
    s = torch.tensor([0, 2, 4])
    for call in (lambda: B.policy_loss_fwd(a, y, v, v), lambda: B.policy_loss_bwd(v, a, v, y, v, v),
                 lambda: B.policy_loss_fwd_bwd(a, y, v, v, v), lambda: B.preference_loss_fwd(a, y, s, v),
                 lambda: B.preference_loss_bwd(v[:1], a, v, y, s, v[:2])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        B.policy_loss_fwd([0.0], y, v, v)


def test_rows_of_views():
    x = torch.zeros(6, 40)
    r, _ = _logit_rows.rows(x[:, :30], torch.zeros(6, dtype=torch.int32), 0.5, -1)
    assert (r.n_rows, r.n_cols, r.row_stride, r.ignored_index, r.labels_dtype) == (6, 30, 40, -1, _lib.I32)
    r, keep = _logit_rows.rows(x.t(), torch.zeros(40, dtype=torch.long), 1.0, -100)
    assert (r.n_rows, r.n_cols, r.row_stride) == (40, 6, 6) and keep[0].is_contiguous()
    r, keep = _logit_rows.rows(x[:1].expand(9, 40), torch.zeros(9, dtype=torch.long), 1.0, -100)
    assert r.row_stride == 40 and keep[0].is_contiguous()  # rows that lie on one another are copied


def test_default_arguments_agree():
    """Forward, backward and both take one set of options with one set of defaults."""
    names = ("clip_low", "clip_high", "kl_coef", "logit_scale", "ignored_index", "ref_logp")
    sigs = [inspect.signature(f).parameters for f in (B.policy_loss_fwd, B.policy_loss_bwd, B.policy_loss_fwd_bwd)]
    assert all(s[n].default == sigs[0][n].default for s in sigs for n in names)
    sigs = [inspect.signature(f).parameters for f in (B.preference_loss_fwd, B.preference_loss_bwd)]
    assert all(s[n].default == sigs[0][n].default for s in sigs for n in ("beta", "smoothing", "logit_scale"))


def rows(**change):
    r = _lib.LogitRows()
    r.logits = r.labels = 16
    r.n_rows, r.n_cols, r.row_stride, r.ignored_index = 4, 10, 10, -100
    r.logit_scale, r.logits_dtype, r.labels_dtype = 1.0, _lib.BF16, _lib.I64
    for k, v in change.items():
        setattr(r, k, v)
    return r


def terms(**change):
    t = _lib.PolicyTerms()
    t.old_logp = t.advantages = t.ref_logp = 16
    t.old_stride = t.advantages_stride = t.ref_stride = 1
    t.clip_low = t.clip_high = 0.2
    for k, v in change.items():
        setattr(t, k, v)
    return t


def pairs(**change):
    t = _lib.PairTerms()
    t.seq_starts = t.ref_logp = 16
    t.n_pairs, t.ref_stride, t.beta, t.starts_dtype = 1, 1, 0.1, _lib.I64
    for k, v in change.items():
        setattr(t, k, v)
    return t


def every(lib, r, t, p):
    """The status of each entry with these structures (None: left out)."""
    at = lambda s: ctypes.addressof(s) if s is not None else None  # noqa: E731
    out = []
    if t is not False:
        out += [lib.dslpg_policy_loss_fwd(at(r), at(t), 16, 16, 16, 16, None),
                lib.dslpg_policy_loss_bwd(at(r), at(t), 16, 1, 16, 16, 10, None),
                lib.dslpg_policy_loss_fwd_bwd(at(r), at(t), 16, 1, 16, 16, 16, 16, 16, 10, None)]
    if p is not False:
        out += [lib.dslpg_preference_loss_fwd(at(r), at(p), 16, 16, 16, 16, None),
                lib.dslpg_preference_loss_bwd(at(r), at(p), 16, 1, 16, 16, 16, 10, None)]
    return set(out)


@pytest.mark.parametrize("change,rc", [
    (dict(logits_dtype=3), -3), (dict(labels_dtype=0), -3), (dict(n_rows=-1), -2), (dict(n_cols=0), -2),
    (dict(n_cols=(1 << 30) + 1, row_stride=1 << 31), -2), (dict(row_stride=9), -2),
    (dict(logit_scale=float("nan")), -5), (dict(logits=None), -1), (dict(labels=None), -1)])
def test_c_entries_refuse_rows(lib, change, rc):
    assert every(lib, rows(**change), terms(), pairs()) == {rc}


@pytest.mark.parametrize("change,rc", [
    (dict(old_logp=None), -1), (dict(advantages=None), -1), (dict(old_stride=-1), -2), (dict(ref_stride=-1), -2),
    (dict(clip_low=1.5), -5), (dict(clip_low=float("nan")), -5), (dict(clip_high=-1), -5),
    (dict(kl_coef=float("inf")), -5)])
def test_c_entries_refuse_policy_terms(lib, change, rc):
    assert every(lib, rows(), terms(**change), False) == {rc}


@pytest.mark.parametrize("change,rc", [
    (dict(seq_starts=None), -1), (dict(starts_dtype=0), -3), (dict(n_pairs=0), -2), (dict(ref_stride=-1), -2),
    (dict(beta=float("nan")), -5), (dict(smoothing=1.5), -5)])
def test_c_entries_refuse_pair_terms(lib, change, rc):
    assert every(lib, rows(), False, pairs(**change)) == {rc}


def test_c_entries_refuse_missing_structures_and_outputs(lib):
    assert every(lib, None, terms(), pairs()) == {-1} and every(lib, rows(), None, None) == {-1}
    held = rows(), terms(), pairs()
    r, t, p = (ctypes.addressof(s) for s in held)
    for i in range(4):
        out = [16] * 4
        out[i] = None
        assert lib.dslpg_policy_loss_fwd(r, t, *out, None) == -1
        assert lib.dslpg_preference_loss_fwd(r, p, *out, None) == -1
    for i in range(6):
        out = [16] * 6
        out[i] = None
        assert lib.dslpg_policy_loss_fwd_bwd(r, t, out[0], 1, *out[1:], 10, None) == -1
    for i in range(3):
        out = [16] * 3
        out[i] = None
        assert lib.dslpg_policy_loss_bwd(r, t, out[0], 1, *out[1:], 10, None) == -1
    for i in range(4):
        out = [16] * 4
        out[i] = None
        assert lib.dslpg_preference_loss_bwd(r, p, out[0], 1, *out[1:], 10, None) == -1
    assert lib.dslpg_policy_loss_bwd(r, t, 16, -1, 16, 16, 10, None) == -2
    assert lib.dslpg_policy_loss_bwd(r, t, 16, 1, 16, 16, 9, None) == -2
    assert lib.dslpg_preference_loss_bwd(r, p, 16, 1, 16, 16, 16, 9, None) == -2


def test_no_rows_is_a_no_op(lib):
    r, t = rows(n_rows=0, logits=None, labels=None), terms(old_logp=None, advantages=None)
    assert lib.dslpg_policy_loss_fwd(ctypes.addressof(r), ctypes.addressof(t), None, None, None, None, None) == 0
    assert lib.dslpg_policy_loss_bwd(ctypes.addressof(r), ctypes.addressof(t), None, 0, None, None, 10, None) == 0

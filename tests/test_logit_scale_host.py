"""logit_scale of the losses on rows of logits: 0, or 1e-30 to 1e30 in size. Beyond that the float32 constant of the
kernels' exponents would no longer be the scale that was asked for."""
import ctypes

import pytest
import torch

from dslperfgap_b200 import _lib, _logit_rows, build
from test_logit_loss_host import every, pairs, rows, terms

GOOD = [0.0, -0.0, 1.0, -1.0, 1e-30, -1e-30, 1e30, -1e30, 40.0]
BAD = [1e-31, -1e-31, 1e-45, 1.1e30, -1e31, 3e38, 1e39, -1e300, float("inf"), float("nan")]


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.mark.parametrize("scale", BAD)
def test_wrappers_refuse(scale):
    x, y = torch.zeros(4, 10), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match="logit_scale"):
        _logit_rows.check_rows(x, y, scale, "t")


@pytest.mark.parametrize("scale", BAD)
def test_c_entries_refuse(lib, scale):
    assert every(lib, rows(logit_scale=scale), terms(), pairs()) == {-5}


@pytest.mark.parametrize("scale", GOOD)
def test_others_are_taken(lib, scale):
    x, y = torch.zeros(4, 10), torch.zeros(4, dtype=torch.long)
    _logit_rows.check_rows(x, y, scale, "t")
    none, none_t = rows(logit_scale=scale, n_rows=0), terms(old_logp=None, advantages=None)
    assert lib.dslpg_policy_loss_fwd(ctypes.addressof(none), ctypes.addressof(none_t), None, None, None, None, None) == 0

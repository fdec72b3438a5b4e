"""A checkout whose library is not built: the wrappers' own checks come first, and what passes them fails at the launch,
naming the build."""
import importlib

import pytest
import torch

from dslperfgap_b200 import _lib

X, V, Y = torch.zeros(4, 10), torch.zeros(4), torch.zeros(4, dtype=torch.long)
Q, POS, FREQ, W = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.long), torch.ones(32), torch.ones(64)
S = torch.tensor([0, 2, 4])
CALLS = [("rms_norm", "rms_norm", (X, (10,), torch.ones(10))), ("softmax", "softmax", (X,)),
         ("rope", "rope", (Q, Q, POS, FREQ)), ("rope", "rope_bwd", (Q, Q, POS, FREQ)),
         ("qk_norm_rope", "qk_norm_rope", (Q, Q, W, W, POS, FREQ)),
         ("qk_norm_rope", "qk_norm_rope_bwd", (Q, Q, Q, Q, W, W, POS, FREQ)),
         ("policy_loss", "policy_loss_fwd", (X, Y, V, V)), ("policy_loss", "policy_loss_bwd", (V, X, V, Y, V, V)),
         ("policy_loss", "policy_loss_fwd_bwd", (X, Y, V, V, V)),
         ("preference_loss", "preference_loss_fwd", (X, Y, S, V)),
         ("preference_loss", "preference_loss_bwd", (V[:1], X, V, Y, S, V[:2]))]


@pytest.fixture
def unbuilt(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "none.so")
    for name in ("_lib", "_fast", "_torch_ops"):
        monkeypatch.setattr(_lib, name, None)


@pytest.mark.parametrize("module,name,args", CALLS)
def test_host_tensors_are_named(unbuilt, monkeypatch, module, name, args):
    mod = importlib.import_module(f"dslperfgap_b200.{module}.cuda_impl")
    monkeypatch.setattr(mod, f"_fast_{name}", _lib.fast_op(name))
    with pytest.raises(ValueError, match="CUDA"):
        getattr(mod, name)(*args)


def test_a_launch_names_the_build(unbuilt):
    with pytest.raises(RuntimeError, match="not built"):
        _lib.launch(torch.device("cuda", 0), "dslpg_softmax_fwd")


def test_a_library_built_later_is_found(unbuilt, monkeypatch, tmp_path):
    op = _lib.fast_op("softmax")
    assert op(X) is None
    (tmp_path / "none.so").touch()
    monkeypatch.setattr(_lib, "torch_ops", lambda: type("M", (), {"softmax": staticmethod(lambda x: "taken")}))
    assert op(X) == "taken"

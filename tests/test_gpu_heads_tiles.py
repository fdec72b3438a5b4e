"""Tiles of the per-head operators beyond the small cases: tokens cut into parts whose tiles outnumber the ring's stages,
and the weights' gradients over a training batch."""
import pytest
import torch

import dslperfgap_b200 as B
import heads_ref as R
from test_gpu_heads import EPS, check_all, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,dt", [((3, 259), 32, 8, 128, "f32"), ((777,), 64, 8, 128, "bf16"),
                                               ((2, 301), 64, 16, 256, "f32"), ((601,), 1, 90, 128, "f16")])
def test_tokens_larger_than_a_stage(tokens, hq, hk, d, dt, inter):
    """More than 32 KB a token (backward: x and dy): 600 to 800 tokens of two parts or more are ten tiles or more for each
    of 148 CTAs, whose rings hold six."""
    check_all(tokens, hq, hk, d, d, dt, inter)


def test_weight_gradients_of_a_training_batch():
    """16384 tokens of 32 + 8 heads: a lane adds 82 rows one after another (28 tiles of 32 groups over 11 warps), then 4
    rows of a group, 11 warps, 19 CTAs and 8 strides: 124 half steps of the terms' sizes at most, beside each term's."""
    q, k, qw, kw, pos, freq, _ = make((4, 4096), 32, 8, 128, 128, "bf16")
    g = torch.Generator(device="cuda").manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in (q, k))
    out = B.qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq, eps=EPS)
    phi = R.angles(pos, freq, None, (4, 4096))
    for i, (dy, x, w) in enumerate(((dq, q, qw), (dk, k, kw))):
        dx, dw, slack, terms = R.backward(dy, x, w, phi, False, EPS)
        R.close(out[i], dx, slack, f"dx[{i}]")
        R.close(out[2 + i], dw, (124 * R.U + R.BWD) * terms, f"dw[{i}]")

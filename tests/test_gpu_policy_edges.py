"""policy_loss at the edges of its formulas: an advantage of 0 with a ratio beyond float32, and a sampled token whose
logit is masked, with a reference."""
import pytest
import torch

import dslperfgap_b200 as B
from loss_ref import U

pytestmark = pytest.mark.gpu

WAYS = ["short", "two_pass", "vocabulary"]


def rows(way, n_rows, seed=0):
    """Logits of a row length that takes the named kernel."""
    n = {"short": 1024, "two_pass": 1001, "vocabulary": 40001}[way]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n_rows, n, generator=g, device="cuda")
    y = torch.randint(0, n, (n_rows,), generator=g, device="cuda")
    return x, y, torch.log_softmax(x.double(), 1).gather(1, y[:, None])[:, 0]


def all_ways(x, y, old, adv, dloss, **how):
    fwd = B.policy_loss_fwd(x, y, old, adv, **how)
    both = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how)
    dx = B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how)
    return fwd, both[:4], both[4], dx


@pytest.mark.parametrize("clip_high", [0.2, float("inf")])
@pytest.mark.parametrize("way", WAYS)
def test_zero_advantage_and_ratio_beyond_float32(way, clip_high):
    """min(r A, clip(r) A) is 0 at A = 0 whatever r is: no loss and no gradient, not 0 times infinity."""
    x, y, logp = rows(way, 6)
    old, adv = logp.float().clone(), torch.zeros(6, device="cuda")
    old[0], old[1], old[2] = logp[0] - 95, logp[1] - 1000, logp[2] + 1000
    adv[1], adv[5] = -0.0, 0.5
    dloss = torch.ones(6, device="cuda")
    fwd, both, g_both, g_bwd = all_ways(x, y, old, adv, dloss, clip_high=clip_high)
    for t in (fwd, both):
        assert (t[0][:5] == 0).all() and t[0][5] != 0
    for g in (g_both, g_bwd):
        assert not g[:5].any() and g[5].any() and g.isfinite().all()
    # beside a KL term: that term alone
    ref = (logp + 0.5).float()
    fwd, both, g_both, g_bwd = all_ways(x, y, old, adv, dloss, ref_logp=ref, kl_coef=0.1, clip_high=clip_high)
    fwd0, both0, g0_both, g0_bwd = all_ways(x, y, logp.float(), adv, dloss, ref_logp=ref, kl_coef=0.1,
                                            clip_high=clip_high)
    assert torch.equal(fwd[0][:5], fwd0[0][:5]) and torch.equal(both[0][:5], both0[0][:5])
    assert torch.equal(g_both[:5], g0_both[:5]) and torch.equal(g_bwd[:5], g0_bwd[:5])
    # a ratio that is not a number still shows, and an infinite one of another advantage too
    old[0], adv[1] = float("nan"), -1.0
    loss = B.policy_loss_fwd(x, y, old, adv)[0]
    assert loss[0].isnan() and loss[1] == float("inf")


@pytest.mark.parametrize("kl_coef", [0.0, 0.1])
@pytest.mark.parametrize("way", WAYS)
def test_masked_sampled_token_with_reference(way, kl_coef):
    """logp = -inf against a finite reference: exp(d) - d - 1 grows without bound, so kl is infinite, not NaN; the other
    infinite differences keep their limits."""
    x, y, logp = rows(way, 5, seed=1)
    old, ref = logp.float(), (logp + 0.25).float()
    x[1, y[1]] = float("-inf")
    ref[2] = float("-inf")
    inf = float("inf")
    fwd, both, _, _ = all_ways(x, y, old, torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), ref_logp=ref,
                               kl_coef=kl_coef)
    for loss, lp, lse, kl in (fwd, both):
        assert lp[1] == -inf and kl[1] == inf and kl[2] == inf
        assert loss[1] == (inf if kl_coef else 0) and (loss[2] == inf if kl_coef else loss[2].isfinite())
        # d is 1/4, off by half steps of lse, logp and the reference's rounding (sizes below 64) and the sum's 160
        d = torch.tensor(0.25, dtype=torch.float64, device="cuda")
        slack = torch.expm1(d) * U * (160 + 4 * 64) + 16 * U
        assert ((kl[[0, 3, 4]].double() - (torch.expm1(d) - d)).abs() <= slack).all()

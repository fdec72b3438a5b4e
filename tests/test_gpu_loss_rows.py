"""Which rows each CTA of the loss kernels takes: fused calls of many more rows than a block of labels or a grid holds,
with left-out rows at random, in long runs and at either end, every output poisoned beforehand so that a row that nothing
writes shows; and rows masked with the type's lowest value throughout that several CTAs share."""
import ctypes

import pytest
import torch

import dslperfgap_b200 as B
import loss_ref as L
from dslperfgap_b200 import _lib, _logit_rows
from dslperfgap_b200.policy_loss.cuda_impl import _terms
from heads_ref import close

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LO, HI, KL, SCALE = 0.2, 0.3, 0.1, 0.8


def left_out(kind, rows, g):
    out = torch.zeros(rows, dtype=torch.bool, device="cuda")
    if kind == "random":
        out = torch.rand(rows, generator=g, device="cuda") < 0.3
    elif kind == "runs":  # 300 left out, 170 counted: longer than a block of 128 labels, and out of step with it
        out = torch.arange(rows, device="cuda") % 470 < 300
    elif kind == "front":
        out[:rows * 2 // 3] = True
    elif kind == "back":
        out[rows // 3:] = True
    return out


def fused_poisoned(x, y, old, adv, dloss, ref):
    """policy_loss_fwd_bwd through the C entry, into outputs full of NaN."""
    n, cols = x.shape
    rows, keep = _logit_rows.rows(x, y, SCALE, -100)
    terms = _terms(old, adv, ref, LO, HI, KL)
    out = [torch.full((n,), float("nan"), device="cuda") for _ in range(4)]
    out.append(torch.full((n, cols), float("nan"), dtype=x.dtype, device="cuda"))
    _lib.launch(x.device, "dslpg_policy_loss_fwd_bwd", ctypes.addressof(rows), ctypes.addressof(terms),
                dloss.data_ptr(), 1, *(t.data_ptr() for t in out), cols)
    return out


@pytest.mark.parametrize("kind", ["none", "random", "runs", "front", "back", "all"])
@pytest.mark.parametrize("rows,cols,pad,dt", [
    (3000, 1001, 0, "bf16"), (2500, 1001, 0, "f32"), (2500, 1001, 7, "f16"),  # blocks of 128 labels, 1184 CTAs
    (2500, 9001, 0, "bf16"), (1100, 9001, 0, "f32"), (2500, 9001, 23, "bf16"),  # blocks of 1024, 148 CTAs
    (1300, 40000, 0, "bf16"), (4001, 1000, 0, "bf16")])  # one phase; short rows
def test_every_row_is_written(rows, cols, pad, dt, kind):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (2.5 * rn(rows, cols + pad)).to(DT[dt])[:, :cols]
    y = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    logp = torch.log_softmax(x.double() * SCALE, 1).gather(1, y[:, None])[:, 0]
    # ratios well inside the borders, or well outside
    old = (logp - torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, 0.1, 0.6)).float()
    ref, adv, dloss = (logp + 0.3 * rn(rows)).float(), rn(rows), torch.rand(rows, generator=g, device="cuda") + 0.5
    if kind == "all":
        y[:] = -100
    else:
        y[left_out(kind, rows, g)] = -100
    want = L.policy(x, y, old, adv, dloss, ref, LO, HI, KL, SCALE, -100)
    got = fused_poisoned(x, y, old, adv, dloss, ref)
    for name, t in zip(("loss", "logp", "lse", "kl", "grad"), got):
        close(t, *want[name], name)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", [128256, 128255])
def test_shared_rows_masked_with_the_lowest_value(cols, dt):
    """A few long rows, of which several CTAs take a stretch each: uniform, so that the backward forms their statistics
    again in each of them."""
    low = torch.finfo(DT[dt]).min
    x = torch.full((4, cols), low, device="cuda", dtype=DT[dt])
    x[1] = -x[1]
    x[2, ::3] = 0
    y = torch.tensor([5, cols - 1, 9, -100], device="cuda")
    count = torch.tensor([cols, cols, (cols + 2) // 3], device="cuda", dtype=torch.float64)
    lp, old, one = -count.log(), torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    old[:3] = lp
    loss, logp, lse, kl = B.policy_loss_fwd(x, y, old, one)
    dx = B.policy_loss_bwd(one, x, lse, y, old, one)
    both = B.policy_loss_fwd_bwd(x, y, old, one, one)
    close(logp[:3], lp, 16 * L.U * lp.abs(), "logp")
    p = torch.where(x[:3] == x[:3].amax(1, keepdim=True), lp.exp()[:, None], 0.0)
    want = p - torch.zeros_like(p).scatter_(1, y[:3, None], 1.0)  # ratio 1, advantage 1
    for t in (dx, both[4]):
        close(t[:3], want, 64 * L.U * want.abs(), "grad")
        assert not t[3].any()
    # the same rows as two sequences of one pair: slope -beta / 2 at margin 0
    starts, ref = torch.tensor([0, 1, 2], device="cuda"), old.clone()
    fwd = B.preference_loss_fwd(x, y, starts, ref, beta=0.5)
    dx = B.preference_loss_bwd(one[:1], x, fwd[3], y, starts, fwd[1], beta=0.5)
    # the margin is off by the two sums' allowances (16 half steps of |lp| < 12 each) times beta = 1/2, sigmoid near 0 by
    # half of that, relative: 96 half steps, beside the 64 of the probabilities
    slope = 0.25 * torch.tensor([1.0, -1.0], device="cuda", dtype=torch.float64)[:, None]
    close(dx[:2], slope * want[:2], 160 * L.U * (slope * want[:2]).abs(), "preference grad")
    assert not dx[2:].any()


@pytest.mark.parametrize("rows,cols,pad,dt", [(3000, 1001, 0, "bf16"), (2500, 1001, 7, "f16"), (2500, 9001, 0, "f32"),
                                              (700, 40001, 0, "bf16"), (5, 1 << 20, 8, "bf16"), (40, 128256, 0, "f32")])
def test_fused_call_of_rows_that_two_kernels_take(rows, cols, pad, dt):
    """Many rows off the 16-byte boundary, and few long ones, are the forward's and the backward's work one after another
    (one kernel for both took up to nine times as long): the same bits as the two calls."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = rn(rows, cols + pad).to(DT[dt])[:, :cols]
    y = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    y[1::5] = -100
    old, adv, dloss, ref = -7 + rn(rows), rn(rows), rn(rows), -7 + rn(rows)
    how = dict(ref_logp=ref, kl_coef=KL, logit_scale=SCALE)
    fwd = B.policy_loss_fwd(x, y, old, adv, **how)
    dx = B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how)
    both = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how)
    for name, a, b in zip(("loss", "logp", "lse", "kl", "grad"), both, (*fwd, dx)):
        assert torch.equal(a, b), name

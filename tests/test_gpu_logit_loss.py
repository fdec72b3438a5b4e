"""policy_loss and preference_loss, forward, backward and both at once, against
a plain 64-bit evaluation: types, row lengths from one column to a vocabulary,
left-out rows, clipping on either side, KL term on and off, strided and
broadcast inputs, masked logits, empty sequences, graphs and streams."""
import importlib
import math

import pytest
import torch

import dslperfgap_b200 as B
import loss_ref as L
from dslperfgap_b200 import _lib
from heads_ref import close

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LO, HI = 0.2, 0.3


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_policy(r, n, dt, seed=0, scale=0.8, pad=0):
    g = gen(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (2.5 * rn(r, n + pad)).to(DT[dt])[:, :n]
    y = torch.randint(0, n, (r,), generator=g, device="cuda")
    y[::2] = x[::2].float().argmax(1)
    logp = torch.log_softmax(x.double() * scale, 1).gather(1, y[:, None])[:, 0]
    d = 0.4 * rn(r)
    for edge in (math.log(1 - LO), math.log(1 + HI)):  # a border decided by rounding has two right gradients
        d = torch.where((d - edge).abs() < 1e-3, d + 3e-3, d)
    ref = (logp + 0.3 * rn(r)).float()
    old, adv, dloss = (logp - d).float(), rn(r), torch.rand(r, generator=g, device="cuda") + 0.5
    if r >= 6:
        y[1], y[3], y[5] = -100, n, -7  # ignored, and no column
    return x, y, old, adv, dloss, ref


def check(got, want, names):
    for name, t in zip(names, got):
        value, slack = want[name]
        assert t.shape == value.shape, name
        close(t, value, slack, name)


def run_policy(x, y, old, adv, dloss, ref, kl=0.1, scale=0.8, ignored=-100):
    how = dict(ref_logp=ref, clip_low=LO, clip_high=HI, kl_coef=kl, logit_scale=scale, ignored_index=ignored)
    want = L.policy(x, y, old, adv, dloss, ref, LO, HI, kl, scale, ignored)
    fwd = B.policy_loss_fwd(x, y, old, adv, **how)
    check(fwd, want, ("loss", "logp", "lse", "kl"))
    both = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how)
    check(both, want, ("loss", "logp", "lse", "kl", "grad"))
    dx = B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how)
    check([dx], want, ("grad",))
    for t in (both[4], dx):
        assert t.dtype == x.dtype and t.is_contiguous()
    return fwd, both, dx


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 37, 64, 1000, 1001, 4096, 32001, 40000])
def test_policy_row_lengths(n, dt):
    run_policy(*make_policy(9, n, dt, seed=n))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("r", [1, 2, 147, 149, 300, 1500])
def test_policy_row_counts(r, dt):
    run_policy(*make_policy(r, 2048, dt, seed=r))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r", [3, 200])
def test_policy_vocabulary(r, dt):
    run_policy(*make_policy(r, 128256, dt, seed=5))


@pytest.mark.parametrize("n", [250000, 700001, 1 << 20])
def test_policy_long_rows(n):
    run_policy(*make_policy(6, n, "bf16", seed=5))


@pytest.mark.parametrize("n", [5, 256, 5000])
def test_policy_scalar_path(n):
    with _lib.kernel_path("stream"):
        run_policy(*make_policy(40, n, "bf16"))


@pytest.mark.parametrize("scale", [1.0, 1 / 0.7, 0.05, -0.8, 0.0, 40.0])
def test_policy_scales(scale):
    run_policy(*make_policy(20, 3000, "f32", scale=scale), scale=scale)


@pytest.mark.parametrize("kl", [0.0, 0.2, -0.1])
def test_policy_kl_term(kl):
    a = make_policy(50, 1000, "f32")
    run_policy(*a, kl=kl)
    out = run_policy(*a[:5], None, kl=kl)
    assert not out[0][3].any()


def test_policy_kl_near_zero_and_far():
    x, y, old, adv, dloss, _ = make_policy(64, 500, "f32")
    logp = torch.log_softmax(x.double() * 0.8, 1).gather(1, y.clamp(0, 499)[:, None])[:, 0]
    for step in (1e-6, 1e-3, 0.2499, 0.2501, 3.0, 20.0):
        for sign in (-1, 1):
            run_policy(x, y, old, adv, dloss, (logp + sign * step).float())


def test_policy_views_strides_and_labels():
    x, y, old, adv, dloss, ref = make_policy(30, 1000, "bf16", pad=24)
    want = run_policy(x, y, old, adv, dloss, ref)
    spread = lambda t: torch.stack([t, t + 1], 1)[:, 0]  # noqa: E731
    got = run_policy(x, y.to(torch.int32), spread(old), spread(adv), spread(dloss), spread(ref))
    for a, b in zip(got[1], want[1]):
        assert torch.equal(a, b)
    run_policy(x, y, old, torch.tensor(0.7, device="cuda").expand(30), torch.ones(1, device="cuda").expand(30), ref)
    run_policy(x[:, 1:999], y.clamp(max=900), old, adv, dloss, ref)  # rows off the 16-byte boundary
    run_policy(x.t().contiguous().t(), y, old, adv, dloss, ref)  # columns first
    run_policy(x[:1].expand(30, 1000), y, old, adv, dloss, ref)  # one row for all
    run_policy(x, y, old, adv, dloss, ref, ignored=int(y[0]))


def test_policy_left_out_rows_are_not_read():
    """Logits, old_logp, advantages, ref_logp and dloss of left-out rows may hold anything."""
    x, y, old, adv, dloss, ref = make_policy(12, 4096, "bf16")
    out = y.clone().fill_(False).bool()
    out[[1, 3, 5]] = True
    for t in (x, old, adv, dloss, ref):
        t[out] = float("nan")
    how = dict(ref_logp=ref, kl_coef=0.1)
    fwd = B.policy_loss_fwd(x, y, old, adv, **how)
    both = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how)
    dx = B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how)
    for t in (*fwd, *both, dx):
        assert not t[out].any() and t[~out].isfinite().all()
    none = torch.full_like(y, -100)
    for t in B.policy_loss_fwd_bwd(x, none, old, adv, dloss, **how):
        assert not t.any()


def test_policy_masked_logits():
    """-inf logits have probability 0; a row of them, a NaN or a +inf logit makes its own row NaN."""
    x, y, old, adv, dloss, ref = make_policy(12, 3000, "f32")
    x[0, :] = float("-inf")
    x[0, y[0]] = 1.0  # one column left: logp 0
    x[2, 100:2900] = float("-inf")
    y[2] = 5
    x[4, 100:2900] = torch.finfo(torch.float32).min
    y[4] = 17
    lp = torch.log_softmax(x.double() * 0.8, 1).gather(1, y.clamp(0, 2999)[:, None])[:, 0]
    old, ref = (lp - 0.1).float(), (lp + 0.1).float()
    fwd, both, dx = run_policy(x, y, old, adv, dloss, ref)
    assert fwd[1][0] == 0 and not dx[2, 100:2900].any() and not both[4][2, 100:2900].any()
    x[6, :], x[8, 9], x[10, 9] = float("-inf"), float("nan"), float("inf")
    how = dict(ref_logp=ref, kl_coef=0.1, logit_scale=0.8)
    fwd = B.policy_loss_fwd(x, y, old, adv, **how)
    both = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how)
    dx = B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how)
    bad = torch.zeros(12, dtype=torch.bool, device="cuda")
    bad[[6, 8, 10]] = True
    for t in fwd[:3] + both[:3]:
        assert t[bad].isnan().all() and t[~bad].isfinite().all()
    for t in (both[4], dx):
        assert t[bad].isnan().all() and t[~bad].isfinite().all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scale", [1.0, 0.8])
def test_rows_masked_with_the_lowest_value(dt, scale):
    """All columns at the type's lowest value: a uniform row, forward and backward."""
    n = 2048
    x = torch.full((3, n), torch.finfo(DT[dt]).min, device="cuda", dtype=DT[dt])
    x[1] = -x[1]
    x[2, ::2] = 0  # half of the columns
    y = torch.tensor([5, 6, 8], device="cuda")
    lp = -torch.tensor([n, n, n // 2], device="cuda", dtype=torch.float64).log()
    old, adv = lp.float(), torch.ones(3, device="cuda")
    loss, logp, lse, kl = B.policy_loss_fwd(x, y, old, adv, logit_scale=scale)
    both = B.policy_loss_fwd_bwd(x, y, old, adv, adv, logit_scale=scale)
    dx = B.policy_loss_bwd(adv, x, lse, y, old, adv, logit_scale=scale)
    close(logp, lp, 16 * L.U * lp.abs(), "logp")
    assert torch.equal(both[1], logp)
    p = torch.where(x == x.amax(1, keepdim=True), lp.exp()[:, None], 0.0)
    want = -scale * (torch.zeros_like(p).scatter_(1, y[:, None], 1.0) - p)  # ratio 1, advantage 1
    for t in (both[4], dx):
        close(t, want, 64 * L.U * want.abs(), "grad")


def test_policy_sampled_token_masked():
    """The label's own logit -inf: ratio 0, no gradient from the policy term."""
    x, y, old, adv, dloss, _ = make_policy(4, 1000, "f32")
    x[0, y[0]] = float("-inf")
    loss, logp, lse, kl, dx = B.policy_loss_fwd_bwd(x, y, old, adv.abs(), dloss, logit_scale=0.8)
    assert logp[0] == float("-inf") and loss[0] == 0 and not dx[0].any() and lse[0].isfinite()


def test_policy_gradient_against_differences():
    x, y, old, adv, dloss, ref = make_policy(5, 11, "f32", seed=3)
    dx = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, ref_logp=ref, clip_low=LO, clip_high=HI, kl_coef=0.1,
                               logit_scale=0.8)[4]
    f = lambda v: (L.policy(v, y, old, adv, dloss, ref, LO, HI, 0.1, 0.8, -100)["loss"][0] * dloss.double()).sum()  # noqa: E731
    h, x64 = 1e-5, x.double()
    for i in range(x.numel()):
        e = torch.zeros_like(x64).view(-1)
        e[i] = h
        slope = (f(x64 + e.view_as(x64)) - f(x64 - e.view_as(x64))) / (2 * h)
        # third derivatives of order 10 times h^2; 256 half steps (lse, ratio, exponent) of terms of order 10
        assert abs(dx.view(-1)[i].item() - slope.item()) < 1e-8 + 2560 * L.U


def test_policy_empty():
    x = torch.empty(0, 100, device="cuda")
    y, v = torch.empty(0, dtype=torch.long, device="cuda"), torch.empty(0, device="cuda")
    assert [t.shape for t in B.policy_loss_fwd(x, y, v, v)] == [(0,)] * 4
    assert [t.shape for t in B.policy_loss_fwd_bwd(x, y, v, v, v)] == [(0,)] * 4 + [(0, 100)]
    assert B.policy_loss_bwd(v, x, v, y, v, v).shape == (0, 100)


# ------------------------------------------------------------- preferences

def make_pairs(lengths, n, dt, seed=0, scale=0.8, before=0, tail=0):
    """Logits of len(lengths) sequences, `before` rows in front of them and `tail` behind."""
    g = gen(seed)
    r = before + sum(lengths) + tail
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (2.5 * rn(r, n)).to(DT[dt])
    y = torch.randint(0, n, (r,), generator=g, device="cuda")
    logp = torch.log_softmax(x.double() * scale, 1).gather(1, y[:, None])[:, 0]
    ref = (logp + 0.3 * rn(r) - 0.1).float()
    y[4::9] = -100
    starts = [before]
    for k in lengths:
        starts.append(starts[-1] + k)
    dloss = torch.rand(len(lengths) // 2, generator=g, device="cuda") + 0.5
    return x, y, torch.tensor(starts, device="cuda"), ref, dloss


def run_pairs(x, y, starts, ref, dloss, beta=0.3, smoothing=0.1, scale=0.8):
    how = dict(beta=beta, smoothing=smoothing, logit_scale=scale)
    want = L.preference(x, y, starts, ref, dloss, beta, smoothing, scale, -100)
    fwd = B.preference_loss_fwd(x, y, starts, ref, **how)
    check(fwd, want, ("loss", "log_ratio", "logp", "lse"))
    dx = B.preference_loss_bwd(dloss, x, fwd[3], y, starts, fwd[1], **how)
    check([dx], want, ("grad",))
    assert dx.dtype == x.dtype and dx.is_contiguous()
    return fwd, dx


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [3, 64, 1001, 32000])
def test_pairs_row_lengths(n, dt):
    run_pairs(*make_pairs([5, 9, 3, 12], n, dt, seed=n))


@pytest.mark.parametrize("lengths", [[1, 1], [0, 4], [0, 0], [3, 0, 0, 0, 7, 2], [1, 0, 1, 0], [300, 1], [700, 900] * 3,
                                     [2] * 66, [1] * 2000])
def test_pairs_sequences(lengths):
    run_pairs(*make_pairs(lengths, 500, "f32", seed=len(lengths)))


@pytest.mark.parametrize("before,tail", [(0, 0), (3, 0), (0, 5), (4, 7)])
def test_pairs_rows_outside(before, tail):
    x, y, starts, ref, dloss = make_pairs([8, 6, 7, 5], 1000, "bf16", before=before, tail=tail)
    x[:before], x[26 + before:], ref[:before], ref[26 + before:] = (float("nan"),) * 4
    fwd, dx = run_pairs(*(torch.nan_to_num(t) if t.is_floating_point() else t for t in (x, y, starts, ref, dloss)))
    got = B.preference_loss_fwd(x, y, starts, ref, beta=0.3, smoothing=0.1, logit_scale=0.8)
    again = B.preference_loss_bwd(dloss, x, got[3], y, starts, got[1], beta=0.3, smoothing=0.1, logit_scale=0.8)
    for a, b in zip((*got, again), (*fwd, dx)):
        assert torch.equal(a, b)


def test_pairs_vocabulary():
    run_pairs(*make_pairs([70, 90, 60, 81], 128256, "bf16", tail=9))


@pytest.mark.parametrize("beta,smoothing", [(0.1, 0.0), (5.0, 0.0), (-0.5, 0.2), (0.0, 0.0), (1.0, 1.0), (200.0, 0.3)])
def test_pairs_constants(beta, smoothing):
    run_pairs(*make_pairs([5, 9, 3, 12], 300, "f32"), beta=beta, smoothing=smoothing)


def test_pairs_types_and_strides():
    x, y, starts, ref, dloss = make_pairs([5, 9, 3, 12], 300, "bf16")
    fwd, dx = run_pairs(x, y, starts, ref, dloss)
    spread = lambda t: torch.stack([t, t + 1], 1)[:, 0]  # noqa: E731
    got, dx2 = run_pairs(x, y.int(), starts.int(), spread(ref), spread(dloss))
    got3, dx3 = run_pairs(x, spread(y), spread(starts), ref, dloss)
    for a, b, c in zip((*fwd, dx), (*got, dx2), (*got3, dx3)):
        assert torch.equal(a, b) and torch.equal(a, c)
    run_pairs(x[:, 1:299], y.clamp(max=290), starts, ref, dloss)
    run_pairs(x, y, starts, ref, torch.ones(1, device="cuda").expand(2))


def test_pairs_no_rows_and_no_bounds_in_order():
    x, y, starts, ref, dloss = make_pairs([5, 9, 3, 12], 300, "bf16")
    loss, ratio, logp, lse = B.preference_loss_fwd(x[:0], y[:0], torch.zeros(5, dtype=torch.long, device="cuda"), ref[:0])
    assert not ratio.any() and (loss - math.log(2)).abs().max() < 1e-6 and logp.numel() == lse.numel() == 0
    assert B.preference_loss_bwd(dloss, x[:0], lse, y[:0], starts, ratio).shape == (0, 300)
    # bounds that do not ascend, or lie outside: no result is promised, and nothing outside is touched
    for bad in ([9, 3, 20, 1, 29], [-5, 4, 1 << 40, 7, 1 << 50], [29, 29, 29, 29, 0], [1 << 62] * 5):
        b = torch.tensor(bad, device="cuda")
        out = B.preference_loss_fwd(x, y, b, ref)
        B.preference_loss_bwd(dloss, x, out[3], y, b, out[1])
    torch.cuda.synchronize()


def test_pairs_gradient_against_differences():
    x, y, starts, ref, dloss = make_pairs([2, 3, 3, 1], 7, "f32", seed=8)
    fwd = B.preference_loss_fwd(x, y, starts, ref, beta=0.5, smoothing=0.1, logit_scale=0.8)
    dx = B.preference_loss_bwd(dloss, x, fwd[3], y, starts, fwd[1], beta=0.5, smoothing=0.1, logit_scale=0.8)
    f = lambda v: (L.preference(v, y, starts, ref, dloss, 0.5, 0.1, 0.8, -100)["loss"][0] * dloss.double()).sum()  # noqa: E731
    h, x64 = 1e-5, x.double()
    for i in range(x.numel()):
        e = torch.zeros_like(x64).view(-1)
        e[i] = h
        slope = (f(x64 + e.view_as(x64)) - f(x64 - e.view_as(x64))) / (2 * h)
        assert abs(dx.view(-1)[i].item() - slope.item()) < 1e-8 + 2560 * L.U


# ------------------------------------------------------------- both

def calls():
    x, y, old, adv, dloss, ref = make_policy(40, 4096, "bf16")
    how = dict(ref_logp=ref, kl_coef=0.1)
    px, py, starts, pref, pd = make_pairs([5, 9, 3, 12], 1000, "bf16", tail=3)

    def run():
        fwd = B.policy_loss_fwd(x, y, old, adv, **how)
        out = (*fwd, *B.policy_loss_fwd_bwd(x, y, old, adv, dloss, **how),
               B.policy_loss_bwd(dloss, x, fwd[2], y, old, adv, **how))
        fwd = B.preference_loss_fwd(px, py, starts, pref)
        return (*out, *fwd, B.preference_loss_bwd(pd, px, fwd[3], py, starts, fwd[1]))
    return run, (x, adv, px)


def test_graph_other_stream_and_repeats():
    run, inputs = calls()
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run()
    torch.cuda.current_stream().wait_stream(side)
    for other in (run(), on_side):
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs, outs = [], []
    for _ in range(2):  # two graphs alive at once
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for t in inputs:
        t.copy_(torch.randn_like(t))
    want = run()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert _lib.take_wait_timeouts() == 0


def test_fast_path_equals_python_path(monkeypatch):
    assert _lib.torch_ops() is not None
    run, _ = calls()
    fast = run()
    for module, names in (("policy_loss", ("policy_loss_fwd", "policy_loss_bwd", "policy_loss_fwd_bwd")),
                          ("preference_loss", ("preference_loss_fwd", "preference_loss_bwd"))):
        mod = importlib.import_module(f"dslperfgap_b200.{module}.cuda_impl")
        for name in names:
            assert getattr(mod, f"_fast_{name}") is not None
            monkeypatch.setattr(mod, f"_fast_{name}", lambda *a: None)
    slow = run()
    assert len(fast) == len(slow) and all(torch.equal(a, b) for a, b in zip(fast, slow))


@pytest.mark.parametrize("n", [4096, 1001, 128256])
def test_guard_bytes_around_outputs(n):
    import ctypes
    from dslperfgap_b200 import _logit_rows as R
    from dslperfgap_b200.policy_loss.cuda_impl import _terms
    x, y, old, adv, dloss, ref = make_policy(13, n, "bf16")
    rows, keep = R.rows(x, y, 0.8, -100)
    terms = _terms(old, adv, ref, LO, HI, 0.1)
    want = B.policy_loss_fwd_bwd(x, y, old, adv, dloss, ref_logp=ref, clip_low=LO, clip_high=HI, kl_coef=0.1,
                                 logit_scale=0.8)
    bufs = [torch.full((t.numel() * t.element_size() + 512,), 0xA5, dtype=torch.uint8, device="cuda") for t in want]
    at = [b.data_ptr() + 256 for b in bufs]
    _lib.launch(x.device, "dslpg_policy_loss_fwd_bwd", ctypes.addressof(rows), ctypes.addressof(terms),
                dloss.data_ptr(), 1, *at, n)
    torch.cuda.synchronize()
    for b, t in zip(bufs, want):
        assert (b[:256] == 0xA5).all() and (b[-256:] == 0xA5).all()
        assert torch.equal(b[256:-256], t.contiguous().view(-1).view(torch.uint8))

"""One post-training step through the operators together: a layer whose queries
and keys are normalised and rotated (time, height and width positions), causal
attention, a head, and the policy or the preference loss on its logits, with the
gradients led back through all of it to the weights. Held against the same step
in 64 bits by differentiation."""
import pytest
import torch

import dslperfgap_b200 as B

pytestmark = pytest.mark.gpu

BATCH, SEQ, DIM, HQ, HK, D, VOCAB = 6, 40, 48, 4, 2, 32, 211
SECTIONS, EPS, SCALE = (8, 4, 4), 1e-6, 1.0 / 0.9
CLIP, KL, BETA = 0.2, 0.05, 0.3


class NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, pos, freq):
        ctx.save_for_backward(q, k, qw, kw, pos, freq)
        return B.qk_norm_rope(q, k, qw, kw, pos, freq, eps=EPS, sections=SECTIONS)

    @staticmethod
    def backward(ctx, dq, dk):
        return *B.qk_norm_rope_bwd(dq, dk, *ctx.saved_tensors, eps=EPS, sections=SECTIONS), None, None


def weights(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return {"qkv": rn(DIM, (HQ + 2 * HK) * D) / DIM ** 0.5, "qw": 1 + 0.1 * rn(D), "kw": 1 + 0.1 * rn(D),
            "out": rn(HQ * D, DIM) / (HQ * D) ** 0.5, "head": 2 * rn(DIM, VOCAB) / DIM ** 0.5}


def data(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(BATCH, SEQ, DIM, generator=g, device="cuda")
    t = torch.arange(SEQ, device="cuda")
    pos = torch.stack([t + 100000, t // 6, t % 6]).unsqueeze(1).expand(-1, BATCH, -1)
    freq = 100.0 ** (-torch.arange(16, device="cuda") / 16)
    labels = torch.randint(0, VOCAB, (BATCH * SEQ,), generator=g, device="cuda")
    labels.view(BATCH, SEQ)[:, :9] = -100  # the prompt
    noise = torch.randn(3, BATCH * SEQ, generator=g, device="cuda")
    return x, pos, freq, labels, noise


def logits_of(w, x, pos, freq, norm_rope):
    qkv = x @ w["qkv"]
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([HQ * D, HK * D, HK * D], -1))
    q, k = norm_rope(q, k, w["qw"], w["kw"], pos, freq)
    k, v = (t.repeat_interleave(HQ // HK, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) / D ** 0.5
    s = s.masked_fill(torch.ones(SEQ, SEQ, device="cuda").triu(1).bool(), float("-inf"))
    y = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v).flatten(-2)
    return (torch.tanh(y @ w["out"]) @ w["head"]).flatten(0, 1)


def plain_norm_rope(q, k, qw, kw, pos, freq):
    axis = torch.repeat_interleave(torch.arange(3), torch.tensor(SECTIONS))
    phi = (pos.double()[axis].movedim(0, -1) * freq.double()).unsqueeze(-2)
    out = []
    for x, w in ((q, qw), (k, kw)):
        u = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        z = torch.complex(u[..., :16].contiguous(), u[..., 16:].contiguous()) * torch.polar(torch.ones_like(phi), phi)
        out.append(torch.cat([z.real, z.imag], -1))
    return out


def plain_logp(logits, labels):
    return torch.log_softmax(logits * SCALE, 1).gather(1, labels.clamp(min=0)[:, None])[:, 0]


def check(losses, grads, ref_losses, ref_grads):
    """Products of at most 240 terms one behind another (240 half steps of their size), six of them in a row between a
    logit and a weight's gradient, each at most doubling what is relative to its result's norm: 240 * 6 * 2 half steps."""
    bound = 240 * 6 * 2 * 2.0 ** -24
    assert (losses.double() - ref_losses).norm() <= bound * ref_losses.norm()
    for name, g in grads.items():
        off = (g.double() - ref_grads[name]).norm() / ref_grads[name].norm()
        assert off <= bound, (name, off.item())


@pytest.mark.parametrize("fused", [True, False])
def test_policy_step(fused):
    w, (x, pos, freq, labels, noise) = weights(1), data(2)
    keep = labels >= 0
    ref_w = {n: t.double().requires_grad_() for n, t in w.items()}
    logits = logits_of(ref_w, x.double(), pos, freq, plain_norm_rope)
    logp = plain_logp(logits, labels)
    # ratios on either side of the borders, none within 0.02 of one
    d = torch.where(noise[0] > 0.5, 0.4, torch.where(noise[0] < -0.5, -0.5, 0.1 * noise[0].clamp(-1, 1)))
    old, ref = (logp.detach() - d).float(), (logp.detach() + 0.3 * noise[1]).float()
    adv = noise[2]
    r, e = (logp - old.double()).exp(), ref.double() - logp
    loss = -torch.minimum(r * adv, r.clamp(1 - CLIP, 1 + CLIP) * adv) + KL * (torch.exp(e) - e - 1)
    ref_loss = torch.where(keep, loss, 0.0)
    weight = 1.0 / int(keep.sum())
    ref_grads = dict(zip(ref_w, torch.autograd.grad(ref_loss.sum() * weight, list(ref_w.values()))))

    own_w = {n: t.clone().requires_grad_() for n, t in w.items()}
    logits = logits_of(own_w, x, pos, freq, NormRope.apply)
    how = dict(ref_logp=ref, clip_low=CLIP, clip_high=CLIP, kl_coef=KL, logit_scale=SCALE)
    dloss = torch.tensor(weight, device="cuda").expand(labels.numel())
    if fused:
        loss, _, _, _, dlogits = B.policy_loss_fwd_bwd(logits.detach(), labels, old, adv, dloss, **how)
    else:
        loss, _, lse, _ = B.policy_loss_fwd(logits.detach(), labels, old, adv, **how)
        dlogits = B.policy_loss_bwd(dloss, logits.detach(), lse, labels, old, adv, **how)
    grads = dict(zip(own_w, torch.autograd.grad(logits, list(own_w.values()), dlogits)))
    check(loss, grads, ref_loss.detach(), ref_grads)


def test_preference_step():
    w, (x, pos, freq, labels, noise) = weights(3), data(4)
    starts = torch.arange(0, BATCH * SEQ + 1, SEQ, device="cuda")  # three chosen sequences, then three rejected
    ref_w = {n: t.double().requires_grad_() for n, t in w.items()}
    logp = plain_logp(logits_of(ref_w, x.double(), pos, freq, plain_norm_rope), labels)
    ref = (logp.detach() + 0.2 * noise[0]).float()
    part = torch.where(labels >= 0, logp - ref.double(), 0.0).view(BATCH, SEQ).sum(1)
    ref_loss = -torch.nn.functional.logsigmoid(BETA * (part[:3] - part[3:]))
    ref_grads = dict(zip(ref_w, torch.autograd.grad(ref_loss.mean(), list(ref_w.values()))))

    own_w = {n: t.clone().requires_grad_() for n, t in w.items()}
    logits = logits_of(own_w, x, pos, freq, NormRope.apply)
    how = dict(beta=BETA, logit_scale=SCALE)
    loss, ratio, _, lse = B.preference_loss_fwd(logits.detach(), labels, starts, ref, **how)
    dloss = torch.full((3,), 1 / 3, device="cuda")
    dlogits = B.preference_loss_bwd(dloss, logits.detach(), lse, labels, starts, ratio, **how)
    grads = dict(zip(own_w, torch.autograd.grad(logits, list(own_w.values()), dlogits)))
    check(loss, grads, ref_loss.detach(), ref_grads)


def test_step_in_a_graph_beside_an_eager_one():
    """A captured forward and backward replays right while the eager step's tensors live."""
    w, (x, pos, freq, labels, noise) = weights(1), data(2)
    q = (x @ w["qkv"])[..., :HQ * D].unflatten(-1, (HQ, D))
    k = (x @ w["qkv"])[..., HQ * D:(HQ + HK) * D].unflatten(-1, (HK, D))
    logits = (x @ w["qkv"] @ torch.randn(w["qkv"].shape[1], VOCAB, device="cuda")).flatten(0, 1)

    def step():
        yq, yk = B.qk_norm_rope(q, k, w["qw"], w["kw"], pos, freq, sections=SECTIONS)
        back = B.qk_norm_rope_bwd(yq, yk, q, k, w["qw"], w["kw"], pos, freq, sections=SECTIONS)
        loss = B.policy_loss_fwd_bwd(logits, labels, noise[0], noise[1], noise[2], ref_logp=noise[0], kl_coef=KL)
        return yq, yk, *back, *loss

    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    logits.mul_(0.5)
    w["qw"].add_(0.25)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
    assert not torch.equal(eager[0], want[0])

"""policy_loss and preference_loss in 64 bits, written from their formulas,
with the errors that a float32 evaluation may have beside them."""
import torch

U = 2.0 ** -24  # half a float32 step, relative


def rows(logits, labels, scale, ignored, inside=None):
    """z, lse, logp, which rows count, and the allowance E of logp and lse.

    E: each term of the sum of exponentials is 2^d with d off by half a step of itself and the exponential by 2^-22; at
    most 64 terms lie one behind another in a thread, then 13 levels of merging: together under 160 half steps of lse's
    sum, and a half step each of lse, of z at the label and of their difference."""
    z = logits.double() * scale
    n = z.shape[1]
    keep = (labels != ignored) & (labels >= 0) & (labels < n)
    if inside is not None:
        keep &= inside
    lse = torch.logsumexp(z, 1)
    zy = z.gather(1, labels.long().clamp(0, n - 1)[:, None])[:, 0]
    logp = zy - lse
    allow = U * (160 + 2 * lse.abs() + 2 * zy.abs())
    zero = lambda t: torch.where(keep, t, torch.zeros_like(t))  # noqa: E731
    return z, zero(lse), zero(logp), keep, zero(allow)


def grad(z, lse, labels, keep, weight, dweight, scale):
    """weight * scale * (onehot - p) and its allowance, weight being off by dweight: p = 2^(z c - lse c) has the rounding
    of both products in its exponent (1.5 half steps of each in natural units, 2 for their constants), 8 for the rest.
    Probabilities below 2^-126, the smallest normal float32, are flushed to 0: off by at most 2^-126 times the weight."""
    z = torch.where(keep[:, None], z, torch.zeros_like(z))
    p = (z - lse[:, None]).exp()
    one = torch.zeros_like(z).scatter_(1, labels.long().clamp(0, z.shape[1] - 1)[:, None], 1.0)
    g = weight[:, None] * scale * (one - p)
    off = U * (8 + 3.5 * z.abs() + 3.5 * lse.abs()[:, None])
    # (p = 0 of z = -inf is exact, where off is infinite)
    slack = abs(scale) * (dweight[:, None] * (one - p).abs() + weight.abs()[:, None] * (torch.where(p > 0, p * off, 0.0) + 2.0 ** -126)) + 4 * U * g.abs()
    zero = lambda t: torch.where(keep[:, None], t, torch.zeros_like(t))  # noqa: E731
    return zero(g), zero(slack)


def policy(logits, labels, old, adv, dloss, ref, lo, hi, kl_coef, scale, ignored):
    """{name: (value, allowance)} of loss, logp, lse, kl and grad."""
    z, lse, logp, keep, e = rows(logits, labels, scale, ignored)
    old, adv, dloss = old.double(), adv.double(), dloss.double()
    zero = lambda t: torch.where(keep, t, torch.zeros_like(t))  # noqa: E731
    r = (logp - old).exp()
    dr = r * (e + U * ((logp - old).abs() + 4))
    clipped = r.clamp(1 - lo, 1 + hi)
    loss = -torch.minimum(r * adv, clipped * adv)
    free = (r * adv <= clipped * adv) | (r * adv).isnan()
    g, dg = torch.where(free, -r * adv, torch.zeros_like(r)), torch.where(free, dr * adv.abs(), torch.zeros_like(r))
    # the borders 1 - lo and 1 + hi are float32 numbers
    dl = adv.abs() * (dr + 2 * U * clipped)
    kl, dkl = torch.zeros_like(r), torch.zeros_like(r)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.expm1(d) - d
        de = e + U * d.abs()
        dkl = torch.expm1(d).abs() * de + de ** 2 * d.exp() + 16 * U * kl + 4 * U * (d.abs() >= 0.25) * d.exp()
        if kl_coef:
            loss = loss + kl_coef * kl
            g = g - kl_coef * torch.expm1(d)
            dl = dl + abs(kl_coef) * (dkl + 2 * U * kl)
            dg = dg + abs(kl_coef) * (d.exp() * de + 4 * U * torch.expm1(d).abs())
    dl = dl + 2 * U * loss.abs()
    dlogits, slack = grad(z, lse, labels, keep, dloss * zero(g), dloss.abs() * zero(dg + 4 * U * g.abs()), scale)
    return {"loss": (zero(loss), zero(dl)), "logp": (logp, e), "lse": (lse, e), "kl": (zero(kl), zero(dkl)),
            "grad": (dlogits, slack)}


def softplus(x):
    return x.clamp(min=0) + torch.log1p((-x.abs()).exp())


def preference(logits, labels, starts, ref, dloss, beta, smoothing, scale, ignored):
    starts = [int(s) for s in starts]
    pairs, n = len(starts) // 2, logits.shape[0]
    at = torch.arange(n, device=logits.device)
    z, lse, logp, keep, e = rows(logits, labels, scale, ignored, (at >= starts[0]) & (at < starts[-1]))
    ratio, off, seq = [], [], torch.zeros(n, dtype=torch.long, device=logits.device)
    for s in range(2 * pairs):
        a, b = starts[s], starts[s + 1]
        seq[a:b] = s
        k = keep[a:b]
        ratio.append((logp[a:b] - ref[a:b].double())[k].sum())
        off.append((e[a:b] + U * logp[a:b].abs())[k].sum())
    ratio, off = torch.stack(ratio), torch.stack(off)
    off = off + U * ratio.abs()
    m, dm = beta * (ratio[:pairs] - ratio[pairs:]), abs(beta) * (off[:pairs] + off[pairs:])
    dm = dm + 2 * U * m.abs() + 2 * U * abs(beta) * (ratio[:pairs].abs() + ratio[pairs:].abs())
    loss = (1 - smoothing) * softplus(-m) + smoothing * softplus(m)
    slope = beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m))
    # sigmoid's own slope is at most the smaller of 1/4 and itself; 8 half steps for its evaluation in either term
    both = smoothing * torch.sigmoid(m) + (1 - smoothing) * torch.sigmoid(-m)
    dslope = abs(beta) * (both * dm.clamp(max=1) * 1.1 + 8 * U * both) + 4 * U * slope.abs()
    w, dw = dloss.double() * slope, dloss.double().abs() * dslope
    g, slack = grad(z, lse, labels, keep, torch.cat([w, -w])[seq], torch.cat([dw, dw])[seq], scale)
    return {"loss": (loss, dm + 4 * U * loss), "log_ratio": (ratio, off), "logp": (logp, e), "lse": (lse, e),
            "grad": (g, slack)}

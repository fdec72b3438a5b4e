"""The per-head operators in 64 bits, written from their formulas, with the
rounding allowances of a float32 evaluation."""
import torch

U = 2.0 ** -24  # half a float32 step, relative


def angles(positions, inv_freq, sections, tokens):
    """[*tokens, 1, n] angles in float64."""
    pos = positions.double()
    if sections is None:
        phi = pos.expand(tokens).unsqueeze(-1) * inv_freq.double()
    else:
        pos = pos.expand((len(sections),) + tuple(tokens))
        parts = inv_freq.double().split(list(sections))
        phi = torch.cat([p.unsqueeze(-1) * f for p, f in zip(pos, parts)], -1)
    return phi.unsqueeze(-2)


def turn(x, phi, interleaved):
    n = phi.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ya, yb = a * phi.cos() - b * phi.sin(), b * phi.cos() + a * phi.sin()
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def pair_size(x, n, interleaved):
    """|x_i| + |x_j| at both members of each pair; |x_d| past them."""
    v = x.abs()
    if interleaved:
        both = (v[..., 0:2 * n:2] + v[..., 1:2 * n:2]).repeat_interleave(2, -1)
    else:
        both = (v[..., :n] + v[..., n:2 * n]).repeat(*[1] * (v.dim() - 1), 2)
    return torch.cat([both, v[..., 2 * n:]], -1)


def norm(x, w, eps):
    rstd = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return x * rstd * w, rstd


def close(got, ref, slack, name=""):
    """got (any dtype) is ref (64 bits) rounded once: half a step of its dtype, the float32 slack on top."""
    dt = got.dtype
    half = torch.finfo(dt).eps / 2
    floor = torch.finfo(dt).smallest_normal * half  # half a step among the subnormals
    off = (got.double().cpu() - ref.cpu()).abs()
    allowed = half * (ref.abs() + slack).cpu() + slack.cpu() + floor
    bad = ~(off <= allowed)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{(off / allowed).nan_to_num(nan=float('inf')).max().item():.3g} times the allowance")


# Allowances, in float32 half steps U of the stated magnitudes. Forward: the D-term sum of squares (at most 16 terms one
# after another in a lane, then a tree: 8 in rstd, which has its square root), rsqrt 4, two products 2, the fraction of a
# turn and sincospi 4, the rotation 3: 21, taken as 32. Backward adds the sum c of the same shape (16 + tree) and its
# three products: 64.
FWD, BWD = 32 * U, 64 * U


def check_forward(got, x, w, phi, interleaved, eps, name=""):
    x = x.double()
    u = x if w is None else norm(x, w.double(), eps)[0]
    close(got, turn(u, phi, interleaved), FWD * pair_size(u, phi.shape[-1], interleaved), name)


def backward(dy, x, w, phi, interleaved, eps):
    """(dx, dw, slack of dx, slack of dw before the count of terms) of one tensor."""
    dy, x, w = dy.double(), x.double(), w.double()
    n = phi.shape[-1]
    g = turn(dy, -phi, interleaved)
    gs = pair_size(dy, n, interleaved)
    _, rstd = norm(x, torch.ones_like(w), eps)
    c = (w * g * x).mean(-1, keepdim=True)
    dx = rstd * (w * g - x * rstd ** 2 * c)
    cs = (w.abs() * gs * x.abs()).mean(-1, keepdim=True)
    slack = BWD * rstd * (w.abs() * gs + x.abs() * rstd ** 2 * cs)
    axes = tuple(range(x.dim() - 1))
    return dx, (g * x * rstd).sum(axes), slack, (gs * x.abs() * rstd).sum(axes)

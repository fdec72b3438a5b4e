"""Angles of rope at far positions, against exact arithmetic: position times
frequency as a fraction, reduced by 2 pi in integers."""
import math
from fractions import Fraction

import pytest
import torch

import dslperfgap_b200 as B
from dslperfgap_b200 import _lib

pytestmark = pytest.mark.gpu

BITS = 400
FREQS = [1.0, 0.75, 0.1, 0.8659643, 1e-2, 1e-4, 3.3e-7, 1e-12, -0.3, 3.7, 1000.5, 2.0 ** 20 - 0.25]
POSITIONS = [0, 1, -1, 5, -5, 131071, (1 << 31) - 1, 1 << 31, -(1 << 31), -(1 << 31) - 1, (1 << 32) + 12345, (1 << 36) + 7,
             (1 << 40) + 3, -(1 << 40) - 3, (1 << 50) + 1, (1 << 62) + 987654321, -(1 << 62) - 1, (1 << 63) - 1, -(1 << 63)]


def two_pi():
    """2 pi * 2^BITS by Machin's formula, pi / 4 = 4 arctan(1/5) - arctan(1/239), off by a few hundred units at most."""
    def arctan(q):
        term, total, k = (1 << BITS) // q, 0, 0
        while term:
            total += (term if k % 2 == 0 else -term) // (2 * k + 1)
            term //= q * q
            k += 1
        return total
    return 8 * (4 * arctan(5) - arctan(239))


def exact(positions, freqs):
    """[positions, freqs] cosines and sines, right to 64 bits."""
    turn = two_pi()
    phi = []
    for p in positions:
        for f in freqs:
            angle = Fraction(p) * Fraction(f)  # a float is a fraction
            whole = (angle.numerator << BITS) // angle.denominator
            phi.append((whole % turn) / (1 << BITS))
    phi = torch.tensor(phi, dtype=torch.float64).view(len(positions), len(freqs))
    return phi.cos(), phi.sin()


def test_two_pi():
    assert abs(two_pi() / (1 << BITS) - 2 * math.pi) < 1e-15


def turned(dt, inter, freq, pos):
    """cos and sin as the operator has them: features (1, 0) of one head, rotated."""
    n = freq.numel()
    x = torch.zeros(pos.numel(), 1, 2 * n, device="cuda", dtype=dt)
    if inter:
        x[..., 0::2] = 1
    else:
        x[..., :n] = 1
    y, _ = B.rope(x, x, pos, freq, interleaved=inter)
    y = y[:, 0].double().cpu()
    return (y[:, 0::2], y[:, 1::2]) if inter else (y[:, :n], y[:, n:])


# The turn of one step is off by half of 2^-64 turns, and by less than 2^-83 f turns in its second part (that part's
# constant by 2^-85 and the product by 2^-84 of f), both times the position. 32 bits: the angle as a fraction of a turn is cut to 2^-32 turns (1.5e-9 rad), then rounded to float32 (pi times half a
# step), sincospi is off by one step of 1 at most (2 half steps), the products with 1 and 0 are exact: below 6 half steps.
# 16 bits: the SFU's sine and cosine are off by 2^-21.2 at most, their argument by three roundings of at most pi half
# steps: below 2^-19.9. Both: one rounding of the result, among the subnormals half of one of them.
@pytest.mark.parametrize("path", ["auto", "stream"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt,slack", [(torch.float32, 6 * 2.0 ** -24), (torch.float16, 2.0 ** -19.9)])
def test_far_positions(dt, slack, inter, path):
    freq = torch.tensor(FREQS + [10000.0 ** (-i / 52) for i in range(52)], dtype=torch.float32)
    want = exact(POSITIONS, freq.tolist())
    pos = torch.tensor(POSITIONS, device="cuda")
    with _lib.kernel_path(path):
        got = turned(dt, inter, freq.cuda(), pos)
    half = torch.finfo(dt).eps / 2
    step = torch.tensor([abs(p) * 2 * math.pi for p in POSITIONS], dtype=torch.float64)[:, None]
    step = step * (2.0 ** -65 + freq.double().abs() * 2.0 ** -83)
    for g, w in zip(got, want):
        allowed = (slack + step) + half * (w.abs() + slack + step) + torch.finfo(dt).smallest_normal * half
        off = (g - w).abs()
        bad = [(POSITIONS[i], freq[j].item(), off[i, j].item()) for i, j in (off > allowed).nonzero().tolist()]
        assert bad == [], len(bad)


def test_far_and_near_positions_in_one_tile():
    """Tokens of one tile, and the axes of one token, far and near: the same bits as each alone."""
    n, g = 32, torch.Generator(device="cuda").manual_seed(0)
    freq = (10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)).float()
    q = torch.randn(6000, 2, 64, generator=g, device="cuda")
    k = torch.randn(6000, 1, 64, generator=g, device="cuda")
    pos = torch.randint(0, 100000, (3, 6000), generator=g, device="cuda")
    far = pos.clone()
    far[:, ::5] += 1 << 45
    far[1, 1::5] = -far[1, 1::5] - (1 << 61)
    sec = (16, 10, 6)
    near_q, near_k = B.rope(q, k, pos, freq, sections=sec)
    far_q, far_k = B.rope(q, k, far, freq, sections=sec)
    same = (far == pos).all(0)
    assert torch.equal(near_q[same], far_q[same]) and torch.equal(near_k[same], far_k[same])
    pick = (~same).nonzero()[:64, 0]
    for t in pick.tolist():
        one_q, _ = B.rope(q[t:t + 1], k[t:t + 1], far[:, t:t + 1], freq, sections=sec)
        assert torch.equal(one_q[0], far_q[t])

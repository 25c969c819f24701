"""Activations and their slopes relative to their own values, where an absolute tolerance would let a small value be anything.

float32: every value is a chain of operations that are off by one step (2^-23: exp2 and the reciprocal) or half of one; each test
counts them.  16-bit results: their rounding, u(t), and what their shorter forms leave."""
import math

import pytest
import torch

from tacotron2_amd import inversion as inv
from test_inversion import BF16, F16, F32, act64, slope64, tiny, u

gpu = pytest.mark.gpu


def through(z, name):
    """act(z) by dense: one input of weight 1."""
    one = torch.ones((1, 1), dtype=z.dtype, device="cuda")
    return inv.dense(z.cuda()[:, None], one, activation=name)[:, 0].double().cpu()


def slopes(z, name, dy=1.0):
    """act'(z) by dense_backward (dbias of one frame each would be many calls: dx of weight 1)."""
    zc = z.cuda()[:, None]
    one = torch.ones((1, 1), dtype=z.dtype, device="cuda")
    return inv.dense_backward(torch.full_like(zc, dy), torch.zeros_like(zc), one, zc, activation=name,
                              needs=(True, False, False))[0][:, 0].double().cpu()


def through_norm(z, name):
    """act(z) by group_norm: no spread, so its argument is the bias alone; a channel a value."""
    flat = torch.zeros((1, 2, z.numel()), dtype=z.dtype, device="cuda")
    return inv.group_norm(flat, 1, None, z.cuda(), activation=name)[0, 0].double().cpu()


def close(got, want, rel, floor, what):
    off = (got - want).abs() - (rel * want.abs() + floor)
    k = int(off.argmax())
    assert off[k] <= 0, f"{what}: {got[k]:.9g} against {want[k]:.9g}"


# -- gelu ------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("way", [through, through_norm])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gelu_keeps_its_negative_tail(dtype, way):
    """float32: Phi(-a) is t P(t) e: 1 + c a half a step, its reciprocal one, and again in P (|t P' / P| < 2): 4.5 half steps for each of
    the two; nine half steps of Horner's terms halved by t < 1; e two, two products, 1 - h and z: 18 half steps, 2^-19.8.
    16 bits: the result's rounding and 2^-14: as much and the exponential's argument of 104, rounded twice, 2^-17 of it."""
    z = torch.cat([torch.linspace(-12, 12, 1001), torch.linspace(-6, 0.5, 1001)]).to(dtype)
    got, want = way(z, "gelu"), act64(z.double(), "gelu")
    if dtype == F32:
        close(got, want, 2.0 ** -19.8, 2.0 ** -126, "gelu")
    else:
        close(got, want, u(dtype) + 2.0 ** -14, tiny(dtype), "gelu")


@gpu
def test_gelu_at_its_ends():
    z = torch.tensor([float("inf"), 3e38, 1e30, -1e30, -40.0, 0.0, float("nan")])
    y = through(z, "gelu")
    assert torch.equal(y[:3], z.double()[:3]) and not y[3:6].any() and y[6].isnan()
    for dtype in (F32, BF16, F16):
        ends = through(torch.tensor([float("inf"), -float("inf"), float("nan")]).to(dtype), "gelu")
        assert ends[0] == float("inf") and ends[1].isnan() and ends[2].isnan()       # as -inf times zero is


@gpu
def test_gelu_slope_in_float32():
    """Phi + z phi, each as above, their sum: of the larger of the two."""
    z = torch.linspace(-12, 12, 2001)
    d = z.double()
    parts = (0.5 * torch.special.erfc(-d / math.sqrt(2))) + (d * torch.exp(-d * d / 2)).abs() / math.sqrt(2 * math.pi)
    got = slopes(z, "gelu")
    assert ((got - slope64(d, "gelu")).abs() <= 2.0 ** -19.8 * parts + 2.0 ** -126).all()


# -- exp, and silu through it ------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("way", [through, through_norm])
def test_exp_and_silu_keep_float32_over_their_range(way):
    """exp: exp2 two half steps, the correction one, the subnormal range's last product one, and one for the argument's own rest.
    silu: that, 1 + e one, its reciprocal two, z one."""
    z = torch.cat([torch.linspace(-87, 88.5, 3001), torch.linspace(-2, 2, 1001)])
    d = z.double()
    close(way(z, "exp"), torch.exp(d), 5 * 2.0 ** -24, 2.0 ** -126, "exp")
    close(way(z, "silu"), d * torch.sigmoid(d), 9 * 2.0 ** -24, 2.0 ** -126 * 88, "silu")


@gpu
def test_exp_at_its_ends():
    inf = float("inf")
    z = torch.tensor([89.0, 200.0, 3e38, inf, -104.5, -200.0, -3e38, -inf, float("nan"), -100.0, 88.72, -87.4])
    y = through(z, "exp")
    assert (y[:4] == inf).all() and not y[4:8].any() and y[8].isnan()
    assert ((y[9:] - torch.exp(z[9:].double())).abs() <= 2.0 ** -21 * y[9:] + 2.0 ** -149).all()
    s = through(torch.tensor([inf, 3e38, -3e38, -200.0, float("nan")]), "silu")
    assert s[0] == inf and s[1] == z[2].double()
    assert not s[2:4].any() and s[4].isnan()


@gpu
def test_slopes_of_exp_and_silu_in_float32():
    """exp as above.  silu: s and 1 - s six half steps each, their product with z two more, the sum one: of the larger part."""
    z = torch.cat([torch.linspace(-80, 80, 2001), torch.linspace(-2, 2, 1001)])
    d = z.double()
    close(slopes(z, "exp"), torch.exp(d), 5 * 2.0 ** -24, 2.0 ** -126, "exp'")
    s, o = torch.sigmoid(d), torch.sigmoid(-d)
    assert ((slopes(z, "silu") - (s + d * s * o)).abs() <= 16 * 2.0 ** -24 * (s + (d * s * o).abs()) + 2.0 ** -126 * 80).all()
    ends = slopes(torch.tensor([200.0, 3e38, -200.0, -3e38]), "silu")
    assert torch.equal(ends.abs(), torch.tensor([1.0, 1.0, 0.0, 0.0]).double())


# -- tanh --------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("way", [through, through_norm])
def test_tanh_keeps_float32_around_the_end_of_its_series(way):
    """Near zero: z^2 and z^3 a half step each, of which at most 0.12 counts, five more in P, the sum one: 2 half steps.  Beyond 0.6:
    e <= 0.31, five half steps of it moved onto 1 - e >= 0.69 (three), 1 - e and 1 + e one each, the reciprocal two, one: 8."""
    z = torch.cat([torch.linspace(-1, 1, 4001), torch.linspace(-12, 12, 1001), torch.tensor([1e-6, -1e-30, 0.0, 50.0, -3e38])])
    close(way(z, "tanh"), torch.tanh(z.double()), 8 * 2.0 ** -24, 2.0 ** -149, "tanh")
    near = z[z.abs() < 0.59]
    close(way(near, "tanh"), torch.tanh(near.double()), 2 * 2.0 ** -24, 2.0 ** -149, "tanh near zero")
    ends = through(torch.tensor([float("inf"), -float("inf"), float("nan")]), "tanh")
    assert ends[0] == 1 and ends[1] == -1 and ends[2].isnan()


@gpu
def test_slope_of_tanh_in_float32():
    """4 e / (1 + e)^2: e five half steps, (1 + e) one, its reciprocal two, both twice, three products: 14."""
    z = torch.cat([torch.linspace(-40, 40, 2001), torch.linspace(-1, 1, 1001)])
    close(slopes(z, "tanh"), torch.cosh(z.double()) ** -2, 14 * 2.0 ** -24, 2.0 ** -126, "tanh'")

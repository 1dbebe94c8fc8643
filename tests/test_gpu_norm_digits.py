"""Group norm where digits or finiteness are easily lost: lanes without channels of
their own, activations near zero and in their tails.  Bounds in e = 2^-24."""
import math

import pytest
import torch

from seq_helpers import EPS, TYPES, assert_within
from test_gpu_group_norm import K, make
from zealot_b200 import sequence as S


# A constant group whose (0 - mean) rstd is infinite, at widths that leave some
# lanes of a group without a channel: nothing of those may reach the sums.  xh is 0
# everywhere, so dgamma is 0 and dbeta the sum of dy act'(0), a slope within 24 e; dx
# is rstd times what the rounding of a mean of equal terms leaves, three roundings.
@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["none", "elu", "silu", "gelu"])
@pytest.mark.parametrize("N,w", [(1, 25), (4, 25), (300, 17), (5, 9), (3, 50), (2, 113)])
def test_row_gradient_of_a_huge_constant(N, w, act, t):
    G = 10
    x = torch.full((N, G * w), 2.0 ** 120, device="cuda", dtype=TYPES[t])
    dy = torch.ones_like(x)
    ones, zeros = torch.ones(G * w, device="cuda"), torch.zeros(G * w, device="cuda")
    mean, rstd = torch.full((N, G), 2.0 ** 120, device="cuda"), torch.full((N, G), 316.0, device="cuda")
    dx, dgamma, dbeta = S.group_norm_grad(x, dy, G, ones, zeros, mean, rstd, act=act)
    slope = 0.5 if act in ("silu", "gelu") else 1.0
    assert torch.equal(dgamma, zeros)
    assert_within(dbeta, torch.full((G * w,), N * slope).double(), 24 * EPS * N * slope, "dbeta")
    assert_within(dx, torch.zeros(N, G * w).double(), 8 * EPS * 316 * slope, "dx")


def direct(z, act, N=1, L=None):
    """(y, act's slope) at z itself: with gamma 0 the norm's output is act(beta) and
    its gradient of beta, where dy is 1 in one row and 0 elsewhere, the slope."""
    C = z.numel()
    shape = (N, C) if L is None else (N, L, C)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(C)).cuda()
    gamma, beta = torch.zeros(C, device="cuda"), z.cuda()
    y, mean, rstd = S.group_norm(x, 16, gamma, beta, act=act, save=True)
    dy = torch.zeros_like(x)
    dy.view(-1, C)[0] = 1.0
    slope = S.group_norm_grad(x, dy, 16, gamma, beta, mean, rstd, act=act)[2]
    return y, slope


FORMS = [(3, None), (200, 30), (2, 3000)]  # rows, samples in a block, in two passes


# e^z - 1 from -1/2 on is a subtraction that at most doubles the exponential's
# 5 e; below it a series within 3 e.  The slope is the exponential: its argument's
# rounding adds |z| e.
@pytest.mark.gpu
@pytest.mark.parametrize("N,L", FORMS)
def test_elu_keeps_the_digits_of_a_small_argument(N, L):
    z = torch.cat([-torch.logspace(-30, 1.9, 960), torch.logspace(-30, 1.9, 48),
                   -torch.tensor([0.5, 0.4999999, 0.5000001, 0.0, 0.25, 1.0, 80.0, 86.0] * 2)])
    y, slope = direct(z, "elu", N, L)
    z = z.double()
    want = torch.where(z > 0, z, torch.expm1(z))
    assert_within(y, want.expand(y.shape), 16 * EPS * want.abs(), "y")
    assert_within(slope, torch.exp(z.clamp(max=0)), (8 + z.abs()) * EPS * torch.exp(z.clamp(max=0)),
                  "slope")


# A residual branch that begins near zero: z has the digits of xh, relative to
# gamma, and y those of z.
@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((64, 250), 10), ((64, 256), 8), ((3, 700, 64), 8)])
@pytest.mark.parametrize("scale", [1e-3, 1e-4, 1e-6])
def test_elu_under_a_small_gamma(shape, groups, scale):
    x = make(shape, "f32", 21)[0]
    gamma = torch.full((shape[-1],), scale)
    y = S.group_norm(x.cuda(), groups, gamma.cuda(), None, act="elu")
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    mu = v.mean((1, 3), keepdim=True)
    mid = v - mu
    rstd = 1 / torch.sqrt((mid * mid).mean((1, 3), keepdim=True) + 1e-5)
    d_xh = K * (mid.abs() + mid.abs().mean((1, 3), keepdim=True) + mu.abs()) * rstd
    z = (mid * rstd).reshape(shape) * gamma.double()
    want = torch.where(z > 0, z, torch.expm1(z))
    slack = d_xh.reshape(shape) * gamma.double() + 18 * EPS * want.abs()
    assert_within(y, want, slack, f"gamma {scale}")


# The tail of Phi keeps its digits: e^(-z^2/2) has its argument's rounding, z^2 e,
# and the factor beside it is within 8 e with its division and products, 16 more.
@pytest.mark.gpu
@pytest.mark.parametrize("N,L", FORMS)
def test_gelu_keeps_the_digits_of_the_tail(N, L):
    z = torch.cat([torch.linspace(-12, 12, 1007), torch.tensor([0.0] + [1e-3, -1e-3, 1e-20, -1e-20] * 4)])
    y, slope = direct(z, "gelu", N, L)
    z = z.double()
    rel = (32 + z * z) * EPS
    phi = torch.special.erfc(-z / math.sqrt(2)) / 2
    e = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    assert_within(y, (z * phi).expand(y.shape), rel * (z * phi).abs(), "y")
    assert_within(slope, phi + z * e, rel * (phi + z.abs() * e), "slope")

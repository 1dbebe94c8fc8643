"""Group norm where digits or finiteness are easily lost: lanes without channels of
their own.  Bounds in e = 2^-24."""
import pytest
import torch

from seq_helpers import EPS, TYPES, assert_within
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

"""Shapes that take the less usual ways through the sequence operators: groups
wider than a block, one channel a group, more samples than a launch's grid or
than meet in L2, rows that share a warp, slabs with marks.  References in 64 bits
on the GPU; bounds as in the operators' own tests."""
import numpy as np
import pytest
import torch

import test_gpu_gated_scan as G
import test_gpu_group_norm as GN
from seq_helpers import EPS, TYPES, assert_within
from test_gpu_dropout import expected, keep_mask
from zealot_b200 import sequence as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((2, 40, 2100), 7), ((1, 30, 5000), 1),
                                          ((3, 9, 4096), 4096), ((2, 33, 2049), 683),
                                          ((4, 5000), 1), ((3, 1111), 11), ((300, 17), 17),
                                          ((2, 3, 1030), 2), ((1, 4000, 3), 1), ((500, 130, 10), 5)])
def test_norm_widths(shape, groups, t):
    x, dy, gamma, beta = (v.cuda() for v in GN.make(shape, t, 11))
    GN.check(x, dy, groups, gamma, beta, "elu")


@pytest.mark.parametrize("shape,groups,t", [((9, 60000, 64), 8, "f32"), ((40, 30000, 51), 3, "bf16"),
                                            ((70000, 2, 8), 2, "f32"), ((66000, 40), 5, "f16")])
def test_norm_of_many_or_large_samples(shape, groups, t):
    """The sums go over up to 3.6e6 terms: serial runs of up to 1,000 merged by trees,
    so a mean is off by a few sqrt(1000) e of the spread; K as in the operator's
    test covers it."""
    x, dy, gamma, beta = (v.cuda() for v in GN.make(shape, t, 12))
    y, mean, rstd = S.group_norm(x, groups, gamma, beta, act="silu", save=True)
    dx, dgamma, dbeta = S.group_norm_grad(x, dy, groups, gamma, beta, mean, rstd, act="silu")
    n, C = shape[0], shape[-1]
    part = max(1, n // 3)
    dg, db = torch.zeros(C).cuda().double(), torch.zeros(C).cuda().double()
    mag_g, mag_b = dg.clone(), db.clone()
    for i in range(0, n, part):
        v = x[i:i + part].double().reshape(-1, int(np.prod(shape[1:-1])), groups, C // groups)
        w = dy[i:i + part].double().reshape_as(v)
        ga, be = (p.double().view(groups, -1) for p in (gamma, beta))
        mu = v.mean((1, 3), keepdim=True)
        rs = 1 / torch.sqrt((v - mu).square().mean((1, 3), keepdim=True) + 1e-5)
        xh = (v - mu) * rs
        d_xh = GN.K * (xh.abs() + 1 + (mu * rs).abs())
        z = xh * ga + be
        s = 1 / (1 + torch.exp(-z))
        want = (z * s).reshape(x[i:i + part].shape)
        slack = (1.13 * (d_xh * ga.abs() + 3 * EPS * (xh * ga).abs()) + 5 * EPS * z.abs().clamp(min=1))
        assert_within(y[i:i + part], want, slack.reshape(want.shape), "y")
        dz = w * (s + z * s * (1 - s))
        dg += (dz * xh).sum((0, 1)).flatten()
        db += dz.sum((0, 1)).flatten()
        mag_g += (dz * xh).abs().sum((0, 1)).flatten() + (w.abs() * d_xh).sum((0, 1)).flatten()
        mag_b += dz.abs().sum((0, 1)).flatten() + (w.abs() * d_xh).sum((0, 1)).flatten()
        d = dz * ga
        m1, m2 = d.mean((1, 3), keepdim=True), (d * xh).mean((1, 3), keepdim=True)
        want = (rs * (d - m1 - xh * m2)).reshape(x[i:i + part].shape)
        slack = rs * ((w.abs() * ga.abs() + m1.abs() + (xh * m2).abs()) * 10 * EPS +
                      w.abs() * ga.abs() * d_xh * (1 + ga.abs()) + d_xh * m2.abs() +
                      GN.K * (1 + xh.abs()) * w.abs().mean((1, 3), keepdim=True) * 2)
        assert_within(dx[i:i + part], want, slack.reshape(want.shape), "dx")
        del v, w, xh, z, s, dz, d, want, slack
    assert_within(dgamma, dg, GN.K * mag_g + EPS * dg.abs(), "dgamma")
    assert_within(dbeta, db, GN.K * mag_b + EPS * db.abs(), "dbeta")


# rows that share a warp, with marks of their own, in one piece and in slabs
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,D", [(33, 40, 6), (21, 64, 10), (9, 65, 4), (50, 130, 3), (7, 1000, 14),
                                   (300, 70, 1), (1300, 64, 66)])
def test_scan_of_narrow_rows(B, T, D, t):
    kw, dh, dh_last = G.make(B, T, D, t, seed=5, resets=0.05)
    G.check(kw, dh, dh_last, what=f"{B}x{T}x{D} {t}")


# decays beyond the series' range, on some channels and on all
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("resets", [0, 0.05])
@pytest.mark.parametrize("T", [1, 24, 200])
def test_scan_of_fast_decays(T, resets, t):
    kw, dh, dh_last = G.make(4, T, 64, t, seed=6, resets=resets)
    kw["lam"] = kw["lam"].clone()
    kw["lam"][::5] = torch.linspace(-2, 3, 13).cuda()
    G.check(kw, dh, dh_last)
    kw["lam"] = torch.linspace(-1, 2, 64).cuda()
    G.check(kw, dh, dh_last, c=3.0)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D", [1, 2, 9, 15, 16, 17, 27, 63, 65, 129, 200, 255, 513, 1025])
def test_dropout_widths(D, t):
    x = torch.randn(37, D, generator=torch.Generator().manual_seed(D)).to(TYPES[t]).cuda()
    mask = keep_mask(np.arange(37), D, 0.3, 123, 9)
    want, slack = expected(x, mask, 0.3, x)
    assert_within(S.dropout(x, 0.3, 123, stream=9, residual=x), want, slack)


# A constant sample whose (0 - mean) rstd is infinite, which nothing but the
# sample's own positions may show (the statistics are given: fp32 sums of so large
# values overflow).  xh is 0 everywhere, so dgamma is 0 and dbeta the sum of
# dy act'(0).
@pytest.mark.parametrize("L", [1, 3, 301, 5001])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_norm_gradient_of_a_huge_constant(L, act):
    C = 64
    x = torch.full((2, L, C), 2.0 ** 120, device="cuda")
    dy = torch.ones_like(x)
    ones, zeros = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    mean, rstd = torch.full((2, 8), 2.0 ** 120, device="cuda"), torch.full((2, 8), 316.0, device="cuda")
    dx, dgamma, dbeta = S.group_norm_grad(x, dy, 8, ones, zeros, mean, rstd, act=act)
    assert torch.equal(dgamma, zeros)
    slope = 1.0 if act == "none" else 0.5
    assert torch.allclose(dbeta, torch.full_like(dbeta, 2 * L * slope), rtol=1e-6 * (1 + L ** 0.5))
    assert torch.isfinite(dx).all()

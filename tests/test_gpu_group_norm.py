"""zealot_b200.sequence.group_norm and its gradient against 64 bits.

Bounds, with e = 2^-24.  A mean of n terms summed in 32 bits, in serial runs
of at most 64 and trees above them, is off by at most (64 + log2 n) e times
the mean of their magnitudes; with random signs of the roundings a tenth of
that is already several standard deviations, and the bound below takes
K = 40 e.  xh = (x - mu) rstd: off by K (|x - mu| + mean |x - mu| + |mu|) rstd.
z = gamma xh + beta and the activation (slope at most 1.13, its own function
within 4 e of max(1, |z|)) carry that on.  A gradient's sums are bounded the
same way from the magnitudes of their terms.
"""
import math

import pytest
import torch

from seq_helpers import EPS, TYPES, assert_within
from zealot_b200 import native as N
from zealot_b200 import sequence as S

K = 40 * EPS
# [N, ..., C], groups: one element, one channel a group, odd widths, rows,
# positions, more rows than a block, groups wider than a block
SHAPES = [((1, 1), 1), ((3, 8), 8), ((5, 12), 3), ((70, 96), 6), ((33, 250), 10), ((4, 512), 1),
          ((2, 1300), 1), ((300, 64), 4), ((3, 7, 24), 4), ((2, 5, 6, 40), 5), ((1, 700, 48), 6),
          ((2, 333, 17), 17), ((3, 257, 18), 2), ((1, 5000, 8), 2), ((2, 90, 256), 32),
          ((1, 1024, 64), 8), ((2, 4096, 128), 8), ((1, 20000, 96), 4)]


def act64(z, act):
    if act == "elu":
        return torch.where(z > 0, z, torch.expm1(z)), torch.exp(z.clamp(max=0))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def reference(x, groups, gamma, beta, act, eps, dy=None):
    """y, dx, dgamma, dbeta in 64 bits and the slack of each."""
    n, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, C // groups)
    ga = (gamma.double() if gamma is not None else torch.ones(C).double()).view(groups, -1)
    be = (beta.double() if beta is not None else torch.zeros(C).double()).view(groups, -1)
    mu = v.mean((1, 3), keepdim=True)
    mid = v - mu
    rstd = 1 / torch.sqrt((mid * mid).mean((1, 3), keepdim=True) + eps)
    xh = mid * rstd
    d_xh = K * (mid.abs() + mid.abs().mean((1, 3), keepdim=True) + mu.abs()) * rstd
    z = xh * ga + be
    d_z = d_xh * ga.abs() + 2 * EPS * (xh * ga).abs() + EPS * be.abs()
    y, slope = act64(z, act)
    out = {"y": (y, 1.13 * d_z + 4 * EPS * z.abs().clamp(min=1))}
    if dy is not None:
        # slopes of the slopes are at most 1
        w = dy.double().reshape_as(v)
        d_slope = d_z + 6 * EPS * z.abs().clamp(min=1)
        dz, d_dz = w * slope, w.abs() * d_slope
        out["dbeta"] = dz.sum((0, 1)), d_dz.sum((0, 1)) + K * dz.abs().sum((0, 1))
        t = dz * xh
        d_t = d_dz * xh.abs() + dz.abs() * d_xh + 2 * EPS * t.abs()
        out["dgamma"] = t.sum((0, 1)), d_t.sum((0, 1)) + K * t.abs().sum((0, 1))
        d, d_d = dz * ga, d_dz * ga.abs() + EPS * (dz * ga).abs()
        dim = dict(dim=(1, 3), keepdim=True)
        m1, d_m1 = d.mean(**dim), d_d.mean(**dim) + K * d.abs().mean(**dim)
        m2 = (d * xh).mean(**dim)
        d_m2 = (d_d * xh.abs() + d.abs() * d_xh).mean(**dim) + K * (d * xh).abs().mean(**dim)
        dx = rstd * (d - m1 - xh * m2)
        out["dx"] = dx, rstd * (d_d + d_m1 + xh.abs() * d_m2 + d_xh * m2.abs() +
                                8 * EPS * (d.abs() + m1.abs() + (xh * m2).abs()))
    shape = {"y": x.shape, "dx": x.shape, "dgamma": (C,), "dbeta": (C,)}
    return {k: (a.reshape(shape[k]), b.reshape(shape[k])) for k, (a, b) in out.items()}


def make(shape, t, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    C = shape[-1]
    x = torch.randn(shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + torch.randn(C, generator=g)
    return (x.to(TYPES[t]), torch.randn(shape, generator=g).to(TYPES[t]),
            1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g))


def check(x, dy, groups, gamma, beta, act, eps=1e-5, **kw):
    want = reference(x.cpu(), groups, None if gamma is None else gamma.cpu(),
                     None if beta is None else beta.cpu(), act, eps, dy.cpu())
    y, mean, rstd = S.group_norm(x, groups, gamma, beta, act=act, eps=eps, save=True, **kw)
    assert_within(y, *want["y"], "y")
    dx, dgamma, dbeta = S.group_norm_grad(x, dy, groups, gamma, beta, mean, rstd, act=act)
    assert_within(dx, *want["dx"], "dx")
    assert_within(dgamma, *want["dgamma"], "dgamma")
    assert_within(dbeta, *want["dbeta"], "dbeta")
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_sizes(shape, groups, t):
    x, dy, gamma, beta = (v.cuda() for v in make(shape, t))
    check(x, dy, groups, gamma, beta, "elu")


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(S.ACTIVATIONS))
@pytest.mark.parametrize("shape,groups", [((65, 96), 8), ((2, 300, 64), 8), ((3, 50, 21), 3)])
def test_activations(shape, groups, act):
    for t in TYPES:
        x, dy, gamma, beta = (v.cuda() for v in make(shape, t, 1))
        check(x, dy, groups, gamma, beta, act)
        check(x, dy, groups, None, None, act, eps=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((9, 48), 4), ((2, 640, 32), 4)])
def test_an_offset_far_above_the_spread(shape, groups):
    # the mean is 1000 times the spread: centred sums, not x^2 - mean^2
    x, dy, gamma, beta = (v.cuda() for v in make(shape, "f32", 2))
    check(x * 1.0 + 1000.0, dy, groups, gamma, beta, "silu")


@pytest.mark.gpu
def test_a_constant_group_gives_beta():
    x = torch.full((4, 10, 16), 3.0).cuda()
    _, dy, gamma, beta = (v.cuda() for v in make((4, 10, 16), "f32"))
    y, mean, rstd = S.group_norm(x, 4, gamma, beta, act="none", save=True)
    assert torch.equal(y, beta.expand_as(y)) and bool((mean == 3).all())
    dx = S.group_norm_grad(x, dy, 4, gamma, beta, mean, rstd, act="none")[0]
    assert bool(torch.isfinite(dx).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(S.ACTIVATIONS))
def test_gradient_against_differences(act):
    # central differences of sum(w y) in 64 bits at the kernel's inputs
    x, w, gamma, beta = make((3, 6, 20), "f32", 5)
    dev = [v.cuda() for v in (x, w, gamma, beta)]
    _, mean, rstd = S.group_norm(dev[0], 5, dev[2], dev[3], act=act, save=True)
    dx, dgamma, dbeta = S.group_norm_grad(dev[0], dev[1], 5, dev[2], dev[3], mean, rstd, act=act)

    def value(x, gamma, beta):
        return (reference(x, 5, gamma, beta, act, 1e-5)["y"][0] * w.double()).sum().item()

    h = 1e-5
    for name, got, at in (("x", dx, (1, 2, 7)), ("x", dx, (2, 5, 19)), ("gamma", dgamma, (4,)),
                          ("beta", dbeta, (11,))):
        args = {"x": x.double(), "gamma": gamma.double(), "beta": beta.double()}
        up, down = dict(args), dict(args)
        up[name], down[name] = args[name].clone(), args[name].clone()
        up[name][at] += h
        down[name][at] -= h
        diff = (value(**up) - value(**down)) / (2 * h)
        # h^2 of the difference, the roundings of a sum of 360 terms over h, 32 bits
        assert abs(got[at].item() - diff) <= 1e-5 * max(1.0, abs(diff)) + 1e-6, (name, at)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides_offsets_and_in_place(t):
    big, dbig, gamma, beta = (v.cuda() for v in make((4, 50, 80), t, 7))
    for sl in ((slice(None), slice(None, None, 2), slice(0, 48)),
               (slice(1, 3), slice(3, 40), slice(5, 53)), (slice(None), slice(None), slice(8, 56))):
        x, dy = big[sl], dbig[sl]
        y = check(x, dy, 6, gamma[:48].contiguous(), beta[:48].contiguous(), "elu")
        out = torch.zeros_like(big)
        S.group_norm(x, 6, gamma[:48].contiguous(), beta[:48].contiguous(), out=out[sl])
        assert torch.equal(out[sl], y)
        out[sl] = 0
        assert not out.any()
    x = big.clone()
    y = S.group_norm(x, 8, gamma, beta)
    assert S.group_norm(x, 8, gamma, beta, out=x) is x and torch.equal(x, y)
    # rows of an [N, C] view with a stride, as in one time step of a rollout
    check(big[:, 7], dbig[:, 7], 8, gamma, beta, "gelu")
    # another order of the positions
    check(big.view(4, 5, 10, 80).transpose(0, 1)[:, :, 3].contiguous(),
          dbig.view(4, 5, 10, 80).transpose(0, 1)[:, :, 3].contiguous(), 8, gamma, beta, "elu")


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_group():
    for bad in (float("inf"), float("nan")):
        x = torch.randn(4, 9, 32, generator=torch.Generator().manual_seed(1)).cuda()
        clean = S.group_norm(x, 4, act="none")
        x[2, 5, 11] = bad
        y = S.group_norm(x, 4, act="none")
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[2, :, 8:16] = True
        assert torch.equal(y[~hit], clean[~hit]) and bool(torch.isnan(y[hit]).any())


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    x, dy, gamma, beta = (v.cuda() for v in make((700, 96), "bf16", 3))
    a = S.group_norm(x, 6, gamma, beta, save=True)
    ga = S.group_norm_grad(x, dy, 6, gamma, beta, *a[1:])
    for _ in range(3):
        b = S.group_norm(x, 6, gamma, beta, save=True)
        gb = S.group_norm_grad(x, dy, 6, gamma, beta, *b[1:])
        assert all(torch.equal(p, q) for p, q in zip(a + ga, b + gb))


@pytest.mark.gpu
def test_empty():
    e = torch.empty(0, 16).cuda()
    y, mean, rstd = S.group_norm(e, 4, save=True)
    assert y.shape == (0, 16) and mean.shape == (0, 4)
    dx, dgamma, dbeta = S.group_norm_grad(e, e, 4, None, None, mean, rstd)
    assert dx.shape == (0, 16) and not dgamma.any() and not dbeta.any()
    e = torch.empty(3, 0, 16).cuda()
    y, mean, rstd = S.group_norm(e, 4, save=True)
    dgamma = S.group_norm_grad(e, e, 4, None, None, mean, rstd)[1]
    assert y.shape == (3, 0, 16) and dgamma.shape == (16,) and not dgamma.any()


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 16).cuda()
    v = torch.zeros(16).cuda()
    m = torch.zeros(4, 4).cuda()
    for kw in (dict(groups=3), dict(groups=0), dict(groups=4, act="tanh"),
               dict(groups=4, gamma=v[:8]), dict(groups=4, out=x[:3]), dict(groups=4, eps=-1.0),
               dict(groups=4, eps=float("nan"))):
        with pytest.raises(N.ZrlError) as e:
            S.group_norm(x, **kw)
        assert e.value.status == N.INVALID_ARG
    with pytest.raises(TypeError):
        S.group_norm(x.double(), 4)
    with pytest.raises(TypeError):
        S.group_norm(x, 4, gamma=v.half())
    with pytest.raises(N.ZrlError):
        S.group_norm(torch.zeros(16, 4).cuda().t(), 4)
    with pytest.raises(N.ZrlError):
        S.group_norm(torch.zeros(2, 6, 8, 16).cuda()[:, :, ::3], 4)
    with pytest.raises(N.ZrlError):
        S.group_norm_grad(x, x, 4, None, None, m[:3], m)
    with pytest.raises(TypeError):
        S.group_norm_grad(x, x.half(), 4, None, None, m, m)


def test_refusals_without_a_gpu():
    with pytest.raises(TypeError):
        S.group_norm(torch.zeros(4, 16), 4)
    L = N.lib()

    def fwd(n=4, l=1, c=16, groups=4, dtype=0, act=1, eps=1e-5, x=64, y=64):
        return L.zrl_group_norm(x, None, None, n, l, c, groups, dtype, act, eps, None, y, None,
                                None, None, 0, None)

    for kw in (dict(n=-1), dict(l=-2), dict(c=-16), dict(groups=0), dict(groups=3),
               dict(dtype=9), dict(act=4), dict(act=-1), dict(eps=-1e-5),
               dict(eps=float("inf")), dict(x=None), dict(y=None), dict(x=65)):
        assert fwd(**kw) == N.INVALID_ARG, kw
        assert b"group_norm" in L.zrl_last_error(None)
    assert fwd(n=0) == N.OK

    def grad(ws=64, nbytes=1 << 30, mean=64, dx=64, groups=4):
        return L.zrl_group_norm_grad(64, 64, None, None, mean, 64, 4, 1, 16, groups, 0, 1, None,
                                     dx, 64, 64, ws, nbytes, None)

    for kw in (dict(ws=None), dict(nbytes=0), dict(mean=None), dict(dx=None), dict(groups=5)):
        assert grad(**kw) == N.INVALID_ARG, kw

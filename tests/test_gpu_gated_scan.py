"""zealot_b200.sequence.gated_scan, its single step and its gradient against
the recurrence step by step in 64 bits.

Bounds, with e = 2^-24.  The gates: a sigmoid, softplus and exponential within
8 e each, so rate s_r is off by 24 e of itself and a by (1 + 24 rate s_r) e
relative, of which rate s_r <= 1 in nearly all of the inputs here and is
bounded by max(rate); m = sqrt(1 - a^2) by 16 e relative.  A step adds two
roundings.  So the term of step s in h_t is off by at most
(64 + (26 R + 2)(t - s)) e relative, R = max(1, max rate), and h_t by
e times the recurrence of the magnitudes, H_t = a_t H_{t-1} + |b_t|, with the
extra weight (26 R + 2) per step carried along.  The test carries exactly that
second recurrence.  The gradients are bounded from theirs in the same way.
"""
import pytest
import torch

from seq_helpers import EPS, TYPES, assert_within
from zealot_b200 import native as N
from zealot_b200 import sequence as S

C8 = 8.0


def reference(x, rec, inp, lam, h0=None, resets=None, c=C8, dh=None, dh_last=None):
    """Everything in 64 bits on the CPU: {name: (value, slack)}."""
    x, rec, inp, lam = (v.detach().cpu().double() for v in (x, rec, inp, lam))
    B, T, D = x.shape
    z = torch.zeros(B, T, 1, dtype=torch.bool) if resets is None else resets.cpu().reshape(B, T, 1) != 0
    rate = c * torch.nn.functional.softplus(lam, threshold=1e9)
    sr, si = 1 / (1 + torch.exp(-rec)), 1 / (1 + torch.exp(-inp))
    a = torch.exp(-rate * sr)
    m = torch.sqrt(-torch.expm1(-2 * rate * sr))
    a, m = a.masked_fill(z, 0), m.masked_fill(z, 1)
    per = (26 * max(1.0, rate.max().item()) + 2) if D else 0.0
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.cpu().double()
    H, E = h.abs(), torch.zeros_like(h)
    hs, Hs, Es = [h], [H], [E]
    for t in range(T):
        b = m[:, t] * si[:, t] * x[:, t]
        h = torch.where(z[:, t], b, a[:, t] * h + b)
        E = torch.where(z[:, t], 0.0, a[:, t] * (E + per * H)) + 64 * b.abs()
        H = torch.where(z[:, t], 0.0, a[:, t] * H) + b.abs()
        hs.append(h), Hs.append(H), Es.append(E)
    hs, Hs, Es = (torch.stack(v, 1) for v in (hs, Hs, Es))
    out = {"h": (hs[:, 1:], EPS * Es[:, 1:]), "h_last": (h, EPS * E)}
    if dh is None:
        return out
    dh = dh.detach().cpu().double()
    g = torch.zeros(B, D, dtype=torch.float64) if dh_last is None else dh_last.cpu().double()
    G, F = g.abs(), torch.zeros_like(g)
    gs, Gs, Fs = [], [], []
    for t in range(T - 1, -1, -1):
        g, F, G = g + dh[:, t], F + 2 * (G + dh[:, t].abs()), G + dh[:, t].abs()
        gs.append(g), Gs.append(G), Fs.append(F)
        F, g, G = a[:, t] * (F + per * G), a[:, t] * g, a[:, t] * G
    dh0 = (g, EPS * F)
    gs, Gs, Fs = (torch.stack(v[::-1], 1) if v else torch.zeros(B, 0, D, dtype=torch.float64)
                  for v in (gs, Gs, Fs))
    b4, H4, E4 = hs[:, :-1], Hs[:, :-1], Es[:, :-1]
    inner = torch.where(z | (m == 0), torch.zeros_like(a), si * x * a * a / m)
    keep = torch.where(z, torch.zeros_like(a), torch.ones_like(a))
    b4, H4, E4 = (torch.where(z, torch.zeros_like(v), v) for v in (b4, H4, E4))
    q = gs * (b4 * a - inner) * keep
    mag = Gs * (H4 * a + inner.abs()) * keep
    d_q = (Fs * (H4 * a + inner.abs()) + Gs * a * E4) * keep + (64 + 2 * per) * mag
    out["dx"] = gs * m * si, EPS * (Fs + 64 * Gs) * m * si
    out["dinp"] = (gs * m * x * si * (1 - si),
                   EPS * (Fs + 64 * Gs) * m * x.abs() * si)
    w = rate * sr * (1 - sr)
    # 1 - s_r is within 2 e of itself or of s_r's rounding, 8 e
    out["drec"] = -w * q, EPS * (w * (d_q + 64 * mag) + 8 * rate * sr * mag)
    k = c * torch.sigmoid(lam)
    total = (sr * q).sum((0, 1))
    n_sum = 40 + 2 * (B * T) ** 0.5
    out["dlam"] = -k * total, EPS * k * (sr * d_q).sum((0, 1)) + EPS * k * n_sum * (sr * mag).sum((0, 1))
    out["dh0"] = dh0
    return out


def make(B, T, D, t, seed=0, resets=0.1, h0=True):
    g = torch.Generator().manual_seed(seed + B + 31 * T + 977 * D)
    x, rec, inp, dh = (torch.randn(B, T, D, generator=g).to(TYPES[t]).cuda() for _ in range(4))
    a = 0.9 + 0.099 * torch.rand(D, generator=g, dtype=torch.float64)
    lam = torch.log(torch.expm1(-torch.log(a) / C8)).float().cuda()
    z = (torch.rand(B, T, generator=g) < resets).to(torch.uint8).cuda() if resets else None
    return dict(x=x, rec=rec, inp=inp, lam=lam, h0=torch.randn(B, D, generator=g).cuda() if h0 else None,
                resets=z), dh, torch.randn(B, D, generator=g).cuda()


def check(kw, dh=None, dh_last=None, c=C8, what=""):
    want = reference(**kw, c=c, dh=dh, dh_last=dh_last)
    h, last, carry = S.gated_scan(**kw, c=c, save=True)
    assert_within(h, *want["h"], what + " h")
    assert_within(last, *want["h_last"], what + " h_last")
    if dh is None:
        return h
    d = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry, dh_last=dh_last,
                          h0=kw["h0"], resets=kw["resets"], c=c)
    for name, got in zip(("dx", "drec", "dinp", "dlam", "dh0"), d):
        if got is None:
            assert kw["h0"] is None
            continue
        assert_within(got, *want[name], f"{what} {name}")
    return h


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (1, 1, 256), (3, 2, 7), (2, 16, 64), (5, 17, 33),
                                   (4, 24, 128), (70, 24, 65), (2, 127, 40), (2, 128, 40),
                                   (3, 129, 30), (1, 300, 96), (9, 65, 66), (1, 1030, 17),
                                   (2, 2100, 8)])
def test_sizes(B, T, D, t):
    kw, dh, dh_last = make(B, T, D, t, resets=0.05)
    check(kw, dh, dh_last, what=f"{B}x{T}x{D} {t}")
    kw, dh, _ = make(B, T, D, t, seed=1, resets=0, h0=False)
    check(kw, dh, None, what=f"{B}x{T}x{D} {t} bare")


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,D", [(1, 9000, 64), (2, 4097, 24), (40, 520, 512)])
def test_long_rows(B, T, D, t):
    kw, dh, dh_last = make(B, T, D, t, resets=0.002)
    check(kw, dh, dh_last, what=f"{B}x{T}x{D} {t}")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["time", "fused", "offset", "expanded"])
@pytest.mark.parametrize("t", list(TYPES))
def test_layouts(layout, t):
    B, T, D = 6, 150, 48
    kw, dh, dh_last = make(B, T, D, t)
    plain = check(kw, dh, dh_last)
    if layout == "time":
        for k in ("x", "rec", "inp"):
            kw[k] = kw[k].transpose(0, 1).contiguous().transpose(0, 1)
        kw["resets"] = kw["resets"].t().contiguous().t()
        dh = dh.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "fused":
        kw["x"], kw["rec"], kw["inp"] = torch.cat([kw["x"], kw["rec"], kw["inp"]], -1).split(D, -1)
    elif layout == "offset":
        for k in ("x", "rec", "inp"):
            big = torch.zeros(B, T + 2, D + 5, dtype=kw[k].dtype, device="cuda")
            big[:, 1:-1, 3:-2] = kw[k]
            kw[k] = big[:, 1:-1, 3:-2]
    else:
        kw["inp"] = kw["inp"][:, :1].expand(B, T, D)
        kw["resets"] = kw["resets"][:1].expand(B, T)
        check(kw, dh, dh_last)
        return
    assert torch.equal(check(kw, dh, dh_last), plain)
    out = torch.zeros(B, T, 3 * D, dtype=TYPES[t], device="cuda").split(D, -1)
    carry = S.gated_scan(**kw, save=True)[2]
    args = (kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry)
    more = dict(dh_last=dh_last, h0=kw["h0"], resets=kw["resets"])
    want = S.gated_scan_grad(*args, **more)
    S.gated_scan_grad(*args, **more, out=out)
    assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_steps_follow_the_scan(t):
    kw, _, _ = make(5, 40, 96, t)
    want = reference(**kw)
    state, place = kw["h0"], kw["h0"].clone()
    for i in range(40):
        z = kw["resets"][:, i]
        x, rec, inp = (kw[k][:, i] for k in ("x", "rec", "inp"))
        h, state = S.gated_step(x, rec, inp, kw["lam"], state, resets=z)
        h2, same = S.gated_step(x.contiguous(), rec, inp, kw["lam"], place, resets=z, out=place)
        assert same is place and torch.equal(h, h2) and torch.equal(state, place)
        assert_within(h, want["h"][0][:, i], want["h"][1][:, i], f"step {i}")
        assert torch.equal(h, state.to(h.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [24, 200])
def test_every_step_an_episode(T):
    kw, dh, dh_last = make(3, T, 40, "f32")
    kw["resets"] = torch.ones(3, T, dtype=torch.bool, device="cuda")
    h = check(kw, dh, dh_last)
    want = torch.sigmoid(kw["inp"].double()) * kw["x"].double()
    assert torch.allclose(h.double(), want, rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_rows_laid_end_to_end_equal_rows_apart():
    # three recordings of different lengths in one row, marked where they begin
    n = [37, 150, 1]
    kw, dh, _ = make(1, sum(n), 64, "f32", resets=0, h0=False)
    kw["resets"] = torch.zeros(1, sum(n), dtype=torch.uint8, device="cuda")
    at = [0, 37, 187]
    kw["resets"][0, at] = 255
    h, _, carry = S.gated_scan(**kw, save=True)
    dx = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry,
                           resets=kw["resets"])[0]
    for a, k in zip(at, n):
        part = {s: (v[:, a:a + k].contiguous() if s in ("x", "rec", "inp", "resets") else v)
                for s, v in kw.items()}
        h2, _, c2 = S.gated_scan(**part, save=True)
        d2 = S.gated_scan_grad(part["x"], part["rec"], part["inp"], kw["lam"],
                               dh[:, a:a + k].contiguous(), c2, resets=part["resets"])[0]
        torch.testing.assert_close(h[:, a:a + k], h2, rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(dx[:, a:a + k], d2, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("T,at", [(24, 9), (24, 16), (300, 128), (300, 200), (2500, 1900)])
def test_nothing_of_the_state_before_an_episode_is_used(bad, T, at):
    kw, dh, dh_last = make(2, T, 40, "f32", resets=0)
    kw["resets"] = torch.zeros(2, T, dtype=torch.uint8, device="cuda")
    kw["resets"][:, at] = 1
    h, last, carry = S.gated_scan(**kw, save=True)
    grad = dict(dh_last=dh_last, h0=kw["h0"], resets=kw["resets"])
    d = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry, **grad)
    kw["x"] = kw["x"].clone()
    kw["x"][0, at - 1, :] = bad
    h2, last2, carry2 = S.gated_scan(**kw, save=True)
    assert torch.equal(h2[:, at:], h[:, at:]) and torch.equal(last2, last)
    assert torch.equal(h2[1], h[1]) and not torch.isfinite(h2[0, at - 1]).any()
    d2 = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry2, **grad)
    for p, q in zip(d[:3], d2[:3]):
        assert torch.equal(p[:, at:], q[:, at:]) and torch.equal(p[1], q[1])
    # and nothing of a gradient behind the episode's end reaches before it
    dh2 = dh.clone()
    dh2[0, at:] = bad
    d3 = S.gated_scan_grad(kw["x"].nan_to_num(posinf=1.0), kw["rec"], kw["inp"], kw["lam"], dh2,
                           S.gated_scan(**{**kw, "x": kw["x"].nan_to_num(posinf=1.0)}, save=True)[2],
                           **grad)
    assert torch.isfinite(d3[0][:, :at]).all() and torch.isfinite(d3[4]).all()


@pytest.mark.gpu
def test_saturated_gates():
    # gates so far open or shut that a is 0 or 1 in 32 bits
    kw, dh, dh_last = make(2, 40, 64, "f32", resets=0)
    kw["rec"] = kw["rec"].clone()
    kw["rec"][..., ::4] = -200.0
    kw["rec"][..., 1::4] = 60.0
    kw["inp"] = kw["inp"].clone()
    kw["inp"][..., 2::4] = -200.0
    kw["lam"] = kw["lam"].clone()
    kw["lam"][1::4] = 40.0
    h, last, carry = S.gated_scan(**kw, save=True)
    d = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry, dh_last=dh_last,
                          h0=kw["h0"])
    assert all(bool(torch.isfinite(v).all()) for v in (h, last) + d)
    # shut: the state stays; wide open: it is replaced
    assert torch.equal(h[..., ::4], kw["h0"][:, None, ::4].expand(2, 40, 16))
    want = (torch.sigmoid(kw["inp"]) * kw["x"])[..., 1::4]
    torch.testing.assert_close(h[..., 1::4], want, rtol=1e-6, atol=1e-7)


@pytest.mark.gpu
def test_gradient_against_differences():
    B, T, D = 2, 150, 5
    kw, dh, dh_last = make(B, T, D, "f32", resets=0.02)
    carry = S.gated_scan(**kw, save=True)[2]
    d = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry, dh_last=dh_last,
                          h0=kw["h0"], resets=kw["resets"])
    got = dict(zip(("x", "rec", "inp", "lam", "h0"), d))

    def value(**k):
        r = reference(**k)
        return ((r["h"][0] * dh.cpu().double()).sum() +
                (r["h_last"][0] * dh_last.cpu().double()).sum()).item()

    base = {k: (v.cpu().double() if k != "resets" else v.cpu()) for k, v in kw.items()}
    for name, at in (("x", (0, 0, 1)), ("x", (1, 149, 4)), ("rec", (0, 60, 2)), ("rec", (1, 128, 0)),
                     ("inp", (0, 127, 3)), ("inp", (1, 5, 1)), ("lam", (2,)), ("lam", (4,)),
                     ("h0", (1, 3))):
        up, down, e = dict(base), dict(base), 1e-5
        up[name], down[name] = base[name].clone(), base[name].clone()
        up[name][at] += e
        down[name][at] -= e
        diff = (value(**up) - value(**down)) / (2 * e)
        assert abs(got[name][at].item() - diff) <= 2e-5 * max(1.0, abs(diff)), (name, at)


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    kw, dh, dh_last = make(3, 700, 130, "bf16")
    a = S.gated_scan(**kw, save=True)
    g = dict(dh_last=dh_last, h0=kw["h0"], resets=kw["resets"])
    da = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, a[2], **g)
    for _ in range(3):
        b = S.gated_scan(**kw, save=True)
        db = S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, b[2], **g)
        assert all(torch.equal(p, q) for p, q in zip(a + da, b + db))


@pytest.mark.gpu
def test_empty():
    for shape in ((0, 5, 8), (3, 0, 8), (3, 5, 0)):
        B, T, D = shape
        e = torch.empty(shape).cuda()
        lam = torch.zeros(D).cuda()
        h0 = torch.randn(B, D).cuda()
        h, last, carry = S.gated_scan(e, e, e, lam, h0=h0, save=True)
        assert h.shape == shape and last.shape == (B, D)
        if T == 0:
            assert torch.equal(last, h0)
        d = S.gated_scan_grad(e, e, e, lam, e, carry, dh_last=h0, h0=h0)
        assert d[0].shape == shape and d[3].shape == (D,) and not d[3].any()
        if T == 0:
            assert torch.equal(d[4], h0)


@pytest.mark.gpu
def test_a_cuda_graph_and_another_stream():
    kw, dh, dh_last = make(4, 300, 64, "f32")

    def both():
        h, last, carry = S.gated_scan(**kw, save=True)
        return (h, last) + S.gated_scan_grad(kw["x"], kw["rec"], kw["inp"], kw["lam"], dh, carry,
                                             dh_last=dh_last, h0=kw["h0"], resets=kw["resets"])

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    kw["x"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, both()))


@pytest.mark.gpu
def test_refusals():
    kw, dh, _ = make(2, 200, 16, "f32")
    x, lam = kw["x"], kw["lam"]
    carry = S.gated_scan(**kw, save=True)[2]

    def bad(error, fn, *args, **k):
        with pytest.raises(error) as e:
            fn(*args, **k)
        if error is N.ZrlError:
            assert e.value.status == N.INVALID_ARG

    bad(TypeError, S.gated_scan, x.double(), x.double(), x.double(), lam)
    bad(TypeError, S.gated_scan, x, x.half(), x, lam)
    bad(TypeError, S.gated_scan, x, x, x, lam.half())
    bad(TypeError, S.gated_scan, x, x, x, lam, resets=torch.zeros(2, 200).cuda())
    bad(TypeError, S.gated_scan, x, x, x, lam, h0=torch.zeros(2, 16))
    bad(N.ZrlError, S.gated_scan, x[0], x[0], x[0], lam)
    bad(N.ZrlError, S.gated_scan, x, x[:, :5], x, lam)
    bad(N.ZrlError, S.gated_scan, x, x, x, lam[:8])
    bad(N.ZrlError, S.gated_scan, x, x, x, lam, resets=kw["resets"][:, :9])
    bad(N.ZrlError, S.gated_scan, x, x, x, lam, c=0.0)
    bad(N.ZrlError, S.gated_scan, x, x, x, lam, c=float("nan"))
    wide = torch.zeros(2, 200, 32).cuda()[..., ::2]
    bad(N.ZrlError, S.gated_scan, wide, x, x, lam)
    bad(N.ZrlError, S.gated_scan_grad, x, x, x, lam, dh, None)
    bad(N.ZrlError, S.gated_scan_grad, x, x, x, lam, dh, carry[:, :0])
    bad(N.ZrlError, S.gated_scan_grad, x, x, x, lam, dh[:, 1:], carry)
    bad(ValueError, S.gated_scan_grad, x, x, x, lam, dh, carry, out=(x, x))
    bad(N.ZrlError, S.gated_step, x, x, x, lam, kw["h0"])
    bad(N.ZrlError, S.gated_step, x[:, 0], x[:, 0], x[:, 0], lam, None)


def test_refusals_without_a_gpu():
    with pytest.raises(TypeError):
        S.gated_scan(*[torch.zeros(2, 3, 4)] * 3, torch.zeros(4))
    L = N.lib()

    def fwd(b=2, t=3, d=4, dtype=0, c=8.0, x=64, lam=64, h=64):
        return L.zrl_gated_scan(x, 64, 64, lam, None, None, b, t, d, dtype, c, None, h, None,
                                None, None, 0, None)

    for kw in (dict(b=-1), dict(t=-1), dict(d=-1), dict(dtype=3), dict(c=0.0), dict(c=-1.0),
               dict(c=float("inf")), dict(x=None), dict(lam=None), dict(h=None), dict(x=66)):
        assert fwd(**kw) == N.INVALID_ARG, kw
        assert b"gated_scan" in L.zrl_last_error(None)
    assert fwd(b=0) == N.OK and fwd(d=0) == N.OK

    def grad(t=3, carry=None, ws=64, nbytes=1 << 30, dlam=64, dx=64):
        return L.zrl_gated_scan_grad(64, 64, 64, 64, None, None, carry, 64, None, 2, t, 4, 0, 8.0,
                                     None, dx, 64, 64, dlam, None, ws, nbytes, None)

    for kw in (dict(t=65), dict(ws=None), dict(nbytes=0), dict(dlam=None), dict(dx=None)):
        assert grad(**kw) == N.INVALID_ARG, kw
    assert L.zrl_gated_scan_carry(2, 8, 4) == 0
    assert L.zrl_gated_scan_carry(2, 9, 4) == 8
    assert L.zrl_gated_scan_carry(2, 17, 4) == 16

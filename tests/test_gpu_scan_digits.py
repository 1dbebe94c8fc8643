"""Where the gated scan's digits go: gates nearly shut, and sums over a long row."""
import pytest
import torch

import test_gpu_gated_scan as G
from seq_helpers import EPS, TYPES, assert_within
from zealot_b200 import sequence as S

pytestmark = pytest.mark.gpu
INF = float("inf")


# The bounds of the operator's own tests are relative to each step's input
# sqrt(1 - a^2) sigmoid(inp) x, so a gate that is nearly shut has to be as exact as
# an open one; from a state of zero nothing larger hides it.
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 5, 24, 200])
@pytest.mark.parametrize("gate", ["inp", "rec"])
def test_gates_nearly_shut(gate, T, t):
    D = 176
    kw, dh, dh_last = G.make(3, T, D, t, seed=9, resets=0, h0=False)
    at = torch.cat([torch.linspace(-72, 72, D - 16), torch.tensor([-INF, INF, -45.0, -41.6, 0.0, -60.0, -70.0, 40.0] * 2)])
    kw[gate] = at.to(TYPES[t]).cuda().expand(3, T, D).contiguous()
    G.check(kw, dh, dh_last, what=gate)
    # every state of its own: a step's input alone
    kw["resets"] = torch.ones(3, T, dtype=torch.uint8, device="cuda")
    G.check(kw, dh, dh_last, what=gate + " apart")


@pytest.mark.parametrize("T", [1, 24, 200])
def test_a_shut_gate_lets_nothing_in(T):
    kw, dh, dh_last = G.make(2, T, 64, "f32", resets=0, h0=False)
    for gate in ("inp", "rec"):
        k = dict(kw)
        k[gate] = torch.full_like(kw[gate], -INF)
        h, last, carry = S.gated_scan(**k, save=True)
        assert not h.any() and not last.any()
        dx, drec, dinp, dlam, _ = S.gated_scan_grad(k["x"], k["rec"], k["inp"], k["lam"], dh, carry,
                                                    dh_last=dh_last)
        assert not dx.any() and not dinp.any()
        if gate == "rec":
            assert not drec.any() and not dlam.any()


# dlam of a long row that one thread sums: as many rows as keep rows in one piece,
# all alike, so that every term has the same value and a single running sum errs to
# one side by up to T / 2 roundings.  Sums of 256 terms, then of those, and of the
# rows: 256 + T / 256 + 60 roundings, on top of the terms' own bound.
def test_dlam_of_a_long_row_in_one_piece():
    B, T, D = 592, 32768, 64
    g = torch.Generator().manual_seed(4)
    row = {k: torch.randn(D, generator=g) for k in ("x", "rec", "inp", "dh")}
    row["x"], row["dh"] = 1 + row["x"].abs(), 1 + row["dh"].abs()
    lam = torch.log(torch.expm1(0.17 + 0.1 * torch.rand(D, generator=g)))
    want, slack = G.reference(*(row[k].expand(1, T, D) for k in ("x", "rec", "inp")), lam,
                              dh=row["dh"].expand(1, T, D))["dlam"]
    x, rec, inp, dh = (row[k].cuda().expand(B, T, D) for k in ("x", "rec", "inp", "dh"))
    carry = S.gated_scan(x, rec, inp, lam.cuda(), save=True)[2]
    dlam = S.gated_scan_grad(x, rec, inp, lam.cuda(), dh, carry)[3]
    assert_within(dlam, B * want, B * (slack + (256 + T / 256 + 60) * EPS * want.abs()), "dlam")


# A row in one piece through hundreds of stretches, the last one short.
@pytest.mark.parametrize("t,B,T,D", [("f32", 592, 1001, 64), ("bf16", 1300, 1003, 66)])
def test_long_rows_in_one_piece(t, B, T, D):
    kw, dh, dh_last = G.make(B, T, D, t, seed=8, resets=0.005)
    G.check(kw, dh, dh_last, what=f"{B}x{T}x{D} {t}")


# A memory of up to some thousand steps.  A step rounds a and h, each by 1.7e-8 at
# the root mean square, to either side: over the n / 2 steps that an error lives on,
# 1.6e-7 of h over these decays.  The gates' and rate's roundings, one sided for a
# channel, come to about 4e-7.  A decay whose rounding has a side would add n / 2
# times it, several times the bound.
@pytest.mark.parametrize("B", [1, 300])
def test_a_long_memory_keeps_its_digits(B):
    T, D = 20000, 256
    kw, dh, dh_last = G.make(1, T, D, "f32", seed=2, resets=0, h0=True)
    x, rec, inp = (kw[k][0].cpu().double() for k in ("x", "rec", "inp"))
    rate = 8.0 * torch.nn.functional.softplus(kw["lam"].cpu().double(), threshold=1e9)
    sr, si = torch.sigmoid(rec), torch.sigmoid(inp)
    a, m = torch.exp(-rate * sr), torch.sqrt(-torch.expm1(-2 * rate * sr))
    s, h = kw["h0"][0].cpu().double(), torch.empty(T, D, dtype=torch.float64)
    b = m * si * x
    for i in range(T):
        s = a[i] * s + b[i]
        h[i] = s
    e, g = dh_last[0].cpu().double(), torch.empty(T, D, dtype=torch.float64)
    d = dh[0].cpu().double()
    for i in range(T - 1, -1, -1):
        e = e + d[i]
        g[i] = e
        e = a[i] * e
    # B rows alike: in slabs, and in one piece
    wide = {k: v if k == "lam" or v is None else v.expand(B, *v.shape[1:]) for k, v in kw.items()}
    wide["h0"] = wide["h0"].contiguous()
    got, last, carry = S.gated_scan(**wide, save=True)
    dx = S.gated_scan_grad(wide["x"], wide["rec"], wide["inp"], wide["lam"],
                           dh.expand(B, T, D), carry, dh_last=dh_last.expand(B, D).contiguous(),
                           h0=wide["h0"])[0]
    for v, want, bound in ((got, h, 6e-7), (last, s, 6e-7), (dx, g * m * si, 8e-7)):
        off = (v[-1].cpu().double() - want).norm() / want.norm()
        assert off <= bound, (v.shape, off.item())

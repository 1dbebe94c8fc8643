"""Shared by the tests of the sequence operators: element types, and the
error that rounding a result once to an element type may add."""
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# half a unit in the last place, relative; and the smallest step (subnormals)
ROUND = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
EPS = 2.0 ** -24  # one rounding in 32 bits


def assert_within(got, want, slack, what=""):
    """|got - want| <= slack + one rounding of want to got's type, element by
    element.  want and slack are 64-bit; infinities and NaN have to agree."""
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    slack = torch.as_tensor(slack, dtype=torch.float64).detach().cpu()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    fine = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), f"{what}: NaN in other places"
    inf = torch.isinf(w)
    assert torch.equal(g[inf], w[inf]), f"{what}: infinities differ"
    tol = slack.expand_as(w)[fine] * (1 + ROUND[got.dtype]) + ROUND[got.dtype] * w[fine].abs() + TINY[got.dtype]
    off = (g[fine] - w[fine]).abs()
    if off.numel():
        worst = (off / tol).max()
        assert worst <= 1, f"{what}: {worst.item():.3g} times the bound"

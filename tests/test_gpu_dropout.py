"""zealot_b200.sequence.dropout against its definition in numpy's unsigned
integers and 64-bit floats: the mask bit for bit, the values to two 32-bit
roundings and the rounding of the result."""
import numpy as np
import pytest
import torch

from seq_helpers import EPS, TYPES, assert_within
from zealot_b200 import native as N
from zealot_b200 import sequence as S


def philox(counter, key):
    """Philox4x32-10 in 64-bit unsigned integers: counter 4 x [...], key 2."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    lo, m32 = np.uint64(32), np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> lo) ^ c[1] ^ np.uint64(k[0]), q & m32,
             (p >> lo) ^ c[3] ^ np.uint64(k[1]), p & m32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def keep_mask(rows, D, p, seed, stream):
    rows = np.asarray(rows, np.int64).astype(np.uint64)
    col = np.arange((D + 7) // 8, dtype=np.uint64)
    z = np.zeros((len(rows), len(col)), np.uint64)
    w = philox((z + col, z + (rows & np.uint64(0xFFFFFFFF))[:, None],
                z + (rows >> np.uint64(32))[:, None], z + np.uint64(stream)),
               (seed % 2 ** 32, seed >> 32))
    lanes = np.stack([h for v in w for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], -1)
    return lanes.reshape(len(rows), -1)[:, :D] >= round(65536 * p)


def expected(x, mask, p, residual=None):
    drop = round(65536 * p)
    y = torch.where(torch.from_numpy(mask), x.double().cpu() * (65536 / max(1, 65536 - drop)),
                    torch.zeros((), dtype=torch.float64))
    size = y.abs()
    if residual is not None:
        y = y + residual.double().cpu()
        size = size + residual.double().cpu().abs()
    return y, 3 * EPS * size


def test_philox_restatement_meets_the_published_vectors():
    # the known-answer vectors of the generator's authors (counter and key all
    # zeros, all ones)
    z = philox((0, 0, 0, 0), (0, 0))
    assert [int(v) for v in z] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    o = philox([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(v) for v in o] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_refusals_without_a_gpu():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError):
        S.dropout(x, 0.1, 1)
    L = N.lib()
    for args in ((-1, 8, 0, 0.1), (4, -8, 0, 0.1), (4, 8, 3, 0.1), (4, 8, 0, -0.1),
                 (4, 8, 0, 1.5), (4, 8, 0, float("nan")), (4, 1 << 40, 0, 0.1)):
        n, d, dt, p = args
        assert L.zrl_dropout(64, None, None, n, d, dt, p, 1, 0, None, 64, None) == N.INVALID_ARG
        assert b"dropout" in L.zrl_last_error(None)
    assert L.zrl_dropout(None, None, None, 4, 8, 0, 0.1, 1, 0, None, 64, None) == N.INVALID_ARG
    assert L.zrl_dropout(66, None, None, 4, 8, 0, 0.1, 1, 0, None, 64, None) == N.INVALID_ARG
    assert b"aligned" in L.zrl_last_error(None)
    # nothing to do: no pointer is needed
    assert L.zrl_dropout(None, None, None, 0, 8, 0, 0.1, 1, 0, None, None, None) == N.OK


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape,p", [((1, 1), 0.5), ((3, 7), 0.25), ((5, 8), 0.1), ((64, 16), 0.5),
                                     ((17, 96), 0.1), ((9, 333), 0.25), ((33, 257), 0.0),
                                     ((4, 6, 40), 0.9), ((130, 512), 0.1), ((7, 1000), 1.0)])
def test_mask_and_values(shape, p, t):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g).to(TYPES[t]).cuda()
    r = torch.randn(shape, generator=g).to(TYPES[t]).cuda()
    seed, stream = 0xFEDCBA9876543210, 0xFFFFFFFF
    n = x.numel() // shape[-1]
    mask = keep_mask(np.arange(n), shape[-1], p, seed, stream).reshape(shape)
    for res in (None, r):
        y = S.dropout(x, p, seed, stream=stream, residual=res)
        want, slack = expected(x, mask, p, res)
        assert_within(y, want, slack, f"{shape} {t} residual={res is not None}")
    # the gradient: a sum over y weighted with w has slope w * mask / P(keep) at x
    dx = S.dropout_grad(r, p, seed, stream=stream)
    assert_within(dx, *expected(r, mask, p))


@pytest.mark.gpu
def test_gradient_against_differences():
    # dropout is linear in x: f(x + e) - f(x) = f(e) for a step along any column
    x = torch.randn(6, 37, generator=torch.Generator().manual_seed(3)).cuda()
    w = torch.randn(6, 37, generator=torch.Generator().manual_seed(4)).cuda()
    dx = S.dropout_grad(w, 0.25, 9)
    step = 2.0 ** -3
    for r, c in ((0, 0), (2, 8), (5, 36), (3, 17)):
        e = x.clone()
        e[r, c] += step
        diff = ((S.dropout(e, 0.25, 9) - S.dropout(x, 0.25, 9)).double() * w.double()).sum() / step
        assert abs(diff.item() - dx[r, c].item()) <= 1e-5 * max(1, abs(dx[r, c].item()))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [48, 45])
def test_row_numbers_beyond_32_bits_in_any_order(D):
    rows = torch.tensor([5, 2 ** 32 + 5, 2 ** 40, 0, 2 ** 62 + 1, 5], dtype=torch.int64)
    x = torch.ones(6, D).cuda()
    y = S.dropout(x, 0.5, 77, stream=2, rows=rows.cuda()).cpu()
    mask = keep_mask(rows.numpy(), D, 0.5, 77, 2)
    assert np.array_equal(y.numpy() != 0, mask)
    assert torch.equal(y[0], y[5]) and not torch.equal(y[0], y[1])


@pytest.mark.gpu
def test_strided_rows_and_in_place():
    big = torch.randn(12, 100, generator=torch.Generator().manual_seed(1)).cuda()
    for lo, D in ((0, 64), (3, 64), (8, 41)):
        x = big[::2, lo:lo + D]
        mask = keep_mask(np.arange(6), D, 0.3, 5, 0)
        want, slack = expected(x, mask, 0.3)
        assert_within(S.dropout(x, 0.3, 5), want, slack)
        out = torch.zeros(12, 100).cuda()
        S.dropout(x, 0.3, 5, out=out[1::2, lo:lo + D])
        assert_within(out[1::2, lo:lo + D], want, slack)
        out[1::2, lo:lo + D] = 0
        assert not out.any()  # nothing outside
        y = x.clone()
        assert S.dropout(y, 0.3, 5, out=y) is y
        assert_within(y, want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 33])
def test_dropped_infinities_and_nan_are_not_used(D):
    mask = keep_mask(np.arange(8), D, 0.5, 11, 0)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.full((8, D), bad).cuda()
        y = S.dropout(x, 0.5, 11).cpu()
        assert np.array_equal((y == 0).numpy(), ~mask)
        kept = y[torch.from_numpy(mask)]
        assert torch.isnan(kept).all() if bad != bad else bool((kept == bad).all())


@pytest.mark.gpu
def test_empty_and_another_stream():
    assert S.dropout(torch.empty(0, 16).cuda(), 0.1, 1).shape == (0, 16)
    assert S.dropout(torch.empty(3, 0).cuda(), 0.1, 1).shape == (3, 0)
    side = torch.cuda.Stream()
    x = torch.randn(256, 512).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = S.dropout(x, 0.1, 1)
    side.synchronize()
    assert torch.equal(y, S.dropout(x, 0.1, 1))


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 8).cuda()
    with pytest.raises(TypeError):
        S.dropout(x.double(), 0.1, 1)
    with pytest.raises(TypeError):
        S.dropout(x, 0.1, 1, rows=torch.zeros(4, dtype=torch.int32).cuda())
    with pytest.raises(TypeError):
        S.dropout(x, 0.1, 1, residual=x.half())
    for kw in (dict(rows=torch.zeros(3, dtype=torch.int64).cuda()), dict(residual=x[:3]),
               dict(stream=1 << 32), dict(stream=-1), dict(out=x[:, :4])):
        with pytest.raises(N.ZrlError) as e:
            S.dropout(x, 0.1, 1, **kw)
        assert e.value.status == N.INVALID_ARG
    for p in (-0.5, 2.0, float("nan")):
        with pytest.raises(N.ZrlError):
            S.dropout(x, p, 1)
    with pytest.raises(N.ZrlError):
        S.dropout(x, 0.1, 1 << 64)
    with pytest.raises(N.ZrlError):
        S.dropout(x.t(), 0.1, 1)  # the last axis is not dense
    with pytest.raises(N.ZrlError):
        S.dropout(torch.zeros(2, 6, 8).cuda()[:, ::4].transpose(0, 1), 0.1, 1)

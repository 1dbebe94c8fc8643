"""The sequence operators on views whose offsets pass 32 bits, on broadcast
(stride 0) inputs, and the strides they refuse."""
import ctypes as C

import pytest
import torch

from zealot_b200 import native as N
from zealot_b200 import sequence as S

FAR = (1 << 32) + 64  # elements


def far_view(shape, stride, t, seed):
    """A view of a large buffer with the given strides, filled with normals, and
    its dense copy."""
    size = 1 + sum((n - 1) * s for n, s in zip(shape, stride))
    v = torch.empty(size, dtype=t, device="cuda").as_strided(shape, stride)
    v.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(seed)))
    return v, v.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 33])
def test_scan_rows_far_apart(D):
    T = 150
    x, dense = far_view((2, T, D), (FAR, D, 1), torch.bfloat16, 1)
    rec, inp = (torch.randn(2, T, D).bfloat16().cuda() for _ in range(2))
    lam, h0 = torch.full((D,), -4.0).cuda(), torch.randn(2, D).cuda()
    a = S.gated_scan(x, rec, inp, lam, h0=h0, save=True)
    b = S.gated_scan(dense, rec, inp, lam, h0=h0, save=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    da = S.gated_scan_grad(x, rec, inp, lam, x, a[2], h0=h0)
    db = S.gated_scan_grad(dense, rec, inp, lam, dense, b[2], h0=h0)
    assert all(torch.equal(p, q) for p, q in zip(da, db))
    out = x.new_empty(0).set_(x.untyped_storage(), 0, x.shape, x.stride())
    S.gated_scan(dense, rec, inp, lam, h0=h0, out=out)
    assert torch.equal(out, b[0])


@pytest.mark.gpu
def test_scan_steps_far_apart():
    # a time stride just under the limit: 2 GiB less one row
    D, step = 32, (1 << 30) - 32
    x, dense = far_view((1, 5, D), (D, step, 1), torch.bfloat16, 2)
    lam = torch.full((D,), -4.0).cuda()
    assert torch.equal(S.gated_scan(x, x, x, lam)[0], S.gated_scan(dense, dense, dense, lam)[0])


@pytest.mark.gpu
def test_norm_and_dropout_far_apart():
    for shape, stride in (((2, 48), (FAR, 1)), ((2, 45), (FAR, 1)), ((2, 30, 48), (FAR, 48, 1)),
                          ((1, 2, 48), (48, FAR, 1)), ((2, 900, 48), (FAR, 48, 1))):
        x, dense = far_view(shape, stride, torch.bfloat16, 3)
        a, b = (S.group_norm(v, 3, save=True) for v in (x, dense))
        assert all(torch.equal(p, q) for p, q in zip(a, b)), shape
        da = S.group_norm_grad(x, x, 3, None, None, *a[1:])
        db = S.group_norm_grad(dense, dense, 3, None, None, *b[1:])
        assert all(torch.equal(p, q) for p, q in zip(da, db)), shape
        if len(shape) == 2:
            assert torch.equal(S.dropout(x, 0.3, 1), S.dropout(dense, 0.3, 1))
        del x, a, da
        torch.cuda.empty_cache()


@pytest.mark.gpu
def test_broadcast_rows():
    row = torch.randn(1, 40).cuda()
    x = row.expand(9, 40)
    assert torch.equal(S.dropout(x, 0.4, 3), S.dropout(x.contiguous(), 0.4, 3))
    y = S.group_norm(x, 5)
    assert torch.equal(y, S.group_norm(x.contiguous(), 5))
    e = row.view(1, 1, 40).expand(3, 70, 40)
    lam = torch.full((40,), -4.0).cuda()
    d = e.contiguous()
    a, b = S.gated_scan(e, e, e, lam, save=True), S.gated_scan(d, d, d, lam, save=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    da = S.gated_scan_grad(e, e, e, lam, e, a[2])
    db = S.gated_scan_grad(d, d, d, lam, d, b[2])
    assert all(p is q is None or torch.equal(p, q) for p, q in zip(da, db))


def test_refused_strides_without_a_gpu():
    L = N.lib()

    def scan(time):
        st = (C.c_int64 * 10)(*([8, time] * 5))
        return L.zrl_gated_scan(64, 64, 64, 64, None, None, 1, 3, 8, 1, 8.0, st, 64, None, None,
                                None, 0, None)

    assert scan(1 << 30) == N.NOT_SUPPORTED and b"stride" in L.zrl_last_error(None)
    assert scan(-(1 << 30)) == N.NOT_SUPPORTED
    # rows of an output that overlap
    st = (C.c_int64 * 3)(8, 8, 4)
    assert L.zrl_dropout(64, None, None, 4, 8, 0, 0.1, 1, 0, st, 64, None) == N.INVALID_ARG
    assert b"overlap" in L.zrl_last_error(None)

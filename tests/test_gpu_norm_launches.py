"""Group norm and dropout as programs launch them: calls of several sizes in one
CUDA graph, on another stream, from two host threads."""
import threading

import pytest
import torch

from zealot_b200 import native as N
from zealot_b200 import sequence as S

pytestmark = pytest.mark.gpu


def sample(L, seed, n=200, C=64):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, L, C, generator=g).cuda(), torch.randn(n, L, C, generator=g).cuda()


def both(x, dy):
    y, mean, rstd = S.group_norm(x, 8, act="silu", save=True)
    return (y,) + S.group_norm_grad(x, dy, 8, None, None, mean, rstd, act="silu")


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


# Samples that a block holds in about 60 and 30 KB of shared memory, through one
# kernel: neither call may take away what the other was given.
SIZES = [480, 256]
GRAD_SIZES = [230, 120]


def test_block_sizes_in_one_graph():
    data = [sample(L, L) for L in SIZES + GRAD_SIZES]
    want = [both(*d) for d in data]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [both(*d) for d in data]
    for d in data:
        d[0].mul_(2.0), d[1].mul_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(same(a, both(*d)) for a, d in zip(got, data))
    assert not any(same(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("grad", [False, True])
def test_block_sizes_from_two_threads(grad):
    """The library's calls themselves, so that the threads are in them at the same
    time and not in turn at the interpreter."""
    L, n, C = N.lib(), 160, 32
    failed, start = [], threading.Barrier(2)

    def work(size):
        s = torch.cuda.Stream()
        x, dy = sample(size, size, n, C)
        y, dx = torch.empty_like(x), torch.empty_like(x)
        mean, rstd = torch.zeros(n, 4).cuda(), torch.ones(n, 4).cuda()
        ws = L.zrl_group_norm_workspace(n, size, C, 4, 1)
        w = torch.empty(ws, dtype=torch.uint8, device="cuda")
        p = [None if v is None else v.data_ptr() for v in (x, dy, mean, rstd, y, dx, w)]
        torch.cuda.synchronize()
        start.wait()
        for k in range(20000):
            if grad:
                status = L.zrl_group_norm_grad(p[0], p[1], None, None, p[2], p[3], n, size, C, 4, 0,
                                               2, None, p[5], None, None, p[6], ws, s.cuda_stream)
            else:
                status = L.zrl_group_norm(p[0], None, None, n, size, C, 4, 0, 2, 1e-5, None, p[4],
                                          None, None, None, 0, s.cuda_stream)
            if status != N.OK:
                failed.append((size, L.zrl_last_error(None)))
            if k % 100 == 0:
                s.synchronize()
        s.synchronize()

    threads = [threading.Thread(target=work, args=(v,)) for v in (GRAD_SIZES if grad else SIZES)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, (len(failed), failed[0])


def forms():
    """Rows; samples in a block; in two passes, one launch and several batches."""
    g = torch.Generator().manual_seed(3)
    out = []
    for shape in ((300, 96), (60, 30, 64), (3, 3000, 64), (9, 60000, 64)):
        out.append(tuple(torch.randn(shape, generator=g).cuda() for _ in range(2)))
    return out


def drops(x, dy):
    x, dy = x.view(-1, x.shape[-1]), dy.view(-1, dy.shape[-1])
    rows = torch.arange(x.shape[0], device="cuda").flip(0)
    return (S.dropout(x, 0.3, 5, stream=2, rows=rows, residual=dy), S.dropout_grad(dy, 0.3, 5),
            S.dropout(x[:, :51], 0.5, 6))


def test_every_form_in_a_graph():
    data = forms()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [both(*d) + drops(*d) for d in data]
    for d in data:
        d[0].mul_(0.5), d[1].add_(1.0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(same(a, both(*d) + drops(*d)) for a, d in zip(got, data))


def test_every_form_on_another_stream():
    data = forms()
    want = [both(*d) + drops(*d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [both(*d) + drops(*d) for d in data]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))


def test_messages_belong_to_their_thread():
    x = torch.zeros(4, 16).cuda()
    seen, met = {}, threading.Barrier(2)

    def work(name, call):
        with pytest.raises(N.ZrlError):
            call()
        met.wait()
        seen[name] = N.lib().zrl_last_error(None).decode()

    threads = [threading.Thread(target=work, args=a) for a in
               (("norm", lambda: S.group_norm(x, 4, eps=-1.0)),
                ("dropout", lambda: S.dropout(x, 2.0, 1)))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert "group_norm" in seen["norm"] and "dropout" in seen["dropout"]

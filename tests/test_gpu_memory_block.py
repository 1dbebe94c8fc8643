"""zealot_b200.memory.MemoryBlock: the operators together, against the same
block in 64 bits with torch's own differentiation, and the properties a PPO
update needs of it."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_gpu_dropout import keep_mask
from zealot_b200.memory import MemoryBlock

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def reference(block, u, h0, resets, dy, dh_last, key):
    """y, last state and all gradients in 64 bits."""
    q = {k: v.detach().cpu().double().requires_grad_() for k, v in block.parameters.items()}
    u, h0 = (t.cpu().double().requires_grad_() for t in (u, h0))
    B, T, D = u.shape
    x, rec, inp = (u @ q["w"].t() + q["b"]).split(D, -1)
    z = resets.cpu().bool().unsqueeze(-1)
    rate = block.c * torch.nn.functional.softplus(q["lam"])
    a = torch.exp(-rate * torch.sigmoid(rec)).masked_fill(z, 0.0)
    b = torch.sqrt(1 - a * a) * torch.sigmoid(inp) * x
    s, h = h0, []
    for t in range(T):
        s = a[:, t] * s + b[:, t]
        h.append(s)
    h = torch.stack(h, 1)
    g = h.reshape(B * T, block.groups, -1)
    g = (g - g.mean(-1, keepdim=True)) / torch.sqrt(g.var(-1, unbiased=False, keepdim=True) + 1e-5)
    n = torch.nn.functional.silu(g.reshape(B * T, D) * q["gamma"] + q["beta"])
    drop = round(65536 * block.p)
    keep = torch.from_numpy(keep_mask(np.arange(B * T), D, block.p, key, block.layer))
    y = u + (n * keep * (65536 / (65536 - drop))).reshape(B, T, D)
    ((y * dy.cpu().double()).sum() + (s * dh_last.cpu().double()).sum()).backward()
    return y.detach(), s.detach(), u.grad, {k: v.grad for k, v in q.items()}, h0.grad


def rel(got, want):
    return ((got.detach().cpu().double() - want).norm() / want.norm()).item()


# 32 bits: a chain of some ten roundings of 6e-8, taken up by sums of terms of
# either sign; the projection's product (tf32 off) adds sqrt(D) of them.
@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D,groups", [(3, 20, 32, 4), (8, 150, 48, 6), (2, 70, 30, 3)])
def test_block_against_64_bits(B, T, D, groups):
    g = torch.Generator().manual_seed(B + T)
    block = MemoryBlock(D, groups=groups, p=0.2, layer=3, seed=2)
    u, dy = (torch.randn(B, T, D, generator=g).cuda() for _ in range(2))
    h0, dl = (torch.randn(B, D, generator=g).cuda() for _ in range(2))
    resets = (torch.rand(B, T, generator=g) < 0.05).cuda()
    want = reference(block, u, h0, resets, dy, dl, key=11)
    y, last, saved = block.forward(u, h0=h0, resets=resets, key=11, save=True)
    du, grads, dh0 = block.backward(saved, dy, dh_last=dl)
    assert rel(y, want[0]) < 1e-5 and rel(last, want[1]) < 1e-5
    assert rel(du, want[2]) < 1e-4 and rel(dh0, want[4]) < 1e-4
    for k, v in want[3].items():
        assert rel(grads[k], v) < 1e-4, k
    assert torch.equal(y, block.forward(u, h0=h0, resets=resets, key=11)[0])


@pytest.mark.gpu
def test_the_rollout_meets_the_updates_masks():
    B, T, D = 5, 30, 64
    block = MemoryBlock(D, p=0.5)
    u = torch.randn(B, T, D, generator=torch.Generator().manual_seed(0)).cuda()
    resets = (torch.rand(B, T, generator=torch.Generator().manual_seed(1)) < 0.1).cuda()
    y, last = block.forward(u, resets=resets, key=5)
    state = torch.zeros(B, D).cuda()
    for t in range(T):
        rows = torch.arange(B).cuda() * T + t
        s, state = block.step(u[:, t].contiguous(), state, resets=resets[:, t], rows=rows, key=5)
        # the same samples are dropped, and the kept values agree
        assert torch.equal(s == u[:, t], y[:, t] == u[:, t])
        torch.testing.assert_close(s, y[:, t], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(state, last, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_bf16_block_stays_near_32_bits():
    B, T, D = 16, 48, 128
    a, b = MemoryBlock(D, seed=4), MemoryBlock(D, seed=4, dtype=torch.bfloat16)
    u = torch.randn(B, T, D, generator=torch.Generator().manual_seed(0)).cuda()
    dy = torch.randn(B, T, D, generator=torch.Generator().manual_seed(1)).cuda()
    ya, _, sa = a.forward(u, key=1, save=True)
    yb, _, sb = b.forward(u.bfloat16(), key=1, save=True)
    assert rel(yb, ya.cpu().double()) < 2e-2
    ga, gb = a.backward(sa, dy)[1], b.backward(sb, dy.bfloat16())[1]
    for k in ga:
        # a handful of bf16 roundings (2^-8 each) on every term
        assert rel(gb[k], ga[k].cpu().double()) < 5e-2, k


@pytest.mark.gpu
def test_the_recall_example_learns():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "recall.py")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    a, b = (float(v) for v in r.stdout.split("squared error")[1].split("\n")[0].split("->"))
    assert a > 0.9 and b < 0.5, r.stdout
    assert float(r.stdout.split("update:")[1]) < 1e-3

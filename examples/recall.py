"""Trains a memory block to recall: an environment shows a sign at the first step
of an episode and noise afterwards, and every step has to name the sign.

    python examples/recall.py [--envs 512] [--steps 48] [--width 64] [--updates 60]

Prints the squared error before and after, then plays the trained block step by
step and prints how far its outputs are from the update's.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from zealot_b200.memory import MemoryBlock  # noqa: E402


def episodes(g, B, T, D):
    """Features, episode starts and the sign of the running episode."""
    resets = torch.rand(B, T, generator=g, device="cuda") < 0.05
    resets[:, 0] = True
    sign = torch.randint(0, 2, (B, T), generator=g, device="cuda") * 2.0 - 1
    # the latest start's column, by a running maximum
    at = torch.where(resets, torch.arange(T, device="cuda"), 0).cummax(1).values
    target = sign.gather(1, at)
    u = 0.3 * torch.randn(B, T, D, generator=g, device="cuda")
    u[..., 0] = torch.where(resets, target, 0.0)
    u[..., 1] = resets.float()
    return u, resets.to(torch.uint8), target


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--envs", type=int, default=512)
    p.add_argument("--steps", type=int, default=48)
    p.add_argument("--width", type=int, default=64)
    p.add_argument("--updates", type=int, default=60)
    a = p.parse_args()
    g = torch.Generator(device="cuda").manual_seed(1)
    block = MemoryBlock(a.width, p=0.1, seed=1)
    out = torch.zeros(a.width, device="cuda")
    params = dict(block.parameters, out=out)
    m = {k: torch.zeros_like(v) for k, v in params.items()}
    v = {k: torch.zeros_like(t) for k, t in params.items()}
    first = None
    for i in range(1, a.updates + 1):
        u, resets, target = episodes(g, a.envs, a.steps, a.width)
        y, _, saved = block.forward(u, resets=resets, key=i, save=True)
        err = y @ out - target
        first = err.square().mean().item() if first is None else first
        de = err * (2 / err.numel())
        _, grads, _ = block.backward(saved, de.unsqueeze(-1) * out)
        grads["out"] = (de.unsqueeze(-1) * y).sum((0, 1))
        for k, t in params.items():  # Adam
            m[k].mul_(0.9).add_(grads[k], alpha=0.1)
            v[k].mul_(0.999).addcmul_(grads[k], grads[k], value=0.001)
            t.sub_(0.02 * (m[k] / (1 - 0.9 ** i)) / ((v[k] / (1 - 0.999 ** i)).sqrt() + 1e-8))
    u, resets, target = episodes(g, a.envs, a.steps, a.width)
    y, _ = block.forward(u, resets=resets, key=7)
    print(f"squared error {first:.3f} -> {(y @ out - target).square().mean().item():.3f}")
    state = torch.zeros(a.envs, a.width, device="cuda")
    far = 0.0
    for t in range(a.steps):
        rows = torch.arange(a.envs, device="cuda") * a.steps + t
        s, state = block.step(u[:, t].contiguous(), state, resets=resets[:, t], rows=rows, key=7)
        far = max(far, (s - y[:, t]).abs().max().item())
    print(f"rollout against update: {far:.2e}")
    return first, (y @ out - target).square().mean().item(), far


if __name__ == "__main__":
    main()

"""A temporal block for recurrent actor-critics, from the operators of ``sequence``.

    y = u + dropout(act(group_norm(gated_scan(x, rec, inp))))
    x, rec, inp = the three parts of W u + b

for features u [B, T, D] of B environments over T steps.  The same block runs
step by step in the rollout (``step``) and over whole rows in the update
(``forward`` / ``backward``).  Episode starts cut the recurrence; every step is
normalized by itself, so nothing of a later step reaches an earlier one; and the
dropout mask of a sample depends on its number alone, so the update meets the
masks of the rollout and an unchanged policy has a ratio of exactly one up to
rounding, whatever the order of its minibatches.  The projection is a plain
library product.
"""
from __future__ import annotations

import math

import torch

from . import sequence as S


class MemoryBlock:
    """``parameters`` holds the block's tensors: ``w`` [3 D, D] in the compute
    type, and float32 ``b`` [3 D], ``lam``, ``gamma``, ``beta`` [D]."""

    def __init__(self, width: int, groups: int = 8, p: float = 0.1, act: str = "silu",
                 layer: int = 0, dtype=torch.float32, device="cuda", seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        k = 1 / math.sqrt(width)
        # decays at an open gate uniform in [0.9, 0.999]
        a = 0.9 + 0.099 * torch.rand(width, generator=g, dtype=torch.float64)
        self.width, self.groups, self.p, self.act, self.layer = width, groups, p, act, layer
        self.c = 8.0
        self.parameters = {
            "w": ((torch.rand(3 * width, width, generator=g) * 2 - 1) * k).to(device, dtype),
            "b": torch.zeros(3 * width, device=device),
            "lam": torch.log(torch.expm1(-torch.log(a) / self.c)).float().to(device),
            "gamma": torch.ones(width, device=device),
            "beta": torch.zeros(width, device=device),
        }

    def _project(self, u):
        """x, rec, inp: slices of one product's output."""
        w, b = self.parameters["w"], self.parameters["b"]
        p = torch.addmm(b.to(w.dtype), u.reshape(-1, self.width), w.t())
        return p.view(*u.shape[:-1], 3 * self.width).split(self.width, -1)

    def _head(self, u, h, rows, key, save):
        q = self.parameters
        flat = h.reshape(-1, self.width)
        n = S.group_norm(flat, self.groups, q["gamma"], q["beta"], act=self.act, save=save)
        y = S.dropout(n[0] if save else n, self.p, key, stream=self.layer, rows=rows,
                      residual=u.reshape(-1, self.width))
        return y.view(u.shape), n[1:] if save else None

    def forward(self, u, h0=None, resets=None, rows=None, key: int = 0, save: bool = False):
        """(y, last state), and with ``save`` what ``backward`` takes.  rows: the
        samples' numbers [B * T]; by default they count the samples env by env."""
        x, rec, inp = self._project(u)
        r = S.gated_scan(x, rec, inp, self.parameters["lam"], h0=h0, resets=resets, c=self.c,
                         save=save)
        y, stats = self._head(u, r[0], rows, key, save)
        if not save:
            return y, r[1]
        return y, r[1], (u, x, rec, inp, r[0], r[2], stats, h0, resets, rows, key)

    def backward(self, saved, dy, dh_last=None):
        """(du, gradients by parameter, dh0) for dy on y and dh_last on the last state."""
        u, x, rec, inp, h, carry, (mean, rstd), h0, resets, rows, key = saved
        q, D = self.parameters, self.width
        dn = S.dropout_grad(dy.reshape(-1, D), self.p, key, stream=self.layer, rows=rows)
        dh, dgamma, dbeta = S.group_norm_grad(h.reshape(-1, D), dn, self.groups, q["gamma"],
                                              q["beta"], mean, rstd, act=self.act, out=dn)
        # the three gradients side by side, as the projection's output was
        dp = torch.empty(*u.shape[:-1], 3 * D, dtype=u.dtype, device=u.device)
        *_, dlam, dh0 = S.gated_scan_grad(x, rec, inp, q["lam"], dh.view(u.shape), carry,
                                          dh_last=dh_last, h0=h0, resets=resets, c=self.c,
                                          out=dp.split(D, -1))
        dp = dp.view(-1, 3 * D)
        du = torch.addmm(dy.reshape(-1, D), dp, q["w"]).view(u.shape)
        return du, {"w": dp.t() @ u.reshape(-1, D), "b": dp.sum(0, dtype=torch.float32),
                    "lam": dlam, "gamma": dgamma, "beta": dbeta}, dh0

    def step(self, u, state, resets=None, rows=None, key: int = 0):
        """One step of the rollout: (y, new state) for u [B, D], state [B, D] fp32.
        rows: the samples' numbers, env * T + t for the masks ``forward`` draws."""
        x, rec, inp = self._project(u)
        h, state = S.gated_step(x, rec, inp, self.parameters["lam"], state, resets=resets,
                                c=self.c)
        return self._head(u, h, rows, key, False)[0], state

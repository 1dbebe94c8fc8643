"""What the sequence operators of zealot_b200 are measured on.

The operators are the parts of a policy with memory that is trained over
rollouts: the gated scan (a gated linear recurrence over time, cut where an
episode begins), its gradient and its single step; group norm with an
activation over channels-last rows, and its gradient; dropout whose mask
comes from a counter and is drawn again wherever it is needed.

``run`` computes an operator in elementary torch operations, in 32 bits,
where ``own`` is false, and with the framework's own kernels where it is
true.  ``exact`` restates the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
GATE_C = 8.0
EPS = 1e-5


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one robot's controller: a single time step of a single row
        dict(name="step_one_robot_f32", op="step", type="f32", B=1, T=1, D=256, resets=0.0),
        # the rollout step of 4,096 environments
        dict(name="step_envs_bf16", op="step", type="bf16", B=4096, T=1, D=512, resets=0.005),
        # a whole rollout run again without gradients (values for the advantages)
        dict(name="scan_rollout_f32", op="scan", type="f32", B=4096, T=24, D=128,
             resets=0.005, layout="plain", h0=True),
        # one minibatch of whole rows (24,576 samples) out of a time-major rollout buffer
        dict(name="scan_train_minibatch_bf16", op="scan_train", type="bf16", B=1024, T=24, D=512,
             resets=0.005, layout="time", h0=True),
        # long recordings, an odd length, the three inputs slices of one projection's output
        dict(name="scan_train_long_bf16", op="scan_train", type="bf16", B=8, T=8191, D=480,
             resets=0.002, layout="fused", h0=False),
        # one very long recording: few rows, the time axis is all there is to split
        dict(name="scan_one_long_f32", op="scan", type="f32", B=1, T=65536, D=512,
             resets=0.0, layout="plain", h0=True),
        # every sample of a minibatch normalized by itself, in a hidden layer's width
        dict(name="norm_rows_bf16", op="norm", type="bf16", N=24576, L=1, C=512, G=16, act="elu"),
        # a rollout's samples at an odd group width, with the gradient
        dict(name="norm_train_rows_f32", op="norm_train", type="f32", N=98304, L=1, C=250, G=10,
             act="silu"),
        # feature maps of a depth camera in inference
        dict(name="norm_maps_f16", op="norm", type="f16", N=64, L=58 * 87, C=64, G=8, act="elu"),
        # wide feature maps of a few cameras, with the gradient
        dict(name="norm_train_maps_bf16", op="norm_train", type="bf16", N=16, L=60 * 106, C=256,
             G=32, act="gelu"),
        # a minibatch of shuffled samples, each with the mask its rollout step drew
        dict(name="dropout_rows_bf16", op="dropout", type="bf16", N=24576, D=512, p=0.1,
             rows=True, residual=True),
        # the gradient of a whole rollout at an odd width
        dict(name="dropout_grad_odd_f32", op="dropout_grad", type="f32", N=98304, D=333, p=0.25,
             rows=False, residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["step", "scan", "scan_train", "norm", "norm_train", "dropout",
                         "dropout_grad"])
        case = dict(op=op, type=rng.choice(["f32", "bf16", "f16"]))
        if op == "step":
            case |= dict(B=_log_int(rng, 1, 16384), T=1, D=_log_int(rng, 32, 1024),
                         resets=rng.choice([0.0, 0.005]))
        elif op in ("scan", "scan_train"):
            case |= dict(B=_log_int(rng, 1, 16384), T=_log_int(rng, 1, 65536),
                         D=_log_int(rng, 32, 1024), resets=rng.choice([0.0, 0.002, 0.05]),
                         layout=rng.choice(["plain", "time", "fused"]),
                         h0=rng.random() < 0.5)
            if case["B"] * case["T"] * case["D"] < 1 << 18:
                continue
        elif op in ("norm", "norm_train"):
            G, width = _log_int(rng, 1, 32), _log_int(rng, 2, 64)
            rows = rng.random() < 0.5
            case |= dict(N=_log_int(rng, 256, 98304) if rows else _log_int(rng, 1, 256),
                         L=1 if rows else _log_int(rng, 16, 20000), C=G * width, G=G,
                         act=rng.choice(["none", "elu", "silu", "gelu"]))
            if case["N"] * case["L"] * case["C"] < 1 << 16:
                continue
        else:
            case |= dict(N=_log_int(rng, 64, 98304), D=_log_int(rng, 8, 1024),
                         p=rng.choice([0.0, 0.1, 0.25, 0.5]), rows=rng.random() < 0.5,
                         residual=op == "dropout" and rng.random() < 0.5)
        if work(case)["bytes"] <= most:
            return case


def work(case):
    s, op = SIZE[case["type"]], case["op"]
    if op in ("step", "scan", "scan_train"):
        B, T, D = case["B"], case["T"], case["D"]
        n = B * T * D
        marks = B * T if case["resets"] else 0
        start = 4 * B * D if op == "step" or case["h0"] else 0
        fwd = 4 * s * n + marks + start + 4 * B * D + 4 * D
        if op != "scan_train":
            return {"bytes": fwd, "flops": 20 * n}
        # the gradient reads the three inputs and dh and writes three gradients;
        # dh_last in, dh0 and dlam out
        return {"bytes": fwd + 7 * s * n + marks + start + 8 * B * D + 8 * D, "flops": 60 * n}
    if op in ("norm", "norm_train"):
        n = case["N"] * case["L"] * case["C"]
        fwd = 2 * s * n + 8 * case["C"]
        if op == "norm":
            return {"bytes": fwd, "flops": 12 * n}
        return {"bytes": fwd + 3 * s * n + 16 * case["C"] + 16 * case["N"] * case["G"],
                "flops": 36 * n}
    n = case["N"] * case["D"]
    return {"bytes": (3 if case["residual"] else 2) * s * n + (8 * case["N"] if case["rows"] else 0),
            "flops": 16 * n}


# ---------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _lam(g, D):
    # the decay at an open gate, exp(-c softplus(lam)), uniform in [0.9, 0.999]
    a = 0.9 + 0.099 * torch.rand(D, generator=g, device=DEV, dtype=torch.float64)
    return torch.log(torch.expm1(-torch.log(a) / GATE_C)).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    op = case["op"]
    st = {"case": case, "op": op}
    if op == "step":
        B, D = case["B"], case["D"]
        for k in ("x", "rec", "inp"):
            st[k] = _normal(g, B, D).to(t)
        st["lam"] = _lam(g, D)
        st["state"] = _normal(g, B, D) * 0.5
        st["resets"] = None
        if case["resets"]:
            st["resets"] = (torch.rand(B, generator=g, device=DEV) < case["resets"]).to(torch.uint8)
    elif op in ("scan", "scan_train"):
        B, T, D = case["B"], case["T"], case["D"]
        if case["layout"] == "fused":  # one projection's output, [B, T, 3 D]
            st["x"], st["rec"], st["inp"] = _normal(g, B, T, 3 * D).to(t).split(D, dim=-1)
        else:
            for k in ("x", "rec", "inp"):
                v = _normal(g, T, B, D) if case["layout"] == "time" else _normal(g, B, T, D)
                st[k] = v.to(t).transpose(0, 1) if case["layout"] == "time" else v.to(t)
        st["lam"] = _lam(g, D)
        st["h0"] = _normal(g, B, D) * 0.5 if case["h0"] else None
        st["resets"] = None
        if case["resets"]:
            m = torch.rand(T, B, generator=g, device=DEV) < case["resets"]
            m = m.to(torch.uint8)
            st["resets"] = m.t() if case["layout"] == "time" else m.t().contiguous()
        if op == "scan_train":
            dh = _normal(g, T, B, D) if case["layout"] == "time" else _normal(g, B, T, D)
            st["dh"] = dh.to(t).transpose(0, 1) if case["layout"] == "time" else dh.to(t)
            st["dh_last"] = _normal(g, B, D)
    elif op in ("norm", "norm_train"):
        N, L, C = case["N"], case["L"], case["C"]
        offset, spread = _normal(g, C) * 0.5, 0.5 + torch.rand(C, generator=g, device=DEV)
        st["x"] = torch.addcmul(offset, _normal(g, N, L, C), spread).to(t)
        st["gamma"] = 1 + 0.2 * _normal(g, C)
        st["beta"] = 0.2 * _normal(g, C)
        if op == "norm_train":
            st["dy"] = _normal(g, N, L, C).to(t)
    else:
        N, D = case["N"], case["D"]
        st["x"] = _normal(g, N, D).to(t)
        st["residual"] = _normal(g, N, D).to(t) if case["residual"] else None
        # shuffled samples of a longer run, whose numbers pass 32 bits
        st["rows"] = None
        if case["rows"]:
            st["rows"] = torch.randperm(N, generator=g, device=DEV) + (1 << 32) - N // 2
        st["seed"] = (0x9E3779B97F4A7C15 * (seed + 1)) % (1 << 63)
        st["stream"] = seed % 1000 + 1
    return st


# ---------------------------------------------------------------- plain forms

def _softplus(v):
    return torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0)


def _gates(st, reset):
    """a, m, sigmoid(inp), sigmoid(rec), softplus(lam) in 32 bits."""
    sp = _softplus(st["lam"])
    sr, si = torch.sigmoid(st["rec"].float()), torch.sigmoid(st["inp"].float())
    la = -GATE_C * sp * sr
    a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    if reset is not None:
        reset = reset.bool().unsqueeze(-1)
        a, m = torch.where(reset, 0.0, a), torch.where(reset, 1.0, m)
    return a, m, si, sr, sp


def _scan(a, b, first):
    """h_t = a_t h_{t-1} + b_t along dim 1, h_{-1} = first: in each pass every
    position takes in the 2^k positions before it, so log2 T passes."""
    h, p = b.clone(), a.clone()
    if first is not None:
        h[:, 0] += a[:, 0] * first
    s = 1
    while s < h.shape[1]:
        h[:, s:] += p[:, s:] * h[:, :-s]
        p[:, s:] = p[:, s:] * p[:, :-s]
        s *= 2
    return h


def _plain_scan(st, grad):
    t = st["x"].dtype
    x = st["x"].float()
    a, m, si, sr, sp = _gates(st, st["resets"])
    h = _scan(a, m * si * x, st["h0"])
    out = {"h": h.to(t), "h_last": h[:, -1].clone()}
    if not grad:
        return out
    dh = st["dh"].float()
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + st["dh_last"].unsqueeze(1)], dim=1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    g = _scan(after.flip(1), dh.flip(1), None).flip(1)
    first = st["h0"] if st["h0"] is not None else torch.zeros_like(h[:, 0])
    before = torch.cat([first.unsqueeze(1), h[:, :-1]], dim=1)
    dla = g * (before * a - torch.where(a * m > 0, si * x * a * a / m, 0.0))
    out["dx"] = (g * m * si).to(t)
    out["drec"] = (dla * (-GATE_C * sp) * sr * (1 - sr)).to(t)
    out["dinp"] = (g * m * x * si * (1 - si)).to(t)
    out["dlam"] = (dla * (-GATE_C * sr)).sum((0, 1)) * torch.sigmoid(st["lam"])
    if st["h0"] is not None:
        out["dh0"] = a[:, 0] * g[:, 0]
    return out


def _plain_step(st):
    a, m, si, _, _ = _gates(st, st["resets"])
    h = a * st["state"] + m * si * st["x"].float()
    return {"h": h.to(st["x"].dtype), "state": h}


def _act(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "elu":
        e = torch.exp(z.clamp(max=0))
        return torch.where(z > 0, z, torch.expm1(z.clamp(max=0))), torch.where(z > 0, 1.0, e)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_norm(st, grad):
    c = st["case"]
    N, L, C, G = c["N"], c["L"], c["C"], c["G"]
    t = st["x"].dtype
    x = st["x"].float().view(N, L, G, C // G)
    gamma, beta = st["gamma"].view(G, C // G), st["beta"].view(G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
    xh = (x - mean) * rstd
    y, dact = _act(xh * gamma + beta, c["act"])
    out = {"y": y.reshape(N, L, C).to(t)}
    if grad:
        dz = st["dy"].float().view_as(xh) * dact
        out["dgamma"] = (dz * xh).sum((0, 1)).reshape(C)
        out["dbeta"] = dz.sum((0, 1)).reshape(C)
        d = dz * gamma
        dx = rstd * (d - d.mean((1, 3), keepdim=True) - xh * (d * xh).mean((1, 3), keepdim=True))
        out["dx"] = dx.reshape(N, L, C).to(t)
    return out


def _mulhilo(k, v):
    """High and low 32 bits of the product of two 32-bit numbers held in 64."""
    lo, hi = k * (v & 0xFFFF), k * (v >> 16)
    mid = hi + (lo >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def _philox(c, k0, k1):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11) on 64-bit tensors."""
    c0, c1, c2, c3 = c
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c0)
        h1, l1 = _mulhilo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def _plain_dropout(st):
    """Eight columns take the eight 16-bit lanes of one Philox call, low half
    of each word first; a value stays where its lane is at least 65536 p."""
    x = st["x"].float()
    N, D = x.shape
    drop = round(65536 * st["case"]["p"])
    row = st["rows"] if st["rows"] is not None else torch.arange(N, device=DEV)
    col = torch.arange((D + 7) // 8, device=DEV)
    zero = torch.zeros(N, len(col), dtype=torch.int64, device=DEV)
    w = _philox((zero + col, zero + (row & 0xFFFFFFFF)[:, None], zero + (row >> 32)[:, None],
                 zero + st["stream"]), st["seed"] & 0xFFFFFFFF, st["seed"] >> 32)
    w = torch.stack(w, -1)
    lanes = torch.stack([w & 0xFFFF, w >> 16], -1).reshape(N, -1)[:, :D]
    y = torch.where(lanes >= drop, x * (65536 / (65536 - drop)), 0.0)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(st["x"].dtype)}


# ---------------------------------------------------------------- one pass

def run(st):
    op, c = st["op"], st["case"]
    if own:
        return _run_own(st, op, c)
    if op == "step":
        return _plain_step(st)
    if op in ("scan", "scan_train"):
        return _plain_scan(st, op == "scan_train")
    if op in ("norm", "norm_train"):
        return _plain_norm(st, op == "norm_train")
    return _plain_dropout(st)


def _run_own(st, op, c):
    from zealot_b200 import sequence as S
    if op == "step":
        h, state = S.gated_step(st["x"], st["rec"], st["inp"], st["lam"], st["state"],
                                resets=st["resets"], c=GATE_C)
        return {"h": h, "state": state}
    if op == "scan":
        h, last = S.gated_scan(st["x"], st["rec"], st["inp"], st["lam"], h0=st["h0"],
                               resets=st["resets"], c=GATE_C)
        return {"h": h, "h_last": last}
    if op == "scan_train":
        h, last, carry = S.gated_scan(st["x"], st["rec"], st["inp"], st["lam"], h0=st["h0"],
                                      resets=st["resets"], c=GATE_C, save=True)
        d = S.gated_scan_grad(st["x"], st["rec"], st["inp"], st["lam"], st["dh"], carry,
                              dh_last=st["dh_last"], h0=st["h0"], resets=st["resets"], c=GATE_C)
        out = {"h": h, "h_last": last, "dx": d[0], "drec": d[1], "dinp": d[2], "dlam": d[3]}
        if st["h0"] is not None:
            out["dh0"] = d[4]
        return out
    if op == "norm":
        return {"y": S.group_norm(st["x"], c["G"], st["gamma"], st["beta"], act=c["act"],
                                  eps=EPS)}
    if op == "norm_train":
        y, mean, rstd = S.group_norm(st["x"], c["G"], st["gamma"], st["beta"], act=c["act"],
                                     eps=EPS, save=True)
        dx, dgamma, dbeta = S.group_norm_grad(st["x"], st["dy"], c["G"], st["gamma"],
                                              st["beta"], mean, rstd, act=c["act"])
        return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "dropout":
        return {"y": S.dropout(st["x"], c["p"], st["seed"], stream=st["stream"],
                               rows=st["rows"], residual=st["residual"])}
    return {"y": S.dropout_grad(st["x"], c["p"], st["seed"], stream=st["stream"],
                                rows=st["rows"])}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("step", "scan", "scan_train"):
        return _exact_scan(st, case)
    if case["op"] in ("norm", "norm_train"):
        return _exact_norm(st, case)
    return _exact_dropout(st, case)


def _exact_scan(st, case):
    """The recurrence step by step; the gradient by the chain rule at each step."""
    one = case["op"] == "step"
    x, rec, inp = (st[k].unsqueeze(1).double() if one else st[k].double()
                   for k in ("x", "rec", "inp"))
    B, T, D = x.shape
    reset = torch.zeros(B, T, 1, dtype=torch.bool, device=DEV)
    if st["resets"] is not None:
        reset = (st["resets"] != 0).reshape(B, T, 1)
    rate = GATE_C * torch.log1p(torch.exp(st["lam"].double()))
    open_r, open_i = 1 / (1 + torch.exp(-rec)), 1 / (1 + torch.exp(-inp))
    decay = torch.exp(-rate * open_r).masked_fill(reset, 0)
    scale = torch.sqrt((1 - decay) * (1 + decay))
    first = st["state"] if one else st["h0"]
    s = torch.zeros(B, D, dtype=torch.float64, device=DEV) if first is None else first.double()
    hs = torch.empty(B, T + 1, D, dtype=torch.float64, device=DEV)
    hs[:, 0] = s
    feed = scale * open_i * x
    for i in range(T):
        s = torch.addcmul(feed[:, i], decay[:, i], s)
        hs[:, i + 1] = s
    if one:
        return {"h": hs[:, 1], "state": hs[:, 1]}
    out = {"h": hs[:, 1:], "h_last": hs[:, -1]}
    if case["op"] != "scan_train":
        return out
    g = torch.empty_like(x)
    s = st["dh_last"].double()
    dh = st["dh"].double()
    for i in range(T - 1, -1, -1):
        s = s + dh[:, i]
        g[:, i] = s
        s = s * decay[:, i]
    # h = decay s' + scale gate x, scale^2 + decay^2 = 1: d scale = -(decay / scale) d decay
    d_decay = g * (hs[:, :-1] - decay / scale * open_i * x)
    d_open = d_decay * -rate * decay
    out["dx"] = g * scale * open_i
    out["drec"] = d_open * open_r * (1 - open_r)
    out["dinp"] = g * scale * x * open_i * (1 - open_i)
    out["dlam"] = (d_decay * decay * -open_r).sum((0, 1)) * GATE_C / (1 + torch.exp(-st["lam"].double()))
    if st["h0"] is not None:
        out["dh0"] = s
    return out


def _exact_norm(st, case):
    """Sums over whole groups; the gradient of the mean and the variance apart."""
    N, L, C, G = case["N"], case["L"], case["C"], case["G"]
    w = C // G
    n = L * w
    x = st["x"].double().reshape(N, L, G, w).permute(0, 2, 1, 3).reshape(N, G, n)
    gamma = st["gamma"].double().reshape(G, 1, w).expand(G, L, w).reshape(G, n)
    beta = st["beta"].double().reshape(G, 1, w).expand(G, L, w).reshape(G, n)

    def back(v):
        return v.reshape(N, G, L, w).permute(0, 2, 1, 3).reshape(N, L, C)

    mid = x - x.sum(-1, keepdim=True) / n
    sd = torch.sqrt((mid * mid).sum(-1, keepdim=True) / n + EPS)
    z = mid / sd * gamma + beta
    act = case["act"]
    if act == "elu":
        y, slope = torch.where(z > 0, z, torch.expm1(z)), torch.exp(z.clamp(max=0))
    elif act == "silu":
        q = 1 + torch.exp(-z)
        y, slope = z / q, 1 / q + z * (q - 1) / (q * q)
    elif act == "gelu":
        cdf = torch.special.ndtr(z)
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    out = {"y": back(y)}
    if case["op"] == "norm_train":
        dz = st["dy"].double().reshape(N, L, G, w).permute(0, 2, 1, 3).reshape(N, G, n) * slope
        out["dbeta"] = back(dz).sum((0, 1))
        out["dgamma"] = back(dz * mid / sd).sum((0, 1))
        d = dz * gamma / sd
        d_var = (d * mid).sum(-1, keepdim=True) / (sd * sd)
        d = d - d_var * mid / n
        out["dx"] = back(d - d.sum(-1, keepdim=True) / n)
    return out


def _exact_dropout(st, case):
    """The mask from numpy's unsigned integers, words and halves by division."""
    N, D = case["N"], case["D"]
    rows = np.arange(N, dtype=np.uint64) if st["rows"] is None else st["rows"].cpu().numpy().astype(np.uint64)
    two32 = np.uint64(1 << 32)
    cols = np.arange((D + 7) // 8, dtype=np.uint64)
    c = [np.broadcast_to(v, (N, len(cols))).copy() for v in
         (cols[None], (rows % two32)[:, None], (rows // two32)[:, None], np.uint64(st["stream"]))]
    k = [st["seed"] % (1 << 32), st["seed"] // (1 << 32)]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [q // two32 ^ c[1] ^ np.uint64(k[0]), q % two32, p // two32 ^ c[3] ^ np.uint64(k[1]),
             p % two32]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    lanes = np.empty((N, len(cols), 8), np.uint32)
    for j in range(8):
        lanes[:, :, j] = c[j // 2] % np.uint64(65536) if j % 2 == 0 else c[j // 2] // np.uint64(65536)
    drop = round(65536 * case["p"])
    keep = torch.from_numpy(lanes.reshape(N, -1)[:, :D] >= drop).to(DEV)
    y = st["x"].double() * 65536 / (65536 - drop) * keep
    if st["residual"] is not None:
        y = y + st["residual"].double()
    return {"y": y}

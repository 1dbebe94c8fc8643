"""Operators of a policy with memory, on torch CUDA tensors.

A recurrent actor-critic trained over rollouts needs, beside the MLP path of
``zealot_rl``: a recurrence over time that episode ends cut, a norm, and
dropout whose mask the update can draw exactly as the rollout step did.

Every call queues its kernels of libzealot_rl.so on the current torch stream
of the tensors' device and returns without waiting, as torch's own operators
do, so calls may be captured in a CUDA graph.  Tensors made on another stream
are ordered by the caller, as with torch.  Element types are float32,
bfloat16 and float16; sums, states, statistics and parameters are float32.
Gradients are calls of their own (``*_grad``), like the rest of this package.
A refused argument raises ``native.ZrlError`` or ``TypeError``.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import native as N

#: what ``act`` of group_norm may be
ACTIVATIONS = {"none": 0, "elu": 1, "silu": 2, "gelu": 3}

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32 = torch.float32
# the cheap forms of torch.cuda.current_device() and current_stream().cuda_stream
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _invalid(msg: str):
    return N.ZrlError(N.INVALID_ARG, msg)


def _dtype(x) -> int:
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"element type {x.dtype}: float32, bfloat16 or float16")
    if not x.is_cuda:
        raise TypeError(f"tensor on {x.device}: these operators take CUDA tensors")
    return dt


def _call(fn, device, *args):
    """fn(*args, stream) on the device's current stream."""
    i = device.index
    if _device() == i:
        status = fn(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            status = fn(*args, _stream(i))
    if status != N.OK:
        raise N.ZrlError(status, N.lib().zrl_last_error(None).decode())


@functools.lru_cache(maxsize=4096)
def _bytes(name: str, *sizes) -> int:
    """The workspace of a call of these sizes."""
    return getattr(N.lib(), name)(*sizes)


def _workspace(name: str, f32, *sizes):
    """(tensor to keep until the call, address, bytes); f32: an fp32 tensor of the device."""
    n = _bytes(name, *sizes)
    if not n:
        return None, None, 0
    t = f32.new_empty(n // 4)
    return t, t.data_ptr(), n


def _same(name, t, shape, dtype, device):
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name}: {t.dtype} on {t.device}, expected {dtype} on {device}")
    if t.shape != shape:
        raise _invalid(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _row_stride(name, t, D):
    """The stride between the rows of D elements that t's leading axes merge into."""
    if D > 1 and t.stride(-1) != 1:
        raise _invalid(f"{name}: the last axis is not dense")
    try:
        v = t.view(-1, D)
    except RuntimeError:
        raise _invalid(f"{name}: the leading axes do not merge into one row axis") from None
    return v.stride(0)


def _dense_like(x):
    """An empty dense tensor of x's shape, in the order the shape is written."""
    if x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _f32(name, t, shape, device):
    """The address of an fp32 parameter, state or statistic; None stays None."""
    if t is None:
        return None
    if t.dtype is _F32 and t.shape == shape and t.is_contiguous() and t.device == device:
        return t.data_ptr()
    _same(name, t, shape, _F32, device)
    raise _invalid(f"{name}: not contiguous")


def _bt(name, t):
    """(batch, time) strides of a [B, T, D] tensor whose last axis is dense."""
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise _invalid(f"{name}: the last axis is not dense")
    return t.stride(0), t.stride(1)


def _like(x):
    """An empty tensor of x's shape: time-major in memory where x is."""
    if x.is_contiguous():
        return torch.empty_like(x)
    B, T, D = x.shape
    if x.stride(0) < x.stride(1) and B > 1 and T > 1:
        return torch.empty((T, B, D), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((B, T, D), dtype=x.dtype, device=x.device)


def _scan_inputs(x, rec, inp, lam, h0, resets, shape, dev):
    """Checks what forward and gradient share; (lam, h0, resets) addresses."""
    t = x.dtype
    if not (rec.dtype is t and inp.dtype is t and rec.shape == shape and inp.shape == shape and
            rec.device == dev and inp.device == dev):
        _same("rec", rec, shape, t, dev)
        _same("inp", inp, shape, t, dev)
    D = shape[-1]
    p_z = None
    if resets is not None:
        if resets.dtype not in (torch.uint8, torch.bool) or resets.device != dev:
            raise TypeError("resets: uint8 or bool on x's device")
        if resets.shape != shape[:-1]:
            raise _invalid(f"resets: shape {tuple(resets.shape)}, expected {tuple(shape[:-1])}")
        p_z = resets.data_ptr()
    return _f32("lam", lam, (D,), dev), _f32("h0", h0, (shape[0], D), dev), p_z


def _strides(tensors, names, resets):
    """The (batch, time) strides of the call's tensors with resets' in fourth
    place, or None where all are dense in [B, T, D] order."""
    for t in tensors:
        if not t.is_contiguous():
            break
    else:
        if resets is None or resets.is_contiguous():
            return None
    st = []
    for i, t in enumerate(tensors):
        if i == 3:
            st += (0, 0) if resets is None else resets.stride()
        st += _bt(names[i], t)
    return (C.c_int64 * len(st))(*st)


def gated_scan(x, rec, inp, lam, h0=None, resets=None, c: float = 8.0, save: bool = False,
               out=None):
    """A gated linear recurrence over the time axis of [B, T, D] tensors.

    With rate = c softplus(lam):
        a_t = exp(-rate sigmoid(rec_t)), 0 where resets_t is set
        h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(inp_t) x_t
    from h_{-1} = h0 (float32 [B, D]; zeros by default).  ``resets`` (uint8 or
    bool [B, T]) marks the steps at which an episode begins; a step's mark is
    the ``done`` of the step before it.  Several recordings laid end to end in
    one row are marked the same way.  x, rec and inp may be slices of one
    projection's output and in any order of batch and time.

    Returns (h, h_last): h in x's type, h_last float32 [B, D].  With ``save``
    also the carry that ``gated_scan_grad`` takes."""
    if x.dim() != 3:
        raise _invalid(f"x: {x.dim()} axes, expected [B, T, D]")
    dt, dev, shape = _dtype(x), x.device, x.shape
    p_lam, p_h0, p_z = _scan_inputs(x, rec, inp, lam, h0, resets, shape, dev)
    B, T, D = shape
    if out is None:
        out = _like(x)
    else:
        _same("out", out, shape, x.dtype, dev)
    last = lam.new_empty((B, D)) if h0 is None else torch.empty_like(h0)
    carry = lam.new_empty((B, max(T - 1, 0) // 8, D)) if save else None
    ws, p_ws, nw = _workspace("zrl_gated_scan_workspace", lam, B, T, D)
    st = _strides((x, rec, inp, out), ("x", "rec", "inp", "out"), resets)
    _call(N.lib().zrl_gated_scan, dev, x.data_ptr(), rec.data_ptr(), inp.data_ptr(), p_lam,
          p_h0, p_z, B, T, D, dt, c, st, out.data_ptr(), last.data_ptr(),
          carry.data_ptr() if save else None, p_ws, nw)
    return (out, last, carry) if save else (out, last)


def gated_step(x, rec, inp, lam, state, resets=None, c: float = 8.0, out=None):
    """One step of ``gated_scan`` for a rollout: x, rec, inp [B, D], state
    float32 [B, D], resets [B].  Returns (h, new state); ``out=state`` updates
    the state in place."""
    if x.dim() != 2:
        raise _invalid(f"x: {x.dim()} axes, expected [B, D]")
    dt, dev, shape = _dtype(x), x.device, x.shape
    if state is None:
        raise _invalid("state: a float32 tensor [B, D]")
    p_lam, p_h0, p_z = _scan_inputs(x, rec, inp, lam, state, resets, shape, dev)
    B, D = shape
    dense = x.is_contiguous()
    h = torch.empty_like(x) if dense else _dense_like(x)
    if out is None:
        out = torch.empty_like(state)
        p_out = out.data_ptr()
    else:
        p_out = _f32("out", out, shape, dev)
    st = None
    if not (dense and rec.is_contiguous() and inp.is_contiguous() and
            (resets is None or resets.is_contiguous())):
        if D > 1 and (x.stride(1) != 1 or rec.stride(1) != 1 or inp.stride(1) != 1):
            raise _invalid("x, rec, inp: the last axis is not dense")
        z = resets.stride(0) if resets is not None else 0
        st = (C.c_int64 * 10)(x.stride(0), 0, rec.stride(0), 0, inp.stride(0), 0, z, 0, D, 0)
    _call(N.lib().zrl_gated_scan, dev, x.data_ptr(), rec.data_ptr(), inp.data_ptr(), p_lam,
          p_h0, p_z, B, 1, D, dt, c, st, h.data_ptr(), p_out, None, None, 0)
    return h, out


def gated_scan_grad(x, rec, inp, lam, dh, carry, dh_last=None, h0=None, resets=None,
                    c: float = 8.0, out=None):
    """The gradient of ``gated_scan`` for dh on h and dh_last on h_last.

    ``carry`` is what the forward call with ``save`` returned; the other
    arguments are that call's.  Returns (dx, drec, dinp, dlam, dh0), dh0 None
    without h0.  ``out``: three tensors for dx, drec and dinp, such as slices
    of one buffer for the projection's gradient."""
    if x.dim() != 3:
        raise _invalid(f"x: {x.dim()} axes, expected [B, T, D]")
    dt, dev, shape = _dtype(x), x.device, x.shape
    p_lam, p_h0, p_z = _scan_inputs(x, rec, inp, lam, h0, resets, shape, dev)
    B, T, D = shape
    _same("dh", dh, shape, x.dtype, dev)
    p_dl = _f32("dh_last", dh_last, (B, D), dev)
    p_c = _f32("carry", carry, (B, max(T - 1, 0) // 8, D), dev)
    if out is None:
        out = _like(x), _like(x), _like(x)
    else:
        for name, t in zip(("dx", "drec", "dinp"), out, strict=True):
            _same(name, t, shape, x.dtype, dev)
    dx, drec, dinp = out
    dlam = torch.empty_like(lam)
    dh0 = None if h0 is None else torch.empty_like(h0)
    ws, p_ws, nw = _workspace("zrl_gated_scan_grad_workspace", lam, B, T, D)
    st = _strides((x, rec, inp, dh, dx, drec, dinp),
                  ("x", "rec", "inp", "dh", "dx", "drec", "dinp"), resets)
    _call(N.lib().zrl_gated_scan_grad, dev, x.data_ptr(), rec.data_ptr(), inp.data_ptr(), p_lam,
          p_h0, p_z, p_c, dh.data_ptr(), p_dl, B, T, D, dt, c, st, dx.data_ptr(),
          drec.data_ptr(), dinp.data_ptr(), dlam.data_ptr(),
          None if dh0 is None else dh0.data_ptr(), p_ws, nw)
    return dx, drec, dinp, dlam, dh0


def _nl(name, t):
    """(n, l) strides of channels-last [N, ..., C], the middle axes as one."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise _invalid(f"{name}: the last axis is not dense")
    if t.dim() == 2:
        return t.stride(0), t.shape[1]
    if t.dim() == 3:
        return t.stride(0), t.stride(1)
    try:
        v = t.view(t.shape[0], -1, t.shape[-1])
    except RuntimeError:
        raise _invalid(f"{name}: the middle axes do not merge into one") from None
    return v.stride(0), v.stride(1)


def _norm_shape(x, groups, act):
    """(dtype, N, L, C, act) of a group-norm call."""
    if x.dim() < 2:
        raise _invalid("x: [N, C] or [N, ..., C]")
    dt, Cn = _dtype(x), x.shape[-1]
    if groups < 1 or Cn % groups:
        raise _invalid(f"{Cn} channels in {groups} groups")
    if act not in ACTIVATIONS:
        raise _invalid(f"activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    L = 1
    for n in x.shape[1:-1]:
        L *= n
    return dt, x.shape[0], L, Cn, ACTIVATIONS[act]


def _norm_strides(tensors, names):
    for t in tensors:
        if not t.is_contiguous():
            break
    else:
        return None
    if not tensors[0].numel():
        return None
    st = [v for name, t in zip(names, tensors) for v in _nl(name, t)]
    return (C.c_int64 * len(st))(*st)


def group_norm(x, groups: int, gamma=None, beta=None, act: str = "elu", eps: float = 1e-5,
               save: bool = False, out=None):
    """Group norm over channels-last x [N, ..., C] and an activation.

    Each n and each of ``groups`` groups of neighbouring channels is
    normalized over its channels and all middle axes; [N, C] normalizes each
    row by itself, which is the form for time steps (nothing of a later step
    reaches an earlier one).  gamma, beta: float32 [C] or None.  ``act`` is one
    of ``ACTIVATIONS``.  ``out`` may be x.  Returns y, and with ``save`` also
    (mean, rstd), float32 [N, groups]."""
    dt, n, L, Cn, a = _norm_shape(x, groups, act)
    dev = x.device
    p_g, p_b = _f32("gamma", gamma, (Cn,), dev), _f32("beta", beta, (Cn,), dev)
    if out is None:
        out = _dense_like(x)
    else:
        _same("out", out, x.shape, x.dtype, dev)
    f32 = gamma if gamma is not None else x if dt == 0 else None
    if save:
        if f32 is None:
            mean = torch.empty((n, groups), dtype=_F32, device=dev)
        else:
            mean = f32.new_empty((n, groups))
        rstd = torch.empty_like(mean)
        p_m, p_r = mean.data_ptr(), rstd.data_ptr()
    else:
        p_m = p_r = None
    p_ws, nw = None, 0
    if x.numel():
        if f32 is None and _bytes("zrl_group_norm_workspace", n, L, Cn, groups, 0):
            f32 = mean if save else torch.empty(0, dtype=_F32, device=dev)
        ws, p_ws, nw = _workspace("zrl_group_norm_workspace", f32, n, L, Cn, groups, 0)
    _call(N.lib().zrl_group_norm, dev, x.data_ptr(), p_g, p_b, n, L, Cn, groups, dt, a, eps,
          _norm_strides((x, out), ("x", "out")), out.data_ptr(), p_m, p_r, p_ws, nw)
    return (out, mean, rstd) if save else out


def group_norm_grad(x, dy, groups: int, gamma, beta, mean, rstd, act: str = "elu", out=None):
    """The gradient of ``group_norm`` for dy: (dx, dgamma, dbeta).  mean and
    rstd are the forward call's; ``out`` (for dx) may be dy."""
    dt, n, L, Cn, a = _norm_shape(x, groups, act)
    dev = x.device
    _same("dy", dy, x.shape, x.dtype, dev)
    p_g, p_b = _f32("gamma", gamma, (Cn,), dev), _f32("beta", beta, (Cn,), dev)
    p_m, p_r = _f32("mean", mean, (n, groups), dev), _f32("rstd", rstd, (n, groups), dev)
    if out is None:
        out = _dense_like(x)
    else:
        _same("out", out, x.shape, x.dtype, dev)
    dgamma = mean.new_empty(Cn) if gamma is None else torch.empty_like(gamma)
    dbeta = torch.empty_like(dgamma)
    ws, p_ws, nw = _workspace("zrl_group_norm_workspace", mean, n, L, Cn, groups, 1)
    _call(N.lib().zrl_group_norm_grad, dev, x.data_ptr(), dy.data_ptr(), p_g, p_b, p_m, p_r, n, L,
          Cn, groups, dt, a, _norm_strides((x, dy, out), ("x", "dy", "out")), out.data_ptr(),
          dgamma.data_ptr(), dbeta.data_ptr(), p_ws, nw)
    return out, dgamma, dbeta


def dropout(x, p: float, seed: int, stream: int = 0, rows=None, residual=None, out=None):
    """residual + x * keep / P(keep) over the last axis's rows.

    The mask is a function of (seed, stream, row number, column), drawn anew
    by every call and never stored: ``seed`` is a 64-bit key, ``stream`` a
    32-bit number that keeps the uses of one seed apart (a layer, an epoch).
    ``rows`` (int64, one per row) numbers the rows; by default they count
    from 0.  A minibatch that passes its samples' numbers meets the masks of
    the rollout that passed the same numbers, whatever the shuffle.  p is
    taken to the nearest 1/65536.  ``out`` may be ``x`` or ``residual``."""
    if x.dim() == 0:
        raise _invalid("x: at least one axis")
    if not 0 <= stream < 1 << 32:
        raise _invalid("stream: a 32-bit number")
    if not 0 <= seed < 1 << 64:
        raise _invalid("seed: a 64-bit number")
    dt, D = _dtype(x), x.shape[-1]
    if residual is not None:
        _same("residual", residual, x.shape, x.dtype, x.device)
    if out is None:
        out = _dense_like(x)
    else:
        _same("out", out, x.shape, x.dtype, x.device)
    n = x.numel() // D if D else 0
    if rows is not None:
        if rows.dtype != torch.int64 or rows.device != x.device or not rows.is_contiguous():
            raise TypeError("rows: a contiguous int64 tensor on x's device")
        if D and rows.numel() != n:
            raise _invalid(f"rows: {rows.numel()} numbers for {n} rows")
    strides = None
    if n and not (x.is_contiguous() and out.is_contiguous() and
                  (residual is None or residual.is_contiguous())):
        strides = (C.c_int64 * 3)(*(D if t is None else _row_stride(name, t, D) for name, t in
                                    (("x", x), ("residual", residual), ("out", out))))
    _call(N.lib().zrl_dropout, x.device, x.data_ptr(),
          None if residual is None else residual.data_ptr(),
          None if rows is None else rows.data_ptr(), n, D, dt, p, seed, stream, strides,
          out.data_ptr())
    return out


def dropout_grad(dy, p: float, seed: int, stream: int = 0, rows=None, out=None):
    """The gradient of ``dropout`` with respect to x: dy under the same mask
    (the residual's gradient is dy itself)."""
    return dropout(dy, p, seed, stream, rows=rows, out=out)

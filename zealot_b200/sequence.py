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

import torch

from . import native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _invalid(msg: str):
    return N.ZrlError(N.INVALID_ARG, msg)


def _dtype(x) -> int:
    if not x.is_cuda:
        raise TypeError(f"tensor on {x.device}: these operators take CUDA tensors")
    try:
        return _DTYPES[x.dtype]
    except KeyError:
        raise TypeError(f"element type {x.dtype}: float32, bfloat16 or float16") from None


def _call(fn, device, *args):
    """fn(*args, stream) on the device's current stream."""
    if torch.cuda.current_device() == device.index:
        status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if status != N.OK:
        raise N.ZrlError(status, N.lib().zrl_last_error(None).decode())


def _same(name, t, shape, dtype, device):
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name}: {t.dtype} on {t.device}, expected {dtype} on {device}")
    if tuple(t.shape) != tuple(shape):
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
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _same("out", out, x.shape, x.dtype, x.device)
    n = x.numel() // D if D else 0
    if rows is not None:
        if rows.dtype != torch.int64 or rows.device != x.device or not rows.is_contiguous():
            raise TypeError("rows: a contiguous int64 tensor on x's device")
        if D and rows.numel() != n:
            raise _invalid(f"rows: {rows.numel()} numbers for {n} rows")
    strides = None
    if n:
        st = [D if t is None or t.is_contiguous() else _row_stride(name, t, D)
              for name, t in (("x", x), ("residual", residual), ("out", out))]
        strides = None if st == [D, D, D] else (C.c_int64 * 3)(*st)
    _call(N.lib().zrl_dropout, x.device, x.data_ptr(),
          None if residual is None else residual.data_ptr(),
          None if rows is None else rows.data_ptr(), n, D, dt, p, seed, stream, strides,
          out.data_ptr())
    return out


def dropout_grad(dy, p: float, seed: int, stream: int = 0, rows=None, out=None):
    """The gradient of ``dropout`` with respect to x: dy under the same mask
    (the residual's gradient is dy itself)."""
    return dropout(dy, p, seed, stream, rows=rows, out=out)

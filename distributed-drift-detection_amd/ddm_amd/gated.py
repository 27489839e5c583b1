"""Gated linear recurrence over ragged sequences: h_t = a_t h_{t-1} + b_t, a channel apart.

The scans (`kernels.scan_streams` and its relatives) carry a detector along streams of error
flags; this carries a decaying state along streams of numbers.  With scale "ewma" the state is the
exponentially weighted chart of a stream of scores (`tokens.token_scores`' log probabilities or
entropies), with a gate a row, so that a row can also forget everything (log gate -inf); with
"none" and "unit" it is a recurrent layer's state, and `gated_scan_grad` its backward pass.
`gated_step` continues every sequence by one row.

Calls are asynchronous on `stream` (default: the current stream of the inputs' device), read
nothing back and can be captured; results do not change from run to run.  They carry no autograd history,
whether the inputs require a gradient or not.
"""
import torch

from ._capi import check, lib
from ._launch import DTYPES, dense, launch_on, overlap, rows_of, scratch_for, shaped, written
from .kernels import _evs, _ptr

SCALES = {"none": 0, "ewma": 1, "unit": 2}
FILL, H_F32 = 1, 2


def _h_type(name, t, x):
    """Flag of an h of x's type or float32."""
    if t not in (x.dtype, torch.float32):
        raise TypeError(f"{name} has type {t}; supported: {x.dtype} (x's) or torch.float32")
    return H_F32 if t == torch.float32 else 0


def _scale(scale):
    if scale not in SCALES:
        raise ValueError(f"scale must be one of {', '.join(SCALES)}, got {scale!r}")
    return SCALES[scale]


def _inputs(x, log_a):
    """rows, channels, gates and the two row strides."""
    ld_x = rows_of("x", x)
    rows, d = x.shape
    if not 1 <= d <= 1 << 20:
        raise ValueError(f"x has {d} channels (1..{1 << 20})")
    if isinstance(log_a, torch.Tensor) and log_a.dim() == 2 and log_a.shape[0] > 1 and log_a.stride(0) == 0:
        rows_of("log_a", log_a[:1])                     # one row of gates for all rows
        ld_a = 0
    else:
        ld_a = rows_of("log_a", log_a)
    if log_a.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"log_a has type {log_a.dtype}; supported: {x.dtype} (x's) or torch.float32")
    if log_a.shape[0] != rows or log_a.shape[1] < 1 or d % log_a.shape[1]:
        raise ValueError(f"log_a must be [{rows}, gates] with gates dividing {d}, got {list(log_a.shape)}")
    return rows, d, log_a.shape[1], ld_x, ld_a


def _sequences(offsets, state, name, d):
    """How many sequences there are."""
    if offsets is None:
        n = 1
    else:
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() < 1 or \
                offsets.dtype != torch.int64:
            raise ValueError("offsets must be an int64 tensor [sequences + 1]")
        n = offsets.numel() - 1
    if state is not None:
        shaped(name, state, (n, d), torch.float32)
    return n


def gated_scan(x, log_a, offsets=None, state=None, scale="none", out=None, stream=None, timer=None, dtype=None):
    """h [rows, d] (x's type) and the state after every sequence [n, d] (float32) of
    h_t = exp(log_a_t) h_{t-1} + b_t, b = x ("none"), (1 - a) x ("ewma") or sqrt(1 - a^2) x ("unit").

    x [rows, d] float32, bfloat16 or float16; log_a [rows, gates] of x's type or float32, channel c
    using gate c // (d // gates), at most 0 (a gate over 1 counts as NaN); rows contiguous, with a row stride
    (log_a's may be 0: expanded) up to 500 KB, or 15 MB from 128 channels on: the rows that one workgroup holds
    lie within 2 GB.
    offsets int64 [n + 1] on the device, not decreasing: sequence s is rows offsets[s] ..
    offsets[s+1] - 1 (None: one sequence of all rows).  state [n, d] float32: before the first rows
    (None: 0).  Rows of no sequence are zero in a new h and left alone in a given `out`, which
    may be x itself.  dtype (or out's): torch.float32 keeps h as it was computed, which gated_scan_grad makes the
    gates' gradients of; None is x's type, and half the bytes of 16-bit inputs' h.  NaN and infinities stay within
    their sequence and channel, where what follows an infinite state is infinite or NaN (its gates' product may be 0)."""
    rows, d, gates, ld_x, ld_a = _inputs(x, log_a)
    mode = _scale(scale)
    n = _sequences(offsets, state, "state", d)
    dtype = dtype or (x.dtype if out is None else out.dtype)
    flags = _h_type("h", dtype, x) | (FILL if out is None else 0)
    if out is not None:
        ld_out = rows_of("out", out)
        if out.shape != x.shape or out.dtype != dtype:
            raise ValueError(f"out must be {dtype} {list(x.shape)}, got {out.dtype} {list(out.shape)}")
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride() and out.dtype == x.dtype
        for t in (x, log_a, offsets, state):
            if t is not None and overlap(out, t) and not (t is x and same):
                raise ValueError("out overlaps an input without being x")
    else:
        ld_out = d
    context, s = launch_on(x, stream, (x, log_a, offsets, state, out))
    with context:
        offsets, state = dense(offsets), dense(state)
        h = torch.empty((rows, d), dtype=dtype, device=x.device) if out is None else out
        after = torch.empty((n, d), dtype=torch.float32, device=x.device)
        scratch = scratch_for(x.device, "ddm_gated_scan_scratch_bytes", rows, d, gates, DTYPES[x.dtype], 0)
        check(lib.ddm_gated_scan(x.data_ptr(), DTYPES[x.dtype], ld_x, log_a.data_ptr(), DTYPES[log_a.dtype], ld_a, rows,
                                 d, gates, _ptr(offsets), n, mode, _ptr(state), after.data_ptr(), h.data_ptr(), ld_out,
                                 flags, _ptr(scratch), s, *_evs(timer)), "ddm_gated_scan")
    written(out)
    return h, after


def gated_scan_grad(x, log_a, h, d_h, offsets=None, state=None, d_state=None, scale="none", stream=None, timer=None):
    """Gradients of a gated_scan that returned h (x's type, or float32: see there): (d_x like x, d_log_a like log_a but dense, the
    gradient of `state` [n, d] float32) from d_h [rows, d] (x's type) and d_state [n, d] float32, the
    gradient of the state after (None: 0).  Rows of no sequence have gradient 0.  At a = 1 the
    "unit" factor's infinite slope counts as 0."""
    rows, d, gates, ld_x, ld_a = _inputs(x, log_a)
    mode = _scale(scale)
    n = _sequences(offsets, state, "state", d)
    strides = []
    for name, t in (("h", h), ("d_h", d_h)):
        strides.append(rows_of(name, t))
        if t.shape != x.shape or t.dtype not in (x.dtype, torch.float32 if name == "h" else x.dtype):
            raise ValueError(f"{name} must be {x.dtype} {list(x.shape)}, got {t.dtype} {list(t.shape)}")
    flags = _h_type("h", h.dtype, x) | FILL
    if d_state is not None:
        shaped("d_state", d_state, (n, d), torch.float32)
    context, s = launch_on(x, stream, (x, log_a, h, d_h, offsets, state, d_state))
    with context:
        offsets, state, d_state = dense(offsets), dense(state), dense(d_state)
        d_x = torch.empty((rows, d), dtype=x.dtype, device=x.device)
        d_a = torch.empty((rows, gates), dtype=log_a.dtype, device=x.device)
        before = torch.empty((n, d), dtype=torch.float32, device=x.device)
        scratch = scratch_for(x.device, "ddm_gated_scan_scratch_bytes", rows, d, gates, DTYPES[x.dtype], 1)
        check(lib.ddm_gated_scan_grad(x.data_ptr(), DTYPES[x.dtype], ld_x, log_a.data_ptr(), DTYPES[log_a.dtype], ld_a,
                                      h.data_ptr(), strides[0], d_h.data_ptr(), strides[1], rows, d, gates,
                                      _ptr(offsets), n, mode, _ptr(state), _ptr(d_state), before.data_ptr(),
                                      d_x.data_ptr(), d, d_a.data_ptr(), gates, flags, _ptr(scratch), s, *_evs(timer)),
              "ddm_gated_scan_grad")
    return d_x, d_a, before


def gated_step(x, log_a, state=None, scale="none", out_state=None, stream=None, timer=None):
    """One row of every sequence: row s of x [n, d] and log_a [n, gates] (as gated_scan's) continues state[s]
    (float32, None: 0).  Returns (h in x's type, the state after); out_state may be `state` itself, and lies apart
    from x and log_a."""
    rows, d, gates, ld_x, ld_a = _inputs(x, log_a)
    mode = _scale(scale)
    for name, t in (("state", state), ("out_state", out_state)):
        if t is not None:
            shaped(name, t, (rows, d), torch.float32)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    if state is not None and out_state is not None and state.data_ptr() != out_state.data_ptr() and \
            overlap(state, out_state):
        raise ValueError("out_state overlaps the state without being it")
    context, s = launch_on(x, stream, (x, log_a, state, out_state))
    with context:
        h = torch.empty((rows, d), dtype=x.dtype, device=x.device)
        after = torch.empty((rows, d), dtype=torch.float32, device=x.device) if out_state is None else out_state
        check(lib.ddm_gated_step(x.data_ptr(), DTYPES[x.dtype], ld_x, log_a.data_ptr(), DTYPES[log_a.dtype], ld_a, rows,
                                 d, gates, mode, _ptr(state), after.data_ptr(), h.data_ptr(), d, s, *_evs(timer)),
              "ddm_gated_step")
    written(out_state)
    return h, after

"""Checks and launches that the language-model operators share.

A call on small operands costs the host more than the GPU, so the common case (the current
stream of the current device) takes no context manager and makes no Stream object.
"""
import ctypes
import functools

import torch

from ._capi import check, lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _Here:
    """The current stream of the current device: nothing to enter."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_here = _Here()


def launch_on(t, stream, inputs):
    """(context, stream address): what is allocated inside the context belongs to the stream
    (None: the current one of t's device), and inputs stay alive for it."""
    device = t.device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on the GPU, got {device}")
    for x in inputs:
        if x is not None and x.device != device:
            raise ValueError(f"tensors on {device} and on {x.device}")
    if stream is None and _raw_stream is not None and device.index == torch.cuda.current_device():
        return _here, _raw_stream(device.index)
    current = torch.cuda.current_stream(device)
    if stream is None:
        stream = current
    if stream.device != device:
        raise ValueError(f"stream of {stream.device}, tensors on {device}")
    if stream != current:
        for x in inputs:
            if x is not None:
                x.record_stream(stream)
    return torch.cuda.stream(stream), stream.cuda_stream    # also makes the stream's device the current one


@functools.lru_cache(maxsize=256)
def scratch_bytes(name, *sizes):
    """Bytes of scratch that the C-ABI's `name` asks for."""
    return int(getattr(lib, name)(*sizes))


def scratch_for(device, name, *sizes):
    need = scratch_bytes(name, *sizes)
    return torch.empty(need, dtype=torch.uint8, device=device) if need else None


def rows_of(name, t, dtypes=DTYPES):
    """The row stride of a matrix whose rows are contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}; supported: {', '.join(str(d) for d in dtypes)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous (strides {t.stride()})")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1]:
        raise ValueError(f"{name}'s rows overlap (strides {t.stride()})")
    return ld


def shaped(name, t, shape, *dtypes):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)} {list(shape)}, got {t.dtype} "
                         f"{list(t.shape)}")


def dense(t):
    """`t` without gaps (a copy on the launch stream if it has any)."""
    return None if t is None else t.contiguous()


def written(t):
    """The caller's `t` was overwritten: autograd refuses a backward pass that saved what it held."""
    if t is not None and not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _span(t):
    if t.is_contiguous():
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    if a.dim() == 2 and b.dim() == 2 and a.stride(1) == 1 and b.stride(1) == 1:
        row = a.stride(0) * a.element_size()
        if row > 0 and row == b.stride(0) * b.element_size():       # columns of one buffer
            apart, wide_a, wide_b = (b0 - a0) % row, a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
            return apart < wide_a or apart + wide_b > row
    return True


def wait_gave_up(device=None):
    """Whether a wait of one workgroup for another has given up on the device (None: the current one) since this was last
    asked: no, unless something kept part of a launch from running for seconds.  Such a wait leaves NaN in the results of
    `topk_distill` (with a gradient), `gated_scan` or `gated_scan_grad`; this tells it from a NaN of the inputs'.
    Waits for the device's work so far."""
    gave_up = ctypes.c_int32()
    with torch.cuda.device(device):
        check(lib.ddm_wait_gave_up(ctypes.byref(gave_up)), "ddm_wait_gave_up")
    return bool(gave_up.value)

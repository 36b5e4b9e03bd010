"""Device-memory plumbing via PyTorch-ROCm (allocation and streams only)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch


def require_cuda(t: torch.Tensor, dtype, name: str, ndim: int | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise TypeError(f"{name} must be a torch tensor on a ROCm device")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D")
    return t.contiguous()


def require_aligned(t: torch.Tensor, dtype, name: str, ndim: int, device=None) -> torch.Tensor:
    """require_cuda, and a copy where the rows start off a 16-byte border (a
    slice of a larger tensor); device: where the call's other tensors are."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype and t.dim() == ndim:
        if not t.is_contiguous():
            t = t.contiguous()
    else:
        t = require_cuda(t, dtype, name, ndim)
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, other tensors of the call on {device}")
    return t if t.data_ptr() % 16 == 0 else t.clone()


def enqueues(fn):
    """For calls that return before their work is done: on_device, and with
    `stream` given it is the current stream inside, so that what is allocated
    belongs to it, and the inputs' memory is kept until its work on them is done."""
    import functools

    @functools.wraps(fn)
    def wrapped(*args, stream=None, **kwargs):
        dev = _first_cuda(args, kwargs)
        if stream is None:
            if dev is None or dev.index == torch.cuda.current_device():
                return fn(*args, **kwargs)
            with torch.cuda.device(dev):
                return fn(*args, **kwargs)
        if dev is not None and dev != stream.device:
            raise ValueError(f"stream is on {stream.device}, the call's tensors on {dev}")
        with torch.cuda.stream(stream):
            for a in (*args, *kwargs.values()):
                for t in (a, getattr(a, "codes", None), getattr(a, "scale", None)):
                    if isinstance(t, torch.Tensor) and t.is_cuda:
                        t.record_stream(stream)
            return fn(*args, **kwargs)
    return wrapped


def raw_stream(t: torch.Tensor) -> int:
    """The handle of the current stream of t's device."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def ptr(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def stream_handle(stream=None) -> C.c_void_p:
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def to_device(a, device="cuda") -> torch.Tensor:
    if isinstance(a, torch.Tensor):
        return a.to(device).contiguous()
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


def _first_cuda(args, kwargs):
    for a in (*args, *kwargs.values()):
        if isinstance(a, torch.Tensor) and a.is_cuda:
            return a.device
        for v in (getattr(a, "indptr", None), getattr(a, "keys", None), getattr(a, "codes", None)):
            if isinstance(v, torch.Tensor) and v.is_cuda:
                return v.device
    return None


def on_device(fn):
    """Run a wrapper with its first device tensor's GPU current, so the
    library's launches, scratch and the default stream (the current stream of
    that device) all land on the device that holds the data."""
    import functools

    @functools.wraps(fn)
    def wrapped(*args, **kwargs):
        dev = _first_cuda(args, kwargs)
        if dev is None or dev.index is None or dev.index == torch.cuda.current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(dev):
            return fn(*args, **kwargs)
    return wrapped

"""Device-side helpers for the host layer: small table uploads through a
pinned ring, the CUDA stream handle, and dtype checks.  PyTorch is used only
for device memory and streams."""
from __future__ import annotations

import contextlib
import ctypes
import threading

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib as L


def require_cuda_tensor(t: torch.Tensor, what: str):
    if not t.is_cuda:
        raise NotImplementedError(f"{what}: tensors must live on a CUDA device (no CPU fallback)")
    if t.is_sparse:
        raise NotImplementedError(f"{what}: sparse gradients are not supported")
    if not t.is_contiguous():
        raise NotImplementedError(f"{what}: tensors must be contiguous")


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return 0
    if dt == torch.bfloat16:
        return 1
    raise NotImplementedError(f"parameter dtype {dt} is not supported (float32 and bfloat16 are)")


def as_float32(v: float) -> float:
    """v as the kernels get it; infinite beyond float32."""
    return ctypes.c_float(v).value


def refuse_tangents(what: str, *tensors):
    """Raises for dual tensors: kernels that are launched outside an autograd
    function would lose their tangents without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode derivatives are not supported")


def stream_handle(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t) -> int:
    return 0 if t is None else int(t.data_ptr())


def aligned16(*ts) -> bool:
    return all(t is None or (t.data_ptr() % 16 == 0) for t in ts)


class DeviceTable:
    """A device buffer refreshed from host bytes each step.  Uploads go
    through a ring of pinned host buffers; a slot is reused only after the
    copy that last read it has completed (an event per slot)."""

    def __init__(self, nbytes: int, device, ring: int = 2):
        self.nbytes = int(nbytes)
        self.device = device
        self.dev = torch.empty(max(1, self.nbytes), dtype=torch.uint8, device=device)
        self.host = [torch.empty(max(1, self.nbytes), dtype=torch.uint8, pin_memory=True) for _ in range(ring)]
        self.events = [None] * ring
        self.slot = 0

    @property
    def ptr(self) -> int:
        return int(self.dev.data_ptr())

    def upload(self, arr: np.ndarray):
        b = arr.view(np.uint8).reshape(-1)
        assert b.size <= self.nbytes
        i = self.slot
        self.slot = (i + 1) % len(self.host)
        if self.events[i] is not None:
            self.events[i].synchronize()
        h = self.host[i]
        h.numpy()[: b.size] = b
        self.dev[: b.size].copy_(h[: b.size], non_blocking=True)
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(self.device))
        self.events[i] = ev


def upload_static(arr: np.ndarray, device) -> torch.Tensor:
    """One-off upload of a table that does not change between steps."""
    b = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
    t = torch.from_numpy(b.copy())
    return t.to(device)


def raw_stream(device) -> int:
    """The current stream of `device`, as the C entry points take it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


_HERE = contextlib.nullcontext()


def on_device(device):
    """A context in which `device` is the current one (free when it is already)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


class ErrorWord:
    """The word that a kernel sets when something is wrong that only the device
    sees (a bounded wait that gave up, an index outside its table): pinned host
    memory that the kernels write directly, so that every call can look at it
    without waiting for the GPU.  One for the process: whichever thread's call
    comes next reports it, for whichever device."""

    def __init__(self, message="an earlier kernel reported an error"):
        self.message = message
        self.word = self.view = None
        self.devices = set()   # whose kernels may set it
        self.lock = threading.Lock()

    def pointer(self, device=None) -> int:
        """For a launch on `device`."""
        if self.word is None:
            if torch.cuda.is_current_stream_capturing():
                return 0   # no allocation of pinned memory during a capture
            with self.lock:
                if self.word is None:
                    word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
                    self.view = word.numpy()   # before the word, which other threads find without the lock
                    self.word = word
        if self.view[0]:
            self.raise_()
        if device is not None:
            self.devices.add(device)
        return self.word.data_ptr()

    def raise_(self):
        self.view[0] = 0
        raise L.AdvOptError(self.message)

    def check(self):
        """Waits for the GPUs that may report, whichever is the current one, and raises what they reported."""
        for device in list(self.devices):
            torch.cuda.synchronize(device)
        if self.word is not None and self.view[0]:
            self.raise_()


def saved(t, what, dtype, shape, device):
    """A saved tensor as the backward pass gets it, contiguous: a hook on saved tensors may have given another one."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        raise RuntimeError(f"a hook on saved tensors gave {t.dtype} {tuple(t.shape)} on {t.device} for the {what}, "
                           f"{dtype} {tuple(shape)} on {device} was saved")
    return t.contiguous()


def empty_as(t):
    """A new contiguous tensor of t's shape and dtype (`empty_like`, the cheapest of torch's calls, keeps other orders of dimensions too)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def rows_of(t):
    """(t, pitch) of a matrix whose rows the kernels may read as they lie; a copy where their elements are not consecutive or rows overlap."""
    if t.is_contiguous():
        return t, t.shape[1]
    (R, C), (pitch, one) = t.shape, t.stride()
    if (C > 1 and one != 1) or (R > 1 and pitch < C):
        return t.contiguous(), C
    return t, pitch if R > 1 else C

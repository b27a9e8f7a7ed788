"""Host plumbing shared by the operator wrappers: dtype codes, streams, workspaces.

PyTorch only supplies device memory and the current CUDA stream here; every kernel
runs from libjetspec_b200.so through the C ABI.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib

DTYPE_CODES = {torch.bfloat16: _lib.JT_BF16, torch.float16: _lib.JT_F16,
               torch.float32: _lib.JT_F32}

_workspaces: dict = {}  # (device index, stream) -> _Workspace


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(device: torch.device) -> int:
    """cudaStream_t (as an int) of the caller's current stream on ``device``, without
    building a torch Stream object (a few microseconds per call saved on the launch path)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(device).cuda_stream


def stream_handle(device: torch.device) -> ctypes.c_void_p:
    """Raw cudaStream_t of the caller's current stream (what Triton launches on)."""
    return ctypes.c_void_p(raw_stream(device))


def remember(sizes: dict, shape: tuple, nbytes: int) -> int:
    """Keeps a launch shape's workspace size, of a bounded number of shapes."""
    if len(sizes) >= 4096:
        sizes.clear()
    return sizes.setdefault(shape, nbytes)


class _Workspace:
    """Scratch of one (device, stream) and the lock that its users hold while they enqueue."""
    __slots__ = ("lock", "buffer", "nbytes")

    def __init__(self):
        self.lock = threading.RLock()
        self.buffer, self.nbytes = None, 0


def with_workspace(device: torch.device, nbytes: int, stream: int, launch):
    """``launch(address)`` with ``nbytes`` of device scratch; returns what it returns.

    Launches on one stream are ordered, so they share one buffer; another stream has its own.
    It grows to the largest request seen, by a quarter at least so that ragged sizes settle
    soon; the smaller one goes back to the allocator, which gives it to later work of the same
    stream only.

    An operator of several kernels hands its state from one to the next through the scratch,
    and the ctypes call that enqueues them gives up the interpreter lock.  The stream's own
    lock, held until all of them are enqueued, keeps another thread's launches on the same
    stream from coming between.  Re-entrant: a finaliser that runs inside completes its own
    launches first.

    A captured call shares nothing: its graph may replay beside other work, on any stream.
    Its scratch is allocated for the call; under torch.cuda.graph (and whatever captures
    through it) that is memory of the graph's own pool, which the allocator hands to later
    calls of the same capture and to nobody else while the graph lives.
    """
    if torch._C._cuda_isCurrentStreamCapturing():
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return launch(scratch.data_ptr())
    key = (device.index, stream)
    held = _workspaces.get(key)
    if held is None:
        held = _workspaces.setdefault(key, _Workspace())
    with held.lock:
        if nbytes > held.nbytes:
            size = max(nbytes, held.nbytes + held.nbytes // 4)
            held.buffer, held.nbytes = None, 0  # freed first: the two need not fit together
            held.buffer = torch.empty(size, dtype=torch.uint8, device=device)
            held.nbytes = size
        buffer = held.buffer  # kept through the launch, whatever a finaliser's call does
        return launch(buffer.data_ptr())


def ptr(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()

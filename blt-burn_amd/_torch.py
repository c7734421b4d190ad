"""Device-memory plumbing: torch CUDA tensors carry the buffers and streams
handed to the C ABI (pointers, element counts, the current HIP stream)."""
import torch
import torch.autograd.forward_ad as _forward_ad

from ._lib import BltError, check


# the raw current-stream handle without building a torch.cuda.Stream object
# (one per call otherwise: about 1.5 us of host time on every launch)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device=None):
    if _raw_stream is not None:
        if isinstance(device, torch.device) and device.index is not None:
            return _raw_stream(device.index)
        if device is None or isinstance(device, int):
            return _raw_stream(torch.cuda.current_device() if device is None else device)
    return torch.cuda.current_stream(device).cuda_stream


# (the same without a lazy initialisation and a Python frame on every call)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def call_on(device, index, fn, what, *args):
    """fn(*args, stream) on `device` (whose index is `index`) and its current stream:
    the library launches on the current device, which may be another one."""
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index) if _raw_stream is not None else stream_ptr(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream_ptr(index))
    if rc:
        check(rc, what)


def require_cuda(*tensors):
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
        if not t.is_cuda:
            raise BltError("tensor must live on a GPU (got device %s)" % t.device)


def no_tangents(what, *tensors):
    """For the calls that autograd follows: forward-mode does not, and a tangent of an input would
    be dropped without a word.  (One comparison where no dual_level is entered.)"""
    if getattr(_forward_ad, "_current_level", 0) >= 0 and any(
            isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None
            for t in tensors):
        raise BltError("%s: forward-mode derivatives are not supported" % what)


def contiguous(t):
    return t if t.is_contiguous() else t.contiguous()


def bf16_bits_to_tensor(arr, device):
    """numpy uint16 bf16 bits -> torch.bfloat16 tensor on `device`."""
    import numpy as np
    return torch.from_numpy(np.ascontiguousarray(arr).view(np.int16)).view(torch.bfloat16).to(device)

"""What the calls of engine.py and linear.py do with their arguments: the current stream, pointers of device
tensors, host arrays of integers."""
from __future__ import annotations

import array

import numpy as np

try:
    import torch
except ImportError:  # the host-only functions need no torch
    torch = None


# A decode step makes two to four of these calls a layer on kernels of 4 to 13 us, so what a call
# costs on the host is the step's time: pointers and streams go to ctypes as plain integers and the
# current stream is asked for as one, not through a Stream object (2.9 us). layer_attention 22.7 ->
# 13.9 us a call (the two C calls alone 7).
_getDevice = getattr(getattr(torch, "_C", None), "_cuda_getDevice", None)
_getRawStream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """The current device's current stream (hipStream_t as an integer)."""
    if _getRawStream is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _getRawStream(_getDevice())


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("bitgpu_amd: expected a device (cuda) tensor")
    if not t.is_contiguous():
        raise ValueError("bitgpu_amd: expected a contiguous tensor")
    return t.data_ptr()


def _f32(t, name):
    if t.dtype is not torch.float32:
        raise TypeError(f"bitgpu_amd: {name} must be float32, got {t.dtype}")
    return t


def _int32(x, name, dims):
    """x (a sequence, array or host tensor of integers) as a contiguous int32 array."""
    if isinstance(x, (list, tuple)) and dims == 1:
        try:  # a list of Python integers, several times faster than through np.asarray
            return np.frombuffer(array.array("i", x), np.int32) if x else np.zeros(0, np.int32)
        except (TypeError, OverflowError):
            pass
    if torch is not None and isinstance(x, torch.Tensor):
        x = x.numpy()
    a = np.asarray(x)
    if a.size == 0 and a.ndim == 1 and dims == 1:
        return np.zeros(0, np.int32)
    if a.ndim != dims or a.dtype.kind not in "iu":
        raise ValueError(f"bitgpu_amd: {name} must hold integers in {dims} dimension{'s' if dims > 1 else ''}")
    if a.dtype != np.int32:
        if a.size and (a.max() > 0x7fffffff or a.min() < -0x80000000):
            raise ValueError(f"bitgpu_amd: {name} exceeds 32 bits")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def _rows_ptr(t, name, rows, width, device):
    """Pointer of an f32 tensor of at least `rows` contiguous rows of `width` values (more: a padded batch)
    on the pool's device; None for None."""
    if t is None:
        return None
    if t.dtype is not torch.float32:
        raise TypeError(f"bitgpu_amd: {name} must be float32, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"bitgpu_amd: expected {name} on cuda:{device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"bitgpu_amd: expected a contiguous tensor ({name})")
    if t.numel() < rows * width:
        raise ValueError(f"bitgpu_amd: {name} holds {t.numel()} values, the batch needs {rows} rows of {width}")
    return t.data_ptr()

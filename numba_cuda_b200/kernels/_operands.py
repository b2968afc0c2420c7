"""Arguments of the head-wise kernels: arrays as (pointer, shape, item strides, format)
and the argument structs of ``include/b2k.h`` as packed bytes.

Arrays are device arrays of this package, torch CUDA tensors (taken as they are: the
CUDA Array Interface has no name for bfloat16 and the fp8 types) or anything else that
exports the CUDA Array Interface; host arrays are copied to the device where they are
only read."""
from __future__ import annotations

import ctypes
import struct

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _lib
from ..api import auto_device, is_cuda_array
from ..devicearray import DeviceNDArray, _torch_stream, bfloat16_dtype, stream_ptr

_Tensor = torch.Tensor
#: Types by torch's names; a torch of fewer types has no tensors of the others.
_TORCH = {getattr(torch, name): fmt for name, fmt in (
    ("float32", _lib.FMT_F32), ("float16", _lib.FMT_F16), ("bfloat16", _lib.FMT_BF16), ("uint16", _lib.FMT_BF16),
    ("uint8", _lib.FMT_U8), ("int32", _lib.FMT_I32), ("int64", _lib.FMT_I64), ("float8_e4m3fn", _lib.FMT_E4M3),
    ("float8_e5m2", _lib.FMT_E5M2), ("float8_e8m0fnu", _lib.FMT_E8M0)) if hasattr(torch, name)}
_NUMPY = {"float32": _lib.FMT_F32, "float16": _lib.FMT_F16, "bfloat16": _lib.FMT_BF16, "uint16": _lib.FMT_BF16,
          "uint8": _lib.FMT_U8, "int32": _lib.FMT_I32, "int64": _lib.FMT_I64, "float8_e4m3fn": _lib.FMT_E4M3,
          "float8_e5m2": _lib.FMT_E5M2, "float8_e8m0fnu": _lib.FMT_E8M0}
INDEX_FORMATS = (_lib.FMT_I64, _lib.FMT_I32)
HEAD_FORMATS = (_lib.FMT_F32, _lib.FMT_F16, _lib.FMT_BF16)

HEADS = struct.Struct("5q")
ROTATION = struct.Struct("13qd12q")
CACHE = struct.Struct("26q")
NO_HEADS = HEADS.pack(0, 0, 0, 0, 0)


def _in_forward_mode() -> bool:
    """Whether a level of forward differentiation is open, where a tensor may carry a tangent."""
    return getattr(forward_ad, "_current_level", 0) != -1


#: An operand is the tuple (pointer, shape, strides in items, format, device, owner); the
#: owner keeps the memory alive until the launch.  Plain tuples, and a first branch for the
#: common argument, because a small call's time is the host's: an attribute of a tensor
#: costs 0.1 us, a named tuple 0.3 us.
def operand(x, what, written=False, stream=0):
    """The description of an array argument named ``what`` in error messages."""
    if isinstance(x, _Tensor):
        fmt = _TORCH.get(x.dtype)
        device = x.get_device()
        if fmt is not None and device >= 0 and not x.requires_grad and not _in_forward_mode():
            return x.data_ptr(), x.shape, x.stride(), fmt, device, x
        if fmt is None:
            raise TypeError(f"{what}: unsupported type {x.dtype}")
        if x.requires_grad:
            raise ValueError(f"{what} requires grad: the call is not recorded for autograd, pass x.detach()")
        if _in_forward_mode() and forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError(f"{what} carries a tangent: the call gives none, pass forward_ad.unpack_dual(x).primal")
        if device >= 0:
            return x.data_ptr(), x.shape, x.stride(), fmt, device, x
        if written:
            raise ValueError(f"{what} must be in device memory")
        with torch.cuda.stream(_torch_stream(stream)):      # its memory goes back in this stream's order
            x = x.cuda()
        return x.data_ptr(), x.shape, x.stride(), fmt, x.get_device(), x
    if not isinstance(x, DeviceNDArray):
        if written and not is_cuda_array(x):
            raise ValueError(f"{what} must be in device memory")
        x, _ = auto_device(x, stream=stream)
    fmt = _NUMPY.get(x.dtype.name)
    if fmt is None:
        raise TypeError(f"{what}: unsupported type {x.dtype}")
    item = x.dtype.itemsize
    strides = x.strides
    if item > 1:
        if any(s % item for s in strides):
            raise ValueError(f"{what}: strides are no multiples of the item size")
        strides = tuple(s // item for s in strides)
    return x._ptr, x.shape, strides, fmt, x._buf.get_device(), x


def heads(x, what, written=False, stream=0):
    """A (tokens, heads, dim) array of floats with unit stride in its last axis."""
    op = operand(x, what, written, stream)
    _, shape, strides, fmt, _, _ = op
    if len(shape) != 3:
        raise ValueError(f"{what} must have the axes (tokens, heads, dim)")
    if fmt not in HEAD_FORMATS:
        raise TypeError(f"{what} must be float32, float16 or bfloat16")
    if strides[2] != 1 and shape[2] > 1:
        raise ValueError(f"{what} must have unit stride in its last axis")
    return op


def pack_heads(op) -> bytes:
    if op is None:
        return NO_HEADS
    ptr, (_, n, dim), (token, head, _), _, _, _ = op
    return HEADS.pack(ptr, token, head, n, dim)


def vector(x, what, length, formats, kind, written=False, stream=0):
    """A contiguous 1-D array of ``length`` items (None: any) of one of ``formats``."""
    op = operand(x, what, written, stream)
    _, shape, strides, fmt, _, _ = op
    if fmt not in formats:
        raise TypeError(f"{what} must be {kind}")
    if len(shape) != 1 or (length is not None and shape[0] != length) or (strides[0] != 1 and shape[0] > 1):
        raise ValueError(f"{what} must be a contiguous 1-D array" + ("" if length is None else f" of {length} items"))
    return op


def indices(x, what, length, stream=0):
    return vector(x, what, length, INDEX_FORMATS, "int32 or int64", False, stream)


def index_bytes(op) -> int:
    return 4 if op[3] == _lib.FMT_I32 else 8


def on_one_device(ops) -> None:
    """Every array on the current device: a kernel is launched there."""
    here = torch.cuda.current_device()
    for op in ops:
        if op is not None and op[4] != here:
            raise ValueError(f"an array is on device {op[4]}, the current device is {here}")


def like(op, stream):
    """A new array of an operand's shape and type."""
    from ..api import device_array
    dtype = {_lib.FMT_F32: np.dtype(np.float32), _lib.FMT_F16: np.dtype(np.float16),
             _lib.FMT_BF16: bfloat16_dtype()}[op[3]]
    return device_array(op[1], dtype, stream=stream)


def _current_stream_ptr() -> int:
    """cudaStream_t of torch's current stream; the object for it would cost 3 us."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(torch.cuda.current_device()) if raw is not None else torch.cuda.current_stream().cuda_stream


def workspace(nbytes, stream):
    """Device memory for one call, from torch's allocator on the call's stream: calls on
    other streams and replays of captured graphs have their own."""
    if _current_stream_ptr() == stream_ptr(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(_torch_stream(stream)):
        return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


def _version_counters():
    """torch's function that raises the version counters of a tuple of tensors."""
    many = getattr(torch._C, "_increment_version", None)
    try:
        many((torch.empty(0, device="cpu"),))
        return many
    except TypeError:                                       # an older torch takes one at a time
        def each(tensors):
            for x in tensors:
                torch.autograd.graph.increment_version(x)
        return each


#: Called for tensors that a call has written through their addresses: autograd then notices
#: that a tensor it saved is not what it was.
_increment_version = _version_counters()


def written(*arrays) -> None:
    """Note that a call has written these arrays (``None`` and arrays of other kinds among them)."""
    tensors = tuple(x for x in arrays if isinstance(x, _Tensor))
    if tensors:
        _increment_version(tensors)


class _NoFast:
    """Stands for the extension where it was not built: every call takes the Python code."""

    @staticmethod
    def _pass(*args):
        return None

    norm_rotate = norm_rotate_backward = cache_write = cache_read = norm_rotate_write = _pass


class _Fast:
    """The extension ``_pyfast``, set up when it is first used (it needs the library)."""

    ENTRIES = ("norm_rotate", "norm_rotate_backward", "cache_write", "cache_read", "norm_rotate_write")

    def __getattr__(self, name):
        if name not in self.ENTRIES:
            raise AttributeError(name)
        try:
            from .. import _pyfast as module
        except ImportError:
            module = _NoFast
        else:
            L = _lib.lib()
            names = ("b2k_norm_rotate", "b2k_norm_rotate_backward_scratch_bytes", "b2k_norm_rotate_backward",
                     "b2k_cache_write", "b2k_cache_read", "b2k_norm_rotate_write", "b2k_current_device")
            module.setup(torch.Tensor, _TORCH, {n: ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in names},
                         stream_ptr, workspace, vars(forward_ad), _increment_version)
        for entry in self.ENTRIES:
            setattr(self, entry, getattr(module, entry))
        return self.__dict__[name]


fast = _Fast()

__all__ = ["operand", "heads", "vector", "indices", "pack_heads", "index_bytes", "on_one_device", "like", "workspace",
           "written", "fast"]

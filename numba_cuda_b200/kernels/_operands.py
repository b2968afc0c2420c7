"""Arguments of the head-wise kernels: arrays as (pointer, shape, item strides, format)
and the argument structs of ``include/b2k.h`` as packed bytes.

Arrays are device arrays of this package, torch CUDA tensors (taken as they are: the
CUDA Array Interface has no name for bfloat16 and the fp8 types) or anything else that
exports the CUDA Array Interface; host arrays are copied to the device where they are
only read."""
from __future__ import annotations

import struct
from typing import NamedTuple

import numpy as np
import torch

from .. import _lib
from ..api import auto_device, is_cuda_array
from ..devicearray import DeviceNDArray, bfloat16_dtype, stream_ptr

#: formats of heads and weights, codes, scales; indices are "i4" / "i8"
_TORCH = {torch.float32: _lib.FMT_F32, torch.float16: _lib.FMT_F16, torch.bfloat16: _lib.FMT_BF16,
          torch.uint16: _lib.FMT_BF16, torch.uint8: _lib.FMT_U8, torch.int32: _lib.FMT_I32, torch.int64: _lib.FMT_I64,
          torch.float8_e4m3fn: _lib.FMT_E4M3, torch.float8_e5m2: _lib.FMT_E5M2, torch.float8_e8m0fnu: _lib.FMT_E8M0}
_NUMPY = {"float32": _lib.FMT_F32, "float16": _lib.FMT_F16, "bfloat16": _lib.FMT_BF16, "uint16": _lib.FMT_BF16,
          "uint8": _lib.FMT_U8, "int32": _lib.FMT_I32, "int64": _lib.FMT_I64, "float8_e4m3fn": _lib.FMT_E4M3,
          "float8_e5m2": _lib.FMT_E5M2, "float8_e8m0fnu": _lib.FMT_E8M0}
HEAD_FORMATS = (_lib.FMT_F32, _lib.FMT_F16, _lib.FMT_BF16)

HEADS = struct.Struct("5q")
ROTATION = struct.Struct("13qd12q")
CACHE = struct.Struct("26q")
NO_HEADS = HEADS.pack(0, 0, 0, 0, 0)


class Operand(NamedTuple):
    ptr: int
    shape: tuple
    strides: tuple        # in items
    format: int
    device: int
    owner: object         # keeps the memory alive until the launch


def operand(x, what, written=False, stream=0) -> Operand:
    """The description of an array argument named ``what`` in error messages."""
    if isinstance(x, torch.Tensor):
        fmt = _TORCH.get(x.dtype)
        if fmt is None:
            raise TypeError(f"{what}: unsupported type {x.dtype}")
        if not x.is_cuda:
            if written:
                raise ValueError(f"{what} must be in device memory")
            x = x.cuda()
        if x.requires_grad:
            raise ValueError(f"{what} requires grad: the call is not recorded for autograd, pass x.detach()")
        return Operand(x.data_ptr(), tuple(x.shape), x.stride(), fmt, x.get_device(), x)
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
    return Operand(x._ptr, x.shape, strides, fmt, x._buf.get_device(), x)


def heads(x, what, written=False, stream=0) -> Operand:
    """A (tokens, heads, dim) array of floats with unit stride in its last axis."""
    op = operand(x, what, written, stream)
    if len(op.shape) != 3:
        raise ValueError(f"{what} must have the axes (tokens, heads, dim)")
    if op.format not in HEAD_FORMATS:
        raise TypeError(f"{what} must be float32, float16 or bfloat16")
    if op.strides[2] != 1 and op.shape[2] > 1:
        raise ValueError(f"{what} must have unit stride in its last axis")
    return op


def pack_heads(op) -> bytes:
    if op is None:
        return NO_HEADS
    return HEADS.pack(op.ptr, op.strides[0], op.strides[1], op.shape[1], op.shape[2])


def indices(x, what, length, stream=0) -> Operand:
    op = operand(x, what, stream=stream)
    if op.format != _lib.FMT_I64 and op.format != _lib.FMT_I32:
        raise TypeError(f"{what} must be int32 or int64")
    if len(op.shape) != 1 or (length is not None and op.shape[0] != length):
        raise ValueError(f"{what} must be a 1-D array" + ("" if length is None else f" of {length} items"))
    if op.shape[0] > 1 and op.strides[0] != 1:
        raise ValueError(f"{what} must be contiguous")
    return op


def index_bytes(op) -> int:
    return 4 if op.format == _lib.FMT_I32 else 8


def on_one_device(ops) -> None:
    """Every array on the current device: a kernel is launched there."""
    here = torch.cuda.current_device()
    for op in ops:
        if op is not None and op.device != here:
            raise ValueError(f"an array is on device {op.device}, the current device is {here}")


def like(op, stream):
    """A new array of an operand's shape and type."""
    from ..api import device_array
    dtype = {_lib.FMT_F32: np.dtype(np.float32), _lib.FMT_F16: np.dtype(np.float16),
             _lib.FMT_BF16: bfloat16_dtype()}[op.format]
    return device_array(op.shape, dtype, stream=stream)


__all__ = ["operand", "heads", "indices", "pack_heads", "index_bytes", "on_one_device", "like", "stream_ptr"]

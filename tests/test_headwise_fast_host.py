"""The extension that makes the head-wise calls, without a GPU: a copy of it over tensors that
only describe themselves and entry points that only record the call."""
import ctypes
import importlib.machinery
import importlib.util
import shutil

import pytest

from numba_cuda_b200 import _build, _lib

FORMATS = {"f32": _lib.FMT_F32, "u8": _lib.FMT_U8, "i64": _lib.FMT_I64, "e4m3": _lib.FMT_E4M3}
NAMES = ("b2k_norm_rotate", "b2k_norm_rotate_backward_scratch_bytes", "b2k_norm_rotate_backward", "b2k_cache_write",
         "b2k_cache_read", "b2k_norm_rotate_write", "b2k_current_device")
_DEVICE = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0)
_SCRATCH = ctypes.CFUNCTYPE(ctypes.c_longlong, ctypes.c_void_p)(lambda r: 64)


class Tensor:
    dtype = shape = None                    # the extension looks them up in the type first
    requires_grad = False

    def __init__(self, shape, dtype="f32", ptr=4096, strides=None):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, ptr
        if strides is None:
            strides, step = [], 1
            for n in reversed(self.shape):
                strides.insert(0, step)
                step *= max(n, 1)
        self.strides = tuple(strides)

    def stride(self):
        return self.strides

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return 0


def load(tmp_path, entry, level=-1, written=lambda tensors: None):
    """A copy of the extension with every entry point at the address `entry`, inside `level` of forward
    differentiation (-1: none); `written` is told what a call has written."""
    path = str(tmp_path / f"_pyfast{len(list(tmp_path.iterdir()))}.so")        # a file in use stays as it is
    shutil.copy(_build.build_pyfast(), path)
    loader = importlib.machinery.ExtensionFileLoader("_pyfast", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_pyfast", loader))
    loader.exec_module(module)
    address = {name: ctypes.cast(entry, ctypes.c_void_p).value for name in NAMES}
    address["b2k_current_device"] = ctypes.cast(_DEVICE, ctypes.c_void_p).value
    address["b2k_norm_rotate_backward_scratch_bytes"] = ctypes.cast(_SCRATCH, ctypes.c_void_p).value
    module.setup(Tensor, FORMATS, address, lambda stream: 0, lambda n, stream: Tensor((n,), "u8"),
                 {"_current_level": level}, written)
    return module


def pool(heads=2, dim=16, ptr=4096):
    return Tensor((5, 4, heads, dim), "e4m3", ptr), Tensor((5, 4, heads, 1), "f32", ptr)


def calls():
    """Arguments of one good call of every entry, by name."""
    x, w, table, at = Tensor((3, 2, 16)), Tensor((16,)), Tensor((7, 8)), Tensor((3,), "i64")
    rotation = (x, x, w, w, table, table, at)
    return {
        "norm_rotate": (*rotation, 1e-6, False, True, x, x, 0),
        "norm_rotate_backward": (*rotation, x, x, 1e-6, False, True, x, x, w, w, 0),
        "cache_write": (x, x, *pool(), *pool(ptr=8192), at, None, 0),
        "cache_read": (*pool(), *pool(), Tensor((2, 3), "i64"), Tensor((3,), "i64"), x, x, None, 0),
        "norm_rotate_write": (*rotation, x, *pool(), *pool(ptr=8192), at, 1e-6, False, True, None, x, 0),
    }


@pytest.mark.parametrize("name", list(calls()))
def test_good_calls_are_made(tmp_path, name):
    fast = load(tmp_path, ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0))
    assert getattr(fast, name)(*calls()[name]) == 0


@pytest.mark.parametrize("name,cache,array", [("cache_write", 4, 1), ("cache_read", 2, 7), ("norm_rotate_write", 10, 7)])
def test_a_cache_without_its_array_is_left_to_the_python_code(tmp_path, name, cache, array):
    """The Python code refuses it; a cache of no heads, which has no memory, is one too."""
    fast = load(tmp_path, ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0))
    args = list(calls()[name])
    args[cache:cache + 2] = pool(heads=0, ptr=0)
    args[array] = None
    assert getattr(fast, name)(*args) is None
    args[cache:cache + 2] = None, None
    assert getattr(fast, name)(*args) == 0


@pytest.mark.parametrize("name", list(calls()))
def test_the_interpreter_lock_is_free_during_a_call(tmp_path, name):
    """A launch can wait for room in the GPU's queue.  The entry point here is the interpreter's own
    question whether this thread holds the lock."""
    fast = load(tmp_path, ctypes.pythonapi.PyGILState_Check)
    assert getattr(fast, name)(*calls()[name]) == 0


@pytest.mark.parametrize("name", list(calls()))
def test_forward_differentiation_is_left_to_the_python_code(tmp_path, name):
    entry = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0)
    assert getattr(load(tmp_path, entry, level=0), name)(*calls()[name]) is None


@pytest.mark.parametrize("name", list(calls()))
def test_written_tensors_are_told(tmp_path, name):
    """After a call that was made, and after no other."""
    told, args = [], list(calls()[name])
    outputs = {"norm_rotate": (10, 11), "norm_rotate_backward": (12, 13, 14, 15), "cache_write": (2, 3, 4, 5),
               "cache_read": (6, 7), "norm_rotate_write": (17, 8, 9, 10, 11)}[name]
    for i in outputs:
        args[i] = Tensor(args[i].shape, args[i].dtype, args[i].ptr)
    for status in (0, 7):
        entry = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: status)
        assert getattr(load(tmp_path, entry, written=told.append), name)(*args) == status
    assert len(told) == 1 and len(told[0]) == len(outputs)
    assert all(t is args[i] for t, i in zip(told[0], outputs))

    def broken(tensors):
        raise RuntimeError("not told")
    with pytest.raises(RuntimeError, match="not told"):
        getattr(load(tmp_path, ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0), written=broken), name)(*args)

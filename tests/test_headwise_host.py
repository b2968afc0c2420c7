"""The head-wise kernels' host side, without a GPU: layout of the argument structs,
index arithmetic of the paged cache (bad slots, pages and offsets included), and the
refusals of the C ABI and of the Python calls."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import numba_cuda_b200 as cuda
from numba_cuda_b200 import _lib
from numba_cuda_b200.devicearray import DeviceNDArray, _c_strides
from numba_cuda_b200.kernels import _operands as ops, headnorm, kvcache

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("shim") / "headwise_shim.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-x", "c++", os.path.join(HERE, "headwise_shim.cpp"),
                    "-o", out], check=True)
    L = ctypes.CDLL(out)
    i64, vp, i32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    out2 = [ctypes.POINTER(i64)] * 2
    L.shim_size.restype, L.shim_size.argtypes = i64, [i32]
    L.shim_place_of_slot.argtypes = [i64, i64, i64, *out2]
    L.shim_sequence_of_row.restype, L.shim_sequence_of_row.argtypes = i64, [vp, i32, i64, i64]
    L.shim_place_in_sequence.argtypes = [i64, vp, i64, i64, i32, i64, i64, i64, *out2]
    return L


def test_packed_structs_have_the_layout_of_the_header(shim):
    assert shim.shim_size(0) == ops.HEADS.size
    assert shim.shim_size(1) == ops.ROTATION.size
    assert shim.shim_size(2) == ops.CACHE.size
    assert shim.shim_size(3) == 13 * 8 and shim.shim_size(4) == ops.ROTATION.size - 16 and shim.shim_size(5) == 15 * 8


def test_division_by_a_constant(shim):
    rng = np.random.default_rng(0)
    shim.shim_quotient.restype, shim.shim_quotient.argtypes = ctypes.c_uint32, [ctypes.c_uint32] * 2
    for d in [*range(1, 70), 127, 128, 1000, 1023, 1024, 65535, 65537, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1]:
        edge = [k * d + e for k in (0, 1, 2, (2 ** 31 - 1) // d) for e in (-1, 0, 1)] + [2 ** 31 - 1]
        for n in [*edge, *rng.integers(0, 2 ** 31, 40).tolist()]:
            if 0 <= n < 2 ** 31:
                assert shim.shim_quotient(n, d) == n // d, (n, d)


@pytest.mark.parametrize("pages,page_size", [(1, 1), (5, 16), (7, 17), (2 ** 20, 2 ** 14), (2 ** 33, 3), (0, 16)])
def test_place_of_slot(shim, pages, page_size):
    page, place = ctypes.c_int64(), ctypes.c_int64()
    total = pages * page_size
    for slot in {-2 ** 63, -1, 0, 1, page_size - 1, page_size, total // 2, total - 1, total, total + 1, 2 ** 63 - 1, 2 ** 32 + 5}:
        ok = shim.shim_place_of_slot(slot, pages, page_size, page, place)
        assert bool(ok) == (0 <= slot < total)
        if ok:
            assert (page.value, place.value) == divmod(slot, page_size)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("offsets", [[0, 4, 4, 9], [3, 3, 8], [0], [0, 0, 0], [2, 5, 100], [0, 1]])
def test_sequence_of_row(shim, offsets, dtype):
    arr = np.array(offsets, dtype=dtype)
    for row in range(0, 12):
        want = [b for b in range(len(offsets) - 1) if offsets[b] <= row < offsets[b + 1]]
        got = shim.shim_sequence_of_row(arr.ctypes.data, arr.itemsize, len(offsets) - 1, row)
        assert got == (want[0] if want else -1), (row, got, want)


def test_sequence_of_row_stays_inside_for_offsets_that_decrease(shim):
    rng = np.random.default_rng(0)
    for _ in range(300):
        n = int(rng.integers(0, 9))
        # the guard values on both sides would make any row's search leave the range
        whole = np.concatenate([[-2 ** 40], rng.integers(-50, 50, n + 1), [-2 ** 40]])
        arr = whole.astype(np.int64)
        for row in (0, 3, 49, 1000):
            assert -1 <= shim.shim_sequence_of_row(arr.ctypes.data + 8, 8, n, row) < max(n, 1)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_place_in_sequence_refuses_bad_pages(shim, dtype):
    table = np.array([[3, -1, 7, 99], [8, 2, 0, 6]], dtype=dtype)      # 4 columns stored, 3 in use
    page, place = ctypes.c_int64(), ctypes.c_int64()

    def at(position, sequence):
        ok = shim.shim_place_in_sequence(position, table.ctypes.data, 4, 3, table.itemsize, sequence, 8, 5, page, place)
        return (page.value, place.value) if ok else None

    assert at(0, 0) == (3, 0) and at(4, 0) == (3, 4) and at(14, 0) == (7, 4)
    assert at(5, 0) is None                 # page -1
    assert at(0, 1) is None                 # page 8 of 8
    assert at(15, 0) is None and at(2 ** 40, 0) is None        # beyond the width
    assert at(-1, 0) is None
    assert at(7, 1) == (2, 2)


# ---- C ABI ------------------------------------------------------------------------------
def _heads(ptr=4096, ts=64, hs=16, heads=4, dim=16):
    return ops.HEADS.pack(ptr, ts, hs, heads, dim)


def _rotation(format=_lib.FMT_F32, tokens=2, q=(4096, 64, 16, 4, 16), k=(8192, 64, 16, 4, 16), norm=1, eps=1e-6, qw=0,
              kw=0, wfmt=0, rot=16, inter=0, cos=4096, sin=4096, cs=8, ss=8, rows=10, pos=4096, pb=8):
    return ops.ROTATION.pack(format, tokens, *q, *k, norm, eps, qw, kw, wfmt, rot, inter, cos, sin, cs, ss, rows, pos, pb)


def _cache(code=_lib.FMT_E4M3, scale=_lib.FMT_F32, pages=4, size=16, k=(4096, 1024, 64, 16, 8192, 64, 4, 1, 4, 16, 16),
           v=(4096, 1024, 64, 16, 8192, 64, 4, 1, 4, 16, 16)):
    return ops.CACHE.pack(code, scale, pages, size, *k, *v)


def test_norm_rotate_refusals():
    L = _lib.lib()
    NONE = ops.NO_HEADS

    def call(r, q=_heads(), k=_heads()):
        return L.b2k_norm_rotate(r, q, k, None)

    assert call(None) == _lib.ERR_INVALID_ARG
    assert call(_rotation(), None) == _lib.ERR_INVALID_ARG
    assert call(_rotation(format=_lib.FMT_F64)) == _lib.ERR_UNSUPPORTED
    assert call(_rotation(tokens=-1)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(q=(4098, 64, 16, 4, 16))) == _lib.ERR_ALIGNMENT
    assert call(_rotation(q=(0, 64, 16, 4, 16))) == _lib.ERR_INVALID_ARG
    assert call(_rotation(q=(4096, 64, 16, 4, 1025)), _heads(dim=1025)) == _lib.ERR_TOO_LARGE
    assert call(_rotation(q=(4096, 64, 16, 2 ** 30, 16)), _heads(heads=2 ** 30)) == _lib.ERR_TOO_LARGE
    assert call(_rotation(q=(4096, 64, 16, -4, 16))) == _lib.ERR_INVALID_ARG
    assert call(_rotation(q=(4096, 64, 16, 4, 0))) == _lib.ERR_INVALID_ARG
    assert call(_rotation(norm=2)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(eps=-1.0)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(eps=float("nan"))) == _lib.ERR_INVALID_ARG
    assert call(_rotation(qw=4096, wfmt=_lib.FMT_I32)) == _lib.ERR_UNSUPPORTED
    assert call(_rotation(qw=4098)) == _lib.ERR_ALIGNMENT
    assert call(_rotation(inter=2)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(rot=7)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(rot=18)) == _lib.ERR_INVALID_ARG
    assert b"rotary_dim" in L.b2k_last_error()
    assert call(_rotation(cos=0)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(sin=4097)) == _lib.ERR_ALIGNMENT
    assert call(_rotation(pos=0)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(pos=4100)) == _lib.ERR_ALIGNMENT
    assert call(_rotation(pb=2)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(rows=-1)) == _lib.ERR_INVALID_ARG
    # outputs: another shape, rows that overlap, a stride of zero
    assert call(_rotation(), _heads(heads=5)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(), _heads(dim=8)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(), _heads(hs=15)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(), _heads(ts=0)) == _lib.ERR_INVALID_ARG
    assert call(_rotation(), _heads(ts=48)) == _lib.ERR_INVALID_ARG
    assert b"overlap" in L.b2k_last_error()
    assert call(_rotation(k=(0, 0, 0, 0, 0)), _heads(ts=0), NONE) == _lib.ERR_INVALID_ARG
    # nothing to do needs no device
    assert call(_rotation(tokens=0)) == 0
    assert call(_rotation(q=(0,) * 5, k=(0,) * 5), NONE, NONE) == 0
    # rows that do not fit one launch's counters
    big = 2 ** 31
    assert call(_rotation(tokens=big, q=(4096, 64, 16, 4, 16)), _heads(), _heads()) == _lib.ERR_TOO_LARGE


def test_backward_refusals():
    L = _lib.lib()
    h = _heads()

    def call(r=_rotation(qw=4096, kw=4096), grads=(h, h), outs=(h, h), dw=(4096, 4096), scratch=4096, size=None):
        need = L.b2k_norm_rotate_backward_scratch_bytes(r)
        return L.b2k_norm_rotate_backward(r, *grads, *outs, *dw, scratch, need if size is None else size, None)

    assert call(scratch=None) == _lib.ERR_SCRATCH
    assert call(size=16) == _lib.ERR_SCRATCH
    assert call(scratch=4098) == _lib.ERR_ALIGNMENT
    assert call(dw=(4097, None)) == _lib.ERR_ALIGNMENT
    assert call(r=_rotation(qw=4096), dw=(None, 4096)) == _lib.ERR_INVALID_ARG          # no such weight
    assert call(r=_rotation(norm=0), dw=(4096, None)) == _lib.ERR_INVALID_ARG
    assert call(grads=(h, None)) == _lib.ERR_INVALID_ARG
    assert call(grads=(h, _heads(heads=3))) == _lib.ERR_INVALID_ARG
    assert call(outs=(_heads(hs=8), h)) == _lib.ERR_INVALID_ARG
    assert call(r=_rotation(tokens=0), dw=(None, None)) == 0


def test_cache_refusals():
    L = _lib.lib()
    h, NONE = _heads(), ops.NO_HEADS

    def write(cache=_cache(), fmt=_lib.FMT_F32, tokens=2, k=h, v=h, slots=4096, sb=8):
        return L.b2k_cache_write(cache, fmt, tokens, k, v, slots, sb, None)

    side = (4096, 1024, 64, 16, 8192, 64, 4, 1, 4, 16, 16)

    def other(**change):
        names = ["codes", "page", "slot", "head", "scales", "spage", "sslot", "shead", "heads", "dim", "group"]
        return tuple(change.get(n, x) for n, x in zip(names, side))

    assert write(None) == _lib.ERR_INVALID_ARG
    assert write(_cache(code=_lib.FMT_F32)) == _lib.ERR_UNSUPPORTED
    assert write(_cache(scale=_lib.FMT_F16)) == _lib.ERR_UNSUPPORTED
    assert write(_cache(pages=-1)) == _lib.ERR_INVALID_ARG
    assert write(_cache(size=0)) == _lib.ERR_INVALID_ARG
    assert write(_cache(pages=2 ** 40, size=2 ** 40)) == _lib.ERR_TOO_LARGE
    assert write(fmt=_lib.FMT_I32) == _lib.ERR_UNSUPPORTED
    assert write(tokens=-2) == _lib.ERR_INVALID_ARG
    assert write(slots=None) == _lib.ERR_INVALID_ARG
    assert write(sb=1) == _lib.ERR_INVALID_ARG
    assert write(slots=4100) == _lib.ERR_ALIGNMENT
    assert write(k=_heads(heads=3)) == _lib.ERR_INVALID_ARG
    assert write(_cache(k=other(codes=0))) == _lib.ERR_INVALID_ARG
    assert write(_cache(k=other(scales=8194))) == _lib.ERR_ALIGNMENT
    assert write(_cache(k=other(group=0))) == _lib.ERR_INVALID_ARG
    assert write(_cache(k=other(group=5))) == _lib.ERR_INVALID_ARG
    assert write(_cache(k=other(group=8))) == _lib.ERR_INVALID_ARG         # blocks are at least 16 items
    assert write(_cache(v=other(slot=32))) == _lib.ERR_INVALID_ARG         # rows that overlap
    assert write(_cache(v=other(page=0))) == _lib.ERR_INVALID_ARG
    assert write(_cache(v=other(shead=0))) == _lib.ERR_INVALID_ARG
    assert write(tokens=0) == 0
    assert write(_cache(pages=0)) == 0

    def read(cache=_cache(), fmt=_lib.FMT_F32, rows=2, k=h, v=h, table=4096, stride=3, width=3, tb=4, offsets=4096, seqs=2,
             ob=4):
        return L.b2k_cache_read(cache, fmt, rows, k, v, table, stride, width, tb, offsets, seqs, ob, None)

    assert read(rows=-1) == _lib.ERR_INVALID_ARG
    assert read(seqs=-1) == _lib.ERR_INVALID_ARG
    assert read(width=-1) == _lib.ERR_INVALID_ARG
    assert read(offsets=None) == _lib.ERR_INVALID_ARG
    assert read(table=None) == _lib.ERR_INVALID_ARG
    assert read(tb=3) == _lib.ERR_INVALID_ARG
    assert read(k=_heads(hs=8)) == _lib.ERR_INVALID_ARG
    assert read(rows=0) == 0 and read(seqs=0) == 0
    assert read(_cache(k=(0,) * 11, v=(0,) * 11), k=NONE, v=NONE) == 0

    def step(r=_rotation(), v=h, q=h, cache=_cache(), slots=4096, sb=8):
        return L.b2k_norm_rotate_write(r, v, q, cache, slots, sb, None)

    assert step(r=None) == _lib.ERR_INVALID_ARG
    assert step(q=_heads(heads=2)) == _lib.ERR_INVALID_ARG
    assert step(v=_heads(dim=8)) == _lib.ERR_INVALID_ARG
    assert step(slots=None) == _lib.ERR_INVALID_ARG
    assert step(cache=_cache(k=other(dim=32, group=32))) == _lib.ERR_INVALID_ARG
    assert step(r=_rotation(tokens=0)) == 0


# ---- Python calls ------------------------------------------------------------------------
def _fake(shape, dtype):
    """A device array over host memory: enough for every check before the launch."""
    dtype = np.dtype(dtype)
    n = max(1, int(np.prod(shape)) * dtype.itemsize)
    return DeviceNDArray(shape, _c_strides(shape, dtype.itemsize), dtype, gpu_data=(torch.zeros(n, dtype=torch.uint8), 0))


def test_python_refusals_of_norm_rotate():
    q, k = _fake((3, 4, 16), np.float32), _fake((3, 2, 16), np.float32)
    cos, pos = _fake((9, 8), np.float32), _fake((3,), np.int64)
    w = _fake((16,), np.float32)
    f = headnorm.norm_rotate
    with pytest.raises(ValueError, match="neither"):
        f(None, None)
    with pytest.raises(ValueError, match="axes"):
        f(_fake((3, 64), np.float32), k)
    with pytest.raises(TypeError, match="float32, float16"):
        f(_fake((3, 4, 16), np.int32), k)
    with pytest.raises(TypeError, match="unsupported"):
        f(_fake((3, 4, 16), np.float64), k)
    with pytest.raises(ValueError, match="same number"):
        f(q, _fake((2, 2, 16), np.float32))
    with pytest.raises(ValueError, match="same"):
        f(q, _fake((3, 2, 16), np.float16))
    with pytest.raises(ValueError, match="16 items"):
        f(q, k, _fake((15,), np.float32))
    with pytest.raises(TypeError, match="same type"):
        f(q, k, w, _fake((16,), np.float16))
    with pytest.raises(ValueError, match="norm=False"):
        f(q, k, w, norm=False)
    with pytest.raises(ValueError, match="go together"):
        f(q, k, cos=cos, sin=cos)
    with pytest.raises(TypeError, match="float32"):
        f(q, k, cos=_fake((9, 8), np.float16), sin=cos, positions=pos)
    with pytest.raises(ValueError, match="same shape"):
        f(q, k, cos=cos, sin=_fake((9, 4), np.float32), positions=pos)
    with pytest.raises(ValueError, match="more items"):
        f(q, k, cos=_fake((9, 9), np.float32), sin=_fake((9, 9), np.float32), positions=pos)
    with pytest.raises(TypeError, match="int32 or int64"):
        f(q, k, cos=cos, sin=cos, positions=_fake((3,), np.float32))
    with pytest.raises(ValueError, match="3 items"):
        f(q, k, cos=cos, sin=cos, positions=_fake((4,), np.int64))
    with pytest.raises(ValueError, match="shape"):
        f(q, k, cos=cos, sin=cos, positions=pos, q_out=_fake((3, 4, 8), np.float32))
    with pytest.raises(TypeError, match="type"):
        f(q, None, cos=cos, sin=cos, positions=pos, q_out=_fake((3, 4, 16), np.float16))
    with pytest.raises(ValueError, match="without its input"):
        f(q, None, cos=cos, sin=cos, positions=pos, q_out=q, k_out=k)
    with pytest.raises(ValueError, match="device memory"):
        f(q, None, q_out=np.zeros((3, 4, 16), np.float32))
    with pytest.raises(ValueError, match="unit stride"):
        f(DeviceNDArray((3, 4, 16), (4 * 128, 4 * 32, 8), np.float32, gpu_data=(torch.zeros(8192, dtype=torch.uint8), 0)), k)
    b = headnorm.norm_rotate_backward
    with pytest.raises(ValueError, match="go together"):
        b(q, k, w, w, cos, cos, pos, q, None)
    with pytest.raises(ValueError, match="shape and type"):
        b(q, k, w, w, cos, cos, pos, q, q)
    with pytest.raises(ValueError, match="without its weight"):
        b(q, k, w, None, cos, cos, pos, q, k, dq=q, dk=k, dq_weight=w, dk_weight=w)
    with pytest.raises(ValueError, match="contiguous"):
        b(q, k, w, None, cos, cos, pos, q, k, dq=q, dk=k, dq_weight=_fake((8,), np.float32))


def test_python_refusals_of_the_cache():
    k, v = _fake((3, 2, 32), np.float32), _fake((3, 2, 48), np.float32)
    kc, ks = _fake((5, 16, 2, 32), np.uint8), _fake((5, 16, 2, 2), np.float32)
    vc, vs = _fake((5, 16, 2, 48), np.uint8), _fake((5, 16, 2, 1), np.float32)
    slots = _fake((3,), np.int64)
    f = kvcache.write
    with pytest.raises(ValueError, match="go together"):
        f(k, v, kc, None, vc, vs, slots)
    with pytest.raises(ValueError, match="neither"):
        f(None, None, None, None, None, None, slots)
    with pytest.raises(ValueError, match="its cache"):
        f(k, None, kc, ks, vc, vs, slots)
    with pytest.raises(ValueError, match="its cache"):
        f(v, k, kc, ks, vc, vs, slots)
    with pytest.raises(ValueError, match="axes"):
        f(k, v, kc, _fake((5, 16, 2), np.float32), vc, vs, slots)
    with pytest.raises(ValueError, match="axes"):
        f(k, v, kc, _fake((5, 8, 2, 2), np.float32), vc, vs, slots)
    with pytest.raises(ValueError, match="divide"):
        f(k, v, kc, _fake((5, 16, 2, 3), np.float32), vc, vs, slots)
    with pytest.raises(ValueError, match="same pages"):
        f(k, v, kc, ks, _fake((6, 16, 2, 48), np.uint8), _fake((6, 16, 2, 1), np.float32), slots)
    with pytest.raises(TypeError, match="fp8 codes"):
        f(k, v, _fake((5, 16, 2, 32), np.float32), ks, vc, vs, slots)
    with pytest.raises(TypeError, match="E8M0"):
        f(k, v, kc, _fake((5, 16, 2, 2), np.float16), vc, vs, slots)
    with pytest.raises(TypeError, match="same type"):
        f(k, v, kc, _fake((5, 16, 2, 2), np.uint8), vc, vs, slots)
    with pytest.raises(ValueError, match="e4m3 or e5m2"):
        f(k, v, kc, ks, vc, vs, slots, format="bf16")
    with pytest.raises(ValueError, match="3 items"):
        f(k, v, kc, ks, vc, vs, _fake((4,), np.int64))
    with pytest.raises(ValueError, match="same number"):
        f(k, _fake((4, 2, 48), np.float32), kc, ks, vc, vs, slots)
    with pytest.raises(ValueError, match="device memory"):
        f(k, v, np.zeros((5, 16, 2, 32), np.uint8), ks, vc, vs, slots)
    g = kvcache.read
    table, offsets = _fake((2, 4), np.int32), _fake((3,), np.int32)
    with pytest.raises(TypeError, match="page_table"):
        g(kc, ks, vc, vs, _fake((2, 4), np.float32), offsets, k, v)
    with pytest.raises(ValueError, match="page_table"):
        g(kc, ks, vc, vs, _fake((8,), np.int32), offsets, k, v)
    with pytest.raises(ValueError, match="offsets"):
        g(kc, ks, vc, vs, table, _fake((2,), np.int32), k, v)
    with pytest.raises(ValueError, match="same number of rows"):
        g(kc, ks, vc, vs, table, offsets, k, _fake((4, 2, 48), np.float32))
    h = kvcache.norm_rotate_write
    with pytest.raises(ValueError, match="v must have"):
        h(k, k, _fake((4, 2, 48), np.float32), None, None, None, None, None, kc, ks, vc, vs, slots, q_out=k)
    if not torch.cuda.is_available():
        # every check is passed: what is missing is the device
        with pytest.raises((RuntimeError, AssertionError, ValueError)):
            f(k, v, kc, ks, vc, vs, slots)


def test_arrays_of_another_device_are_refused(monkeypatch):
    """The launch goes to the current device: arrays that live elsewhere are an error."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    q = _fake((3, 4, 16), np.float32)                   # "device" -1
    with pytest.raises(ValueError, match="current device is 0"):
        headnorm.norm_rotate(q, None, q_out=q)
    with pytest.raises(ValueError, match="current device is 0"):
        kvcache.write(q, None, _fake((2, 4, 4, 16), np.uint8), _fake((2, 4, 4, 1), np.float32), None, None, _fake((3,), np.int32))


def test_names_are_reachable_from_the_package():
    assert cuda.kernels.headnorm.norm_rotate is headnorm.norm_rotate
    assert cuda.kernels.kvcache.read is kvcache.read

"""Head-wise calls at the edges of their arguments, without a GPU."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from numba_cuda_b200 import _lib
from numba_cuda_b200.kernels import _operands as ops, headnorm, kvcache
from test_headwise_host import _cache, _fake, _heads, _rotation


def test_positions_are_checked_where_nothing_is_rotated():
    """They tell padding tokens; without a rotation they may be left out."""
    L = _lib.lib()

    def call(**change):
        return L.b2k_norm_rotate(_rotation(rot=0, cos=0, sin=0, **change), _heads(), _heads(), None)

    assert call(pos=4100) == _lib.ERR_ALIGNMENT
    assert call(pb=2) == _lib.ERR_INVALID_ARG
    assert call(rows=-1) == _lib.ERR_INVALID_ARG
    assert call(tokens=0, pos=0, pb=0) == 0


def test_rows_whose_last_chunk_has_no_successor_in_32_bits():
    """A thread of the cache read counts a row's chunks in steps of a block's threads."""
    L = _lib.lib()
    heads, dim = 2099202, 1023                                  # 2^31 - 2 single items
    side = (4096, 0, 0, dim, 8192, 0, 0, 1, heads, dim, dim)
    out = ops.HEADS.pack(4096, heads * dim, dim, heads, dim)
    for k, v in ((1, 0), (0, 1)):
        cache = _cache(pages=1, size=1, k=side if k else (0,) * 11, v=side if v else (0,) * 11)
        got = L.b2k_cache_read(cache, _lib.FMT_F16, 1, out if k else ops.NO_HEADS, out if v else ops.NO_HEADS, 4096, 1, 1, 4,
                               4096, 1, 4, None)
        assert got == _lib.ERR_TOO_LARGE


def test_tensors_with_a_tangent_are_refused():
    """The results would have none, without a word."""
    x, w = torch.ones(3, 2, 16), torch.ones(16)
    q, slots = _fake((3, 2, 16), np.float32), _fake((3,), np.int64)
    codes, scales = _fake((5, 4, 2, 16), np.uint8), _fake((5, 4, 2, 1), np.float32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        dual_w = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: headnorm.norm_rotate(dual, None), lambda: headnorm.norm_rotate(q, None, dual_w),
                     lambda: headnorm.norm_rotate(q, None, q_out=dual),
                     lambda: headnorm.norm_rotate_backward(q, None, None, None, None, None, None, dual, None),
                     lambda: kvcache.write(dual, None, codes, scales, None, None, slots),
                     lambda: kvcache.norm_rotate_write(None, q, dual, None, None, None, None, None, codes, scales, codes, scales, slots)):
            with pytest.raises(ValueError, match="tangent"):
                call()


def test_the_package_imports_with_a_torch_of_fewer_types():
    """Types that a torch does not have are types that no tensor of it has."""
    code = ("import torch\n"
            "for name in ('float8_e8m0fnu', 'float8_e5m2', 'float8_e4m3fn'):\n"
            "    delattr(torch, name)\n"
            "import numba_cuda_b200 as cuda\n"
            "from numba_cuda_b200.kernels import _operands\n"
            "assert torch.bfloat16 in _operands._TORCH and cuda.casts.cast and cuda.reduce and cuda.kernels.kvcache.read\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_version_counters_rise_with_a_torch_that_takes_one_tensor_at_a_time():
    code = ("import torch\n"
            "many = torch._C._increment_version\n"
            "def one(x):\n"
            "    if not isinstance(x, torch.Tensor):\n"
            "        raise TypeError('one tensor')\n"
            "    many((x,))\n"
            "torch._C._increment_version = torch.autograd.graph.increment_version = one\n"
            "from numba_cuda_b200.kernels import _operands\n"
            "a, b = torch.zeros(2), torch.zeros(3)\n"
            "_operands.written(a, None, b)\n"
            "assert (a._version, b._version) == (1, 1)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_two_outputs_in_one_memory_are_refused():
    """Keys and values would overwrite each other.  Inputs may share theirs, and so may outputs of no tokens."""
    L = _lib.lib()
    a, b, none = _heads(ptr=1 << 20), _heads(ptr=1 << 21), ops.NO_HEADS
    rotation = _rotation(qw=4096, kw=4096)

    def refused(status):
        return status == _lib.ERR_INVALID_ARG and b"same memory" in L.b2k_last_error()

    assert refused(L.b2k_norm_rotate(rotation, a, a, None))
    assert L.b2k_norm_rotate(_rotation(tokens=0), a, a, None) == 0
    need = L.b2k_norm_rotate_backward_scratch_bytes(rotation)
    assert refused(L.b2k_norm_rotate_backward(rotation, a, a, a, a, 4096, 8192, 4096, need, None))
    assert refused(L.b2k_norm_rotate_backward(rotation, a, a, a, b, 4096, 4096, 4096, need, None))
    side = (4096, 1024, 64, 16, 8192, 64, 4, 1, 4, 16, 16)
    codes, scales = (1 << 16, *side[1:]), (*side[:4], 1 << 16, *side[5:])
    for v in (side, codes, scales):
        cache = _cache(k=side, v=v)
        assert refused(L.b2k_cache_write(cache, _lib.FMT_F32, 2, a, b, 4096, 8, None))
        assert refused(L.b2k_norm_rotate_write(rotation, b, a, cache, 4096, 8, None))
    assert refused(L.b2k_cache_read(_cache(), _lib.FMT_F32, 2, a, a, 4096, 3, 3, 4, 4096, 2, 4, None))
    empty = _cache(pages=0, k=(0, *side[1:4], 0, *side[5:]), v=(0, *side[1:4], 0, *side[5:]))
    assert L.b2k_cache_write(empty, _lib.FMT_F32, 2, a, b, 4096, 8, None) == 0
    assert L.b2k_cache_read(_cache(), _lib.FMT_F32, 0, a, a, 4096, 3, 3, 4, 4096, 2, 4, None) == 0


def test_the_import_makes_no_tensor_on_the_default_device():
    code = ("import torch\n"
            "torch.set_default_device('cuda')\n"
            "from numba_cuda_b200.kernels import _operands\n"
            "assert not torch.cuda.is_initialized()\n"
            "a = torch.zeros(2, device='cpu')\n"
            "_operands.written(a)\n"
            "assert a._version == 1\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

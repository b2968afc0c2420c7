"""Head-wise calls at the ends of their ranges."""
import numpy as np
import pytest
import torch

import headwise_ref as ref
from numba_cuda_b200.kernels import headnorm, kvcache
from test_headnorm_gpu import TORCH, angles, check, f64, setup
from test_kvcache_gpu import pool

pytestmark = pytest.mark.gpu

LARGE = [("bfloat16", 128, 128, False), ("bfloat16", 128, 64, True), ("float32", 64, 64, True), ("float32", 50, 24, False),
         ("float32", 33, 10, True), ("bfloat16", 576, 64, False), ("float32", 64, 0, False)]


def large(dtype, dim, rot, kind):
    """Heads of which some have squares that add up to more than float32 holds."""
    rng, q, _, qw, _, cos, sin, pos = setup(9, 3, 1, dim, rot, dtype, "contiguous", "float32", 1)
    qw[:] = 1.2
    top = torch.finfo(TORCH[dtype]).max
    q[2, 1] = top * 0.99
    q[4, 2] = torch.where(torch.arange(dim, device="cuda") % 2 == 0, top, -top).to(q)
    q[5, 0, dim // 2] = 2e19
    return rng, q, qw, cos, sin, pos, [(2, 1), (4, 2), (5, 0)]


@pytest.mark.parametrize("dtype,dim,rot,inter", LARGE)
def test_squares_beyond_float32_give_zeros(dtype, dim, rot, inter):
    _, q, qw, cos, sin, pos, rows = large(dtype, dim, rot, "forward")
    got = headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, interleaved=inter)[0].as_torch()
    rest = torch.ones(9, 3, dtype=torch.bool)
    for t, h in rows:
        assert not got[t, h].any()
        rest[t, h] = False
    c, s = angles(cos, sin, pos)
    x = f64(q)
    x[~rest.numpy()] = 0.0
    want, size = ref.norm_rotate(x, f64(qw), c, s, 1e-6, inter, True)
    check(torch.where(rest[..., None].cuda(), got, 0.0), want, size, dtype)
    # quantised: codes of zero under the smallest scale
    codes, scales = pool(3, 4, 3, dim, dim, "e4m3", "f32", np.random.default_rng(0))
    kvcache.norm_rotate_write(None, q, None, None, qw, cos, sin, pos, codes, scales, None, None, torch.arange(9, device="cuda"),
                              interleaved=inter)
    for t, h in rows:
        assert not (codes.flatten(0, 1)[t, h] & 0x7F).any() and (scales.flatten(0, 1)[t, h] == 2.0 ** -126).all()

"""Norm and rotation of heads on the GPU against the 64-bit definition.

Tolerances, with u = 2^-24 (half a float32 step): a lane adds at most 32 squares one
after the other, the lanes' sums go through 5 more additions and one scaling, so the
mean is off by at most 39u relative and its root by half of that; rsqrtf adds 2 steps
(4u), the products with x and the weight 3u, a rotation's products and sum 2u more.
That is under 32u of the magnitudes that meet in an item; on top comes half a step of
the stored type."""
import numpy as np
import pytest
import torch

import headwise_ref as ref
import numba_cuda_b200 as cuda
from numba_cuda_b200.kernels import headnorm

pytestmark = pytest.mark.gpu
U = ref.U
TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def f64(t):
    return t.detach().double().cpu().numpy()


def tables(rows, rot, rng):
    angle = rng.uniform(-np.pi, np.pi, (rows, rot // 2))
    return torch.tensor(np.cos(angle), dtype=torch.float32).cuda(), torch.tensor(np.sin(angle), dtype=torch.float32).cuda()


def layout(shape, how, dtype, rng, scale=1.0):
    """Random values of `shape` (tokens, heads, dim) in one of the memory layouts a model has."""
    t, h, d = shape
    x = torch.tensor(rng.standard_normal(shape) * scale, dtype=torch.float32).to(TORCH[dtype]).cuda()
    if how == "contiguous":
        return x
    if how == "packed":                       # a column range of one projection's output
        whole = torch.zeros(t, h * d + 48, dtype=x.dtype, device="cuda")
        view = whole[:, 16:16 + h * d].unflatten(1, (h, d))
    elif how == "heads first":
        view = torch.zeros(h, t, d, dtype=x.dtype, device="cuda").transpose(0, 1)
    elif how == "odd":                        # nothing is aligned to more than an item
        view = torch.zeros(t * (h * (d + 3) + 5) + 1, dtype=x.dtype, device="cuda")[1:].as_strided(
            (t, h, d), (h * (d + 3) + 5, d + 3, 1))
    view.copy_(x)
    return view


def weight(d, dtype, rng):
    return None if dtype is None else torch.tensor(1 + 0.3 * rng.standard_normal(d), dtype=torch.float32).to(TORCH[dtype]).cuda()


def w64(w, d):
    return np.ones(d) if w is None else f64(w)


def check(got, want, size, dtype, factor=32):
    err = np.abs(f64(got) - want)
    bound = factor * U * size + ref.half_step(dtype) * (np.abs(want) + factor * U * size) + ref.tiny_step(dtype)
    assert (err <= bound).all(), float((err / bound).max())


def setup(tokens, qh, kh, dim, rot, dtype, how, wdtype, seed, kdim=None):
    rng = np.random.default_rng(seed)
    q = layout((tokens, qh, dim), how, dtype, rng, 3.0)
    k = layout((tokens, kh, kdim or dim), how, dtype, rng, 0.5)
    cos, sin = tables(61, rot, rng) if rot else (None, None)
    pos = torch.tensor(rng.integers(0, 61, tokens), dtype=torch.int64 if seed % 2 else torch.int32).cuda() if rot else None
    return rng, q, k, weight(dim, wdtype, rng), weight(kdim or dim, wdtype, rng), cos, sin, pos


def angles(cos, sin, pos):
    return (None, None) if cos is None else (f64(cos)[pos.cpu().numpy()], f64(sin)[pos.cpu().numpy()])


SHAPES = [  # tokens, q heads, k heads, dim, rotated, interleaved
    (5, 4, 2, 128, 128, False), (5, 4, 2, 128, 128, True), (33, 3, 3, 64, 64, False), (7, 5, 1, 80, 40, True),
    (7, 5, 1, 80, 80, False), (3, 6, 2, 96, 48, False), (9, 2, 2, 100, 50, False), (1, 1, 1, 256, 256, True),
    (2, 7, 1, 192, 64, False), (4, 2, 1, 576, 64, True), (3, 2, 2, 1024, 1024, False), (3, 1, 1, 1022, 510, True),
    (6, 2, 2, 127, 6, False), (6, 2, 2, 127, 126, True), (2, 1, 1, 2, 2, False), (3, 2, 1, 1, 0, False), (11, 9, 3, 72, 0, False),
    (40, 33, 5, 32, 16, False), (9, 3, 2, 100, 100, False), (9, 3, 2, 50, 50, True), (5, 2, 1, 300, 100, False), (3, 1, 1, 516, 20, False), (257, 12, 4, 112, 112, False), (2, 3, 2, 24, 8, True),
]


@pytest.mark.parametrize("tokens,qh,kh,dim,rot,inter", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float32"),
                                          ("bfloat16", None), ("float32", "float16")])
def test_forward(tokens, qh, kh, dim, rot, inter, dtype, wdtype):
    for seed, how in enumerate(("contiguous", "packed", "heads first", "odd")):
        rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, how, wdtype, seed)
        qo, ko = layout((tokens, qh, dim), how, dtype, rng), layout((tokens, kh, dim), "contiguous", dtype, rng)
        got = headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, eps=1e-5, interleaved=inter, q_out=qo, k_out=ko)
        assert got[0] is qo and got[1] is ko
        c, s = angles(cos, sin, pos)
        for x, w, out in ((q, qw, qo), (k, kw, ko)):
            want, size = ref.norm_rotate(f64(x), w64(w, dim), c, s, 1e-5, inter, True)
            check(out, want, size, dtype)


@pytest.mark.parametrize("tokens,qh,kh,dim,rot,inter", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [("bfloat16", "float32"), ("float16", "float16"), ("float32", "float32")])
def test_backward(tokens, qh, kh, dim, rot, inter, dtype, wdtype):
    # h n and its mean: 39u + the mean's own error again (r^2) + the products' 8u, under 128u of the
    # magnitudes behind an item.  A weight's sum adds at most (tokens * heads) rows one after the other.
    for seed, how in enumerate(("contiguous", "packed", "heads first", "odd")):
        rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, how, wdtype, seed)
        dy = [layout(tuple(x.shape), how, dtype, rng, 0.1) for x in (q, k)]
        out = [layout(tuple(x.shape), how, dtype, rng) for x in (q, k)]
        got = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, *dy, eps=1e-5, interleaved=inter, dq=out[0], dk=out[1])
        c, s = angles(cos, sin, pos)
        for i, (x, w) in enumerate(((q, qw), (k, kw))):
            dx, size, dw, dw_size = ref.norm_rotate_backward(f64(x), w64(w, dim), c, s, f64(dy[i]), 1e-5, inter, True)
            check(out[i], dx, size, dtype, 128)
            sums = got[2 + i].as_torch()
            assert sums.dtype == TORCH[wdtype]
            check(sums, dw, dw_size, wdtype, 64 + x.shape[0] * x.shape[1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradient_against_differences(dtype):
    """The backward call against central differences of the 64-bit forward: their own error
    is h^2/6 of a third derivative, below 1e-6 here."""
    rng, q, k, qw, kw, cos, sin, pos = setup(3, 2, 1, 16, 8, dtype, "contiguous", "float32", 1)
    dy = [layout(tuple(x.shape), "contiguous", dtype, rng) for x in (q, k)]
    dq, dk, dqw, dkw = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, *dy, eps=1e-3)
    c, s = angles(cos, sin, pos)
    for x, w, g, dx, dw in ((q, qw, dy[0], dq, dqw), (k, kw, dy[1], dk, dkw)):
        x, w, g = f64(x), f64(w), f64(g)

        def loss(x, w):
            return (ref.norm_rotate(x, w, c, s, 1e-3, False, True)[0] * g).sum()

        h = 1e-5
        num = np.zeros_like(x)
        for i in np.ndindex(*x.shape):
            step = np.zeros_like(x)
            step[i] = h
            num[i] = (loss(x + step, w) - loss(x - step, w)) / (2 * h)
        np.testing.assert_allclose(f64(dx.as_torch()), num, rtol=2 * ref.half_step(dtype) + 1e-5, atol=1e-5)
        numw = np.array([(loss(x, w + h * e) - loss(x, w - h * e)) / (2 * h) for e in np.eye(len(w))])
        np.testing.assert_allclose(f64(dw.as_torch()), numw, rtol=1e-4, atol=1e-4)


def test_no_norm_no_rotation_and_single_arrays():
    rng, q, k, qw, kw, cos, sin, pos = setup(9, 3, 2, 64, 32, "bfloat16", "packed", "float32", 3)
    c, s = angles(cos, sin, pos)
    qo, ko = headnorm.norm_rotate(q, k, cos=cos, sin=sin, positions=pos, norm=False)
    for x, out in ((q, qo), (k, ko)):
        check(out.as_torch(), *ref.norm_rotate(f64(x), None, c, s, 0, False, False), "bfloat16")
    qo, none = headnorm.norm_rotate(q, None, qw)
    assert none is None
    check(qo.as_torch(), *ref.norm_rotate(f64(q), f64(qw), None, None, 1e-6, False, True), "bfloat16")
    none, ko = headnorm.norm_rotate(None, k, None, kw, cos, sin, pos, interleaved=True)
    check(ko.as_torch(), *ref.norm_rotate(f64(k), f64(kw), c, s, 1e-6, True, True), "bfloat16")
    # one weight only; without the norm the gradient is the inverse rotation
    qo, ko = headnorm.norm_rotate(q, k, None, kw)
    check(qo.as_torch(), *ref.norm_rotate(f64(q), np.ones(64), None, None, 1e-6, False, True), "bfloat16")
    check(ko.as_torch(), *ref.norm_rotate(f64(k), f64(kw), None, None, 1e-6, False, True), "bfloat16")
    dq, dk, a, b = headnorm.norm_rotate_backward(q, k, None, None, cos, sin, pos, q, k, norm=False)
    assert a is None and b is None
    check(dq.as_torch(), *ref.norm_rotate(f64(q), None, c, -s, 0, False, False), "bfloat16")
    dq, dk, a, b = headnorm.norm_rotate_backward(None, k, None, kw, None, None, None, None, k)
    assert dq is None and a is None
    dx, size, dw, dw_size = ref.norm_rotate_backward(f64(k), f64(kw), None, None, f64(k), 1e-6, False, True)
    check(dk.as_torch(), dx, size, "bfloat16", 128)
    check(b.as_torch(), dw, dw_size, "float32", 64 + 18)


def test_heads_of_different_sizes():
    rng, q, k, qw, kw, cos, sin, pos = setup(13, 4, 2, 64, 32, "float16", "contiguous", "float16", 2, kdim=192)
    qo, ko = headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos)
    c, s = angles(cos, sin, pos)
    check(qo.as_torch(), *ref.norm_rotate(f64(q), f64(qw), c, s, 1e-6, False, True), "float16")
    check(ko.as_torch(), *ref.norm_rotate(f64(k), f64(kw), c, s, 1e-6, False, True), "float16")
    got = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        dx, size, dw, dw_size = ref.norm_rotate_backward(f64(x), f64(w), c, s, f64(x), 1e-6, False, True)
        check(got[i].as_torch(), dx, size, "float16", 128)
        check(got[2 + i].as_torch(), dw, dw_size, "float16", 64 + x.shape[0] * x.shape[1])


@pytest.mark.parametrize("dim,kdim", [(50, 1024), (1024, 50), (1022, 64), (36, 1000), (3, 1024)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_long_rows_beside_narrow_chunks(dim, kdim, dtype):
    rng, q, k, qw, kw, _, _, _ = setup(5, 2, 3, dim, 0, dtype, "contiguous", "float32", 0, kdim=kdim)
    qo, ko = headnorm.norm_rotate(q, k, qw, kw)
    got = headnorm.norm_rotate_backward(q, k, qw, kw, None, None, None, q, k)
    for i, (x, w, y) in enumerate(((q, qw, qo), (k, kw, ko))):
        check(y.as_torch(), *ref.norm_rotate(f64(x), f64(w), None, None, 1e-6, False, True), dtype)
        dx, size, dw, dw_size = ref.norm_rotate_backward(f64(x), f64(w), None, None, f64(x), 1e-6, False, True)
        check(got[i].as_torch(), dx, size, dtype, 128)
        check(got[2 + i].as_torch(), dw, dw_size, "float32", 64 + x.shape[0] * x.shape[1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_in_place_is_the_same(dtype):
    rng, q, k, qw, kw, cos, sin, pos = setup(50, 8, 2, 128, 64, dtype, "packed", dtype, 0)
    qo, ko = headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos)
    g = layout(tuple(q.shape), "packed", dtype, rng), layout(tuple(k.shape), "packed", dtype, rng)
    dq, dk, dqw, dkw = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, *g)
    d2 = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, *g, dq=g[0], dk=g[1])
    assert torch.equal(g[0], dq.as_torch()) and torch.equal(g[1], dk.as_torch())
    assert torch.equal(d2[2].as_torch(), dqw.as_torch()) and torch.equal(d2[3].as_torch(), dkw.as_torch())
    headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=q, k_out=k)
    assert torch.equal(q, qo.as_torch()) and torch.equal(k, ko.as_torch())


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_padding_tokens(index):
    rng, q, k, qw, kw, cos, sin, _ = setup(12, 4, 2, 64, 64, "bfloat16", "packed", "float32", 0)
    pos = torch.tensor([0, -1, 5, 61, 60, 2 ** 31 - 1, -2 ** 31, 7, 8, 9, -5, 62], dtype=index, device="cuda")
    valid = ((pos >= 0) & (pos < 61)).cpu().numpy()
    # what padding rows hold reaches nothing
    q[~torch.tensor(valid)] = float("nan")
    k[~torch.tensor(valid)] = float("inf")
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, eps=0.0, q_out=qo, k_out=ko)
    c, s = f64(cos)[pos.cpu().numpy()[valid]], f64(sin)[pos.cpu().numpy()[valid]]
    for x, w, out in ((q, qw, qo), (k, kw, ko)):
        assert (f64(out)[~valid] == 7.0).all()
        check(out[torch.tensor(valid)], *ref.norm_rotate(f64(x)[valid], f64(w), c, s, 0.0, False, True), "bfloat16")
    got = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k, eps=0.0)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        dx, size, dw, dw_size = ref.norm_rotate_backward(f64(x)[valid], f64(w), c, s, f64(x)[valid], 0.0, False, True)
        out = got[i].as_torch()
        assert (f64(out)[~valid] == 0.0).all()
        check(out[torch.tensor(valid)], dx, size, "bfloat16", 128)
        check(got[2 + i].as_torch(), dw, dw_size, "float32", 64 + 48)
    # a batch of padding only, and tables without a row
    qo.fill_(3.0)
    nothing = torch.full_like(pos, -1)
    headnorm.norm_rotate(q, None, qw, None, cos, sin, nothing, q_out=qo)
    headnorm.norm_rotate(q, None, qw, None, cos[:0], sin[:0], torch.zeros_like(pos), q_out=qo)
    assert (f64(qo) == 3.0).all()
    dq, _, dqw, _ = headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, nothing, q, None)
    assert not f64(dq.as_torch()).any() and not f64(dqw.as_torch()).any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_that_are_not_there_add_nothing_whatever_shared_memory_holds(dtype):
    """A call whose tables are NaN leaves NaNs in shared memory; padding tokens and the empty
    places behind the last item of the next call must not pick them up."""
    tokens = 4001
    _, q, k, qw, kw, cos, sin, _ = setup(tokens, 16, 8, 64, 64, dtype, "contiguous", "float32", 0)
    bad = torch.full_like(cos, float("nan"))
    pos = torch.randint(0, 61, (tokens,), device="cuda")
    for every in (1, 2, 3):
        some = pos.clone()
        some[::every] = -1
        valid = (some >= 0).cpu()
        headnorm.norm_rotate_backward(q, k, qw, kw, bad, bad, pos, q, k)
        got = [g.as_torch() for g in headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, some, q, k)]
        want = [g.as_torch() for g in headnorm.norm_rotate_backward(q[valid], k[valid], qw, kw, cos, sin, some[valid.cuda()], q[valid], k[valid])]
        for g, w in zip(got[:2], want[:2]):
            assert torch.equal(g[valid], w) and not g[~valid].any()
        for g, w in zip(got[2:], want[2:]):
            # the same rows in another order of addition: at most that many roundings
            np.testing.assert_allclose(f64(g), f64(w), rtol=0, atol=tokens * 16 * 2 * U * float(w.abs().max() + 1))
    headnorm.norm_rotate_backward(q, k, qw, kw, bad, bad, pos, q, k)
    few = 33                                             # empty places in every role's last warp
    got = headnorm.norm_rotate_backward(q[:few], k[:few], qw, kw, cos, sin, pos[:few], q[:few], k[:few])
    assert all(torch.isfinite(g.as_torch()).all() for g in got)


def test_no_tokens():
    _, q, k, qw, kw, cos, sin, pos = setup(4, 2, 2, 64, 64, "float32", "contiguous", "float32", 0)
    qo, ko = headnorm.norm_rotate(q[:0], k[:0], qw, kw, cos, sin, pos[:0])
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 2, 64)
    dq, dk, dqw, dkw = headnorm.norm_rotate_backward(q[:0], k[:0], qw, kw, cos, sin, pos[:0], q[:0], k[:0])
    assert dq.shape == (0, 2, 64) and not f64(dqw.as_torch()).any() and not f64(dkw.as_torch()).any()


def test_special_values_stay_in_their_rows():
    _, q, _, qw, _, cos, sin, pos = setup(6, 2, 1, 128, 128, "bfloat16", "contiguous", "float32", 0)
    before = headnorm.norm_rotate(q, None, qw, None, cos, sin, pos)[0].as_torch()
    q[1, 0, 3] = float("nan")
    q[2, 1, 5] = float("inf")
    q[3, 0] = 0.0
    got = headnorm.norm_rotate(q, None, qw, None, cos, sin, pos)[0].as_torch()
    same = torch.ones(6, 2, dtype=torch.bool)
    same[1, 0] = same[2, 1] = same[3, 0] = False
    assert torch.equal(got[same], before[same])
    assert got[1, 0].isnan().all()                      # the mean is a NaN
    assert got[2, 1, 5].isnan() and got[3, 0].eq(0).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype,dim", [("bfloat16", 128), ("float32", 64), ("float16", 20)])
def test_an_infinity_reaches_its_own_pair_only(dtype, dim, inter):
    """Without the norm, nothing but the two items of a pair meet."""
    _, q, _, _, _, cos, sin, pos = setup(3, 2, 1, dim, dim // 4 * 2, dtype, "contiguous", None, 0)
    i, j = ref.pairs(dim // 4 * 2, inter)
    for at in (1, dim // 2 + 1, dim - 1):
        x = q.clone()
        x[1, 1, at] = float("inf")
        partner = int(j[list(i).index(at)]) if at in i else int(i[list(j).index(at)]) if at in j else at
        for got in (headnorm.norm_rotate(x, None, None, None, cos, sin, pos, interleaved=inter, norm=False)[0],
                    headnorm.norm_rotate_backward(q, None, None, None, cos, sin, pos, x, None, interleaved=inter, norm=False)[0]):
            bad = ~torch.isfinite(got.as_torch())
            assert set(bad.nonzero()[:, 2].tolist()) <= {at, partner} and bad[1, 1, at]
    # with the norm: a weight's sum is spoilt where the infinite gradient's pair is, and there only
    g = q.clone()
    g[1, 1, dim - 1] = float("inf")
    w = torch.ones(dim, device="cuda", dtype=q.dtype)
    dw = headnorm.norm_rotate_backward(q, None, w, None, cos, sin, pos, g, None, interleaved=inter)[2].as_torch()
    assert (~torch.isfinite(dw)).nonzero().flatten().tolist() == [dim - 1]


def test_device_arrays_host_arrays_and_raw_bf16():
    rng = np.random.default_rng(5)
    q, w = rng.standard_normal((10, 4, 64)).astype(np.float32), rng.standard_normal(64).astype(np.float32)
    c, s = np.cos(rng.random((20, 32))).astype(np.float32), np.sin(rng.random((20, 32))).astype(np.float32)
    pos = rng.integers(0, 20, 10)
    want, size = ref.norm_rotate(q.astype(np.float64), w.astype(np.float64), c[pos].astype(np.float64),
                                 s[pos].astype(np.float64), 1e-6, False, True)
    for put in (lambda x: x, cuda.to_device):
        got, _ = headnorm.norm_rotate(put(q), None, put(w), None, put(c), put(s), put(pos))
        assert got.dtype == np.float32
        err = np.abs(got.copy_to_host() - want)
        assert (err <= 32 * U * size + U * np.abs(want) + 1e-30).all()
    half = cuda.casts.cast(q, "f32", "bf16")
    bits = half.view(np.uint16)
    a = headnorm.norm_rotate(half, None, put(w))[0]
    b = headnorm.norm_rotate(bits, None, put(w))[0]
    assert a.view(np.uint16).copy_to_host().tobytes() == b.view(np.uint16).copy_to_host().tobytes()
    # a combined table's two halves are views with a row stride
    both = torch.tensor(np.concatenate([c, s], 1)).cuda()
    got2, _ = headnorm.norm_rotate(put(q), None, put(w), None, both[:, :32], both[:, 32:], put(pos))
    assert got2.copy_to_host().tobytes() == got.copy_to_host().tobytes()
    with pytest.raises(ValueError, match="autograd"):
        headnorm.norm_rotate(torch.zeros(2, 2, 8, device="cuda", requires_grad=True), None)


def test_equal_calls_give_equal_bits_on_any_stream():
    _, q, k, qw, kw, cos, sin, pos = setup(3000, 16, 4, 128, 128, "bfloat16", "packed", "float32", 0)
    first = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k)
    torch.cuda.synchronize()
    streams = [cuda.stream() for _ in range(3)]
    again = [headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k, stream=st) for st in streams for _ in range(2)]
    torch.cuda.synchronize()
    for got in again:
        for a, b in zip(first, got):
            assert torch.equal(a.as_torch(), b.as_torch())


def test_two_captured_graphs_replayed_at_once():
    """Each captured backward call has its own workspace: graphs that run side by side do
    not disturb each other."""
    sets = [setup(2000, 8, 2, 128, 128, "bfloat16", "contiguous", "float32", seed)[1:] for seed in (0, 2)]
    want = [headnorm.norm_rotate_backward(*s, s[0], s[1]) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, k, qw, kw, cos, sin, pos in sets:
        out = dict(dq=torch.empty_like(q), dk=torch.empty_like(k), dq_weight=torch.empty_like(qw), dk_weight=torch.empty_like(kw))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k, stream=torch.cuda.current_stream(), **out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        for a, b in zip(w, out.values()):
            assert torch.equal(a.as_torch(), b)


def test_offsets_beyond_32_bits():
    """Two tokens more than 2^31 items apart."""
    apart = 2 ** 31 + 64
    buf = torch.empty(apart + 2 * 64, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((2, 2, 64), (apart, 64, 1))
    rng = np.random.default_rng(0)
    q.copy_(torch.tensor(rng.standard_normal((2, 2, 64)), dtype=torch.float32))
    cos, sin = tables(8, 64, rng)
    pos = torch.tensor([3, 4], device="cuda")
    w = weight(64, "float32", rng)
    want, size = ref.norm_rotate(f64(q), f64(w), f64(cos)[[3, 4]], f64(sin)[[3, 4]], 1e-6, False, True)
    out = torch.empty(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    headnorm.norm_rotate(q, None, w, None, cos, sin, pos, q_out=out)
    check(out, want, size, "bfloat16")
    headnorm.norm_rotate(q, None, w, None, cos, sin, pos, q_out=q)
    assert torch.equal(q, out)


def test_heads_of_a_large_batch_match_a_small_one():
    """Every row of a batch that fills the GPU many times over is the row a call of its own gives."""
    _, q, k, qw, kw, cos, sin, pos = setup(20011, 6, 2, 64, 64, "bfloat16", "packed", "bfloat16", 0)
    qo, ko = headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos)
    for at in (0, 1, 9999, 20010):
        a, b = headnorm.norm_rotate(q[at:at + 1], k[at:at + 1], qw, kw, cos, sin, pos[at:at + 1])
        assert torch.equal(a.as_torch()[0], qo.as_torch()[at]) and torch.equal(b.as_torch()[0], ko.as_torch()[at])
    c, s = angles(cos, sin, pos)
    check(qo.as_torch(), *ref.norm_rotate(f64(q), f64(qw), c, s, 1e-6, False, True), "bfloat16")

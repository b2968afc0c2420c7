"""Head-wise calls at the ends of their ranges."""
import threading

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import headwise_ref as ref
from headwise_plan import Plan
from numba_cuda_b200.kernels import _operands, headnorm, kvcache
from test_headnorm_gpu import TORCH, angles, check, f64, layout, setup
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


@pytest.mark.parametrize("dtype,dim,rot,inter", LARGE)
def test_gradient_of_squares_beyond_float32_is_zero(dtype, dim, rot, inter):
    """The result is zeros whatever the items are, so is its gradient; an infinity or a NaN still shows."""
    rng, q, qw, cos, sin, pos, rows = large(dtype, dim, rot, "backward")
    g = layout(tuple(q.shape), "contiguous", dtype, rng, 3.0)
    dq, _, dw, _ = headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, pos, g, None, interleaved=inter)
    dq = dq.as_torch()
    there = q.clone()
    for t, h in rows:
        assert not dq[t, h].any()
        there[t, h] = 0.0
        g[t, h] = 0.0
    want = headnorm.norm_rotate_backward(there, None, qw, None, cos, sin, pos, g, None, interleaved=inter)
    assert torch.equal(dq, want[0].as_torch()) and torch.equal(dw.as_torch(), want[2].as_torch())
    q[2, 1, 1] = float("inf")
    dq = headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, pos, torch.ones_like(g), None, interleaved=inter)[0].as_torch()
    assert dq[2, 1].isnan().all() and not dq[4, 2].any()


@pytest.mark.parametrize("dtype,dim,rot,inter", [("bfloat16", 128, 128, False), ("bfloat16", 80, 40, True), ("float32", 64, 32, False)])
def test_gradient_of_squares_beyond_float32_with_copies_ahead(dtype, dim, rot, inter):
    """Groups of one warp of which some have such a head and others not."""
    tokens, heads = 5001, 16
    assert Plan(dtype, tokens, (heads,), (dim,), (rot,), inter, backward=True).ahead
    rng, q, _, qw, _, cos, sin, pos = setup(tokens, heads, 1, dim, rot, dtype, "contiguous", "float32", 1)
    g = layout(tuple(q.shape), "contiguous", dtype, rng, 3.0)
    t, h = (torch.tensor(rng.integers(0, n, 3000), device="cuda") for n in (tokens, heads))
    there, there_g = q.clone(), g.clone()
    q[t, h] = torch.finfo(TORCH[dtype]).max * 0.99
    there[t, h], there_g[t, h] = 0.0, 0.0
    got = headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, pos, g, None, interleaved=inter)
    want = headnorm.norm_rotate_backward(there, None, qw, None, cos, sin, pos, there_g, None, interleaved=inter)
    assert torch.equal(got[0].as_torch(), want[0].as_torch()) and torch.equal(got[2].as_torch(), want[2].as_torch())
    assert not got[0].as_torch()[t, h].any()
    q[t[0], h[0], 1] = float("-inf")
    dq = headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, pos, g, None, interleaved=inter)[0].as_torch()
    assert dq[t[0], h[0]].isnan().all()
    dq[t[0], h[0]] = 0.0
    assert torch.equal(dq, want[0].as_torch())


@pytest.mark.parametrize("dtype,tokens,qh,kh,dim,rot,inter", [
    ("bfloat16", 4001, 16, 8, 128, 128, False), ("float32", 4001, 16, 8, 64, 32, True),          # with copies ahead
    ("bfloat16", 40, 4, 2, 128, 128, False), ("float32", 40, 4, 2, 33, 10, True), ("float16", 40, 4, 2, 576, 64, False)])
def test_padding_tokens_have_zero_gradients_whatever_the_weight(dtype, tokens, qh, kh, dim, rot, inter):
    assert Plan(dtype, tokens, (qh, kh), (dim, dim), (rot, rot), inter, backward=True).ahead == (tokens > 4000)
    rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, "contiguous", "float32", 1)
    qw[dim - 1], kw[0] = float("nan"), float("inf")
    pos[::3] = -1
    pos[1] = 61
    padding = ((pos < 0) | (pos >= 61)).cpu()
    dq, dk, dqw, dkw = [g.as_torch() for g in headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k, interleaved=inter)]
    assert not dq[padding].any() and not dk[padding].any()
    assert torch.isfinite(dqw).all() and torch.isfinite(dkw).all()         # the weight itself is no part of its gradient


@pytest.mark.parametrize("dim", [64, 33])
def test_tables_without_columns_still_tell_padding(dim):
    """Nothing is rotated, and a token whose position is no row of the tables is padding."""
    rng, q, k, qw, kw, _, _, _ = setup(6, 2, 2, dim, 0, "float32", "contiguous", "float32", 1)
    empty = torch.zeros(5, 0, device="cuda")
    pos = torch.tensor([0, -1, 4, 5, 2, 2 ** 40], device="cuda")
    valid = torch.tensor([True, False, True, False, True, False])
    qo = torch.full_like(q, 7.0)
    headnorm.norm_rotate(q, None, qw, None, empty, empty, pos, q_out=qo)
    assert (qo[~valid] == 7.0).all()
    check(qo[valid], *ref.norm_rotate(f64(q[valid]), f64(qw), None, None, 1e-6, False, True), "float32")
    dq, _, dw, _ = headnorm.norm_rotate_backward(q, None, qw, None, empty, empty, pos, q, None)
    dx, size, dsum, dsize = ref.norm_rotate_backward(f64(q[valid]), f64(qw), None, None, f64(q[valid]), 1e-6, False, True)
    check(dq.as_torch()[valid], dx, size, "float32", 128)
    assert not dq.as_torch()[~valid].any()
    check(dw.as_torch(), dsum, dsize, "float32", 64 + 12)
    codes, scales = pool(2, 4, 2, dim, dim, "e4m3", "f32", rng)
    before = codes.clone()
    kvcache.norm_rotate_write(None, k, None, None, kw, empty, empty, pos, codes, scales, None, None, torch.arange(6, device="cuda"))
    assert torch.equal(codes.flatten(0, 1)[1::2][:3], before.flatten(0, 1)[1::2][:3])
    # tables without rows: padding only
    qo.fill_(7.0)
    headnorm.norm_rotate(q, None, qw, None, empty[:0], empty[:0], pos, q_out=qo)
    assert (qo == 7.0).all()


def test_tensors_inside_forward_differentiation():
    """A tensor with a tangent is refused; others give what they give outside."""
    rng, q, k, qw, kw, cos, sin, pos = setup(9, 4, 2, 64, 32, "float32", "contiguous", "float32", 1)
    out, inside = (torch.empty_like(q), torch.empty_like(k)), (torch.empty_like(q), torch.empty_like(k))
    headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=out[0], k_out=out[1])
    codes, scales = pool(3, 4, 2, 64, 64, "e4m3", "f32", rng)
    with forward_ad.dual_level():
        headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=inside[0], k_out=inside[1])
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        for call in (lambda: headnorm.norm_rotate(q, dual, qw, kw, cos, sin, pos, q_out=out[0], k_out=out[1]),
                     lambda: headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=out[0], k_out=dual),
                     lambda: kvcache.write(dual, None, codes, scales, None, None, pos),
                     lambda: kvcache.read(codes, scales, None, None, pos[None], torch.tensor([0, 1]), dual, None)):
            with pytest.raises(ValueError, match="tangent"):
                call()
    assert torch.equal(out[0], inside[0]) and torch.equal(out[1], inside[1])


@pytest.mark.parametrize("fast", [True, False])
def test_autograd_notices_what_a_call_has_written(fast, monkeypatch):
    """Every output's version counter rises, so a tensor that another operation saved for its backward
    is not taken for what it was; an input's does not."""
    if not fast:
        for module in (headnorm, kvcache):
            monkeypatch.setattr(module, "fast", _operands._NoFast)
    rng, q, k, qw, kw, cos, sin, pos = setup(9, 4, 2, 64, 32, "float32", "contiguous", "float32", 1)
    v = layout((9, 2, 64), "contiguous", "float32", rng)
    pools = [a for _ in range(2) for a in pool(3, 4, 2, 64, 64, "e4m3", "f32", rng)]
    qo, ko, dq, dk, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dw = torch.empty_like(qw), torch.empty_like(kw)
    inputs = (q, k, v, qw, kw, cos, sin, pos)
    slots = torch.arange(9, device="cuda")
    table, offsets = torch.zeros(1, 3, dtype=torch.int64, device="cuda"), torch.tensor([0, 9], device="cuda")
    for call, outputs in (
            (lambda: headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=qo, k_out=ko), (qo, ko)),
            (lambda: headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, q_out=qo), (qo,)),
            (lambda: headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, qo, ko, dq=dq, dk=dk, dq_weight=dw[0], dk_weight=dw[1]),
             (dq, dk, *dw)),
            (lambda: kvcache.write(k, v, *pools, slots), pools), (lambda: kvcache.write(None, v, None, None, *pools[2:], slots), pools[2:]),
            (lambda: kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools, slots, q_out=qo), (qo, *pools)),
            (lambda: kvcache.read(*pools, table, offsets, out, ko), (out, ko))):
        before, still = [o._version for o in outputs], [x._version for x in inputs]
        call()
        assert all(o._version > b for o, b in zip(outputs, before))
        assert [x._version for x in inputs] == still
    # in place over a tensor that a product keeps for its backward
    leaf = torch.ones_like(q, requires_grad=True)
    product = (leaf * qo).sum()
    headnorm.norm_rotate(qo, None, qw, None, cos, sin, pos, q_out=qo)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():                       # tensors without a counter
        made = torch.empty(9, 4, 64, device="cuda")
        headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, q_out=made)
    headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, q_out=made)


def test_calls_of_several_threads_at_once():
    """The lock is free during a call, so threads are inside the library at the same time: each gets its own
    results, and the message of its own error."""
    sets = [setup(500 + 300 * i, 8, 4, 64, 64, "bfloat16", "contiguous", "float32", i)[1:] for i in range(4)]
    want = [[g.as_torch() for g in (*headnorm.norm_rotate(*s), *headnorm.norm_rotate_backward(*s, s[0], s[1]))] for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        q, k, qw, kw, cos, sin, pos = sets[i]
        st = torch.cuda.Stream()
        out = [torch.empty_like(t) for t in (q, k, q, k, qw, kw)]
        for n in range(40):
            headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=out[0], k_out=out[1], stream=st)
            headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, q, k, dq=out[2], dk=out[3], dq_weight=out[4],
                                          dk_weight=out[5], stream=st)
            try:
                headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, eps=-1.0 if i % 2 else 1e-6, q_out=out[0], k_out=out[i % 2],
                                     stream=st)
                wrong.append((i, "no error"))
            except ValueError as e:
                if ("eps" if i % 2 else "shape") not in str(e):
                    wrong.append((i, str(e)))
            if n % 10 == 0:
                st.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(out, want[i])):
                    wrong.append((i, "results"))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dim,rot,inter", [(64, 64, False), (64, 32, True), (33, 10, False), (64, 0, False)])
@pytest.mark.parametrize("items,weights", [(1e15, 1e25), (1e-17, 1e-25)])
def test_weights_and_items_far_from_one(dim, rot, inter, items, weights):
    """Their product leaves float32's range, the normed item's product with the weight does not."""
    _, q, _, qw, _, cos, sin, pos = setup(5, 3, 1, dim, rot, "float32", "contiguous", "float32", 1)
    q *= items
    qw *= weights
    c, s = angles(cos, sin, pos)
    got = headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, eps=0.0, interleaved=inter)[0].as_torch()
    check(got, *ref.norm_rotate(f64(q), f64(qw), c, s, 0.0, inter, True), "float32")

"""The head-wise kernels at sizes where a group of lanes works through several heads of a
token and the gradient's rows are copied ahead, against the 64-bit definition.  Every test
states which kernel its sizes reach.

Tolerances as in test_headnorm_gpu.py and test_kvcache_gpu.py.  A weight's gradient adds
terms that are each off by at most 64u of their magnitude, over as many additions one
after the other as headwise_plan.Plan.additions counts."""
import numpy as np
import pytest
import torch

import headwise_ref as ref
from headwise_plan import Plan
from numba_cuda_b200.kernels import headnorm, kvcache
from test_headnorm_gpu import TORCH, angles, check, f64, layout, setup, w64
from test_kvcache_gpu import LIMIT, check_quantised, expected_after_write, pool, values

pytestmark = pytest.mark.gpu


def check_gradient(plan, got, q, k, qw, kw, cos, sin, pos, dy, inter, norm, dtype, eps=1e-5):
    """Gradients of all tokens against the definition; padding tokens have zeros and add nothing."""
    valid = np.ones(q.shape[0], bool) if pos is None else ((pos >= 0) & (pos < cos.shape[0])).cpu().numpy()
    at = torch.tensor(valid, device="cuda")
    c, s = angles(cos, sin, None if pos is None else pos[at])
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        dx, size, dw, dw_size = ref.norm_rotate_backward(f64(x[at]), w64(w, x.shape[2]), c, s, f64(dy[i][at]), eps, inter, norm)
        check(got[i][at], dx, size, dtype, 128)
        assert not got[i][~at].any()
        if w is not None:
            check(got[2 + i], dw, dw_size, "float32", 64 + plan.additions(i))


def backward(q, k, qw, kw, cos, sin, pos, dy, inter, norm=True, **out):
    got = headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, *dy, eps=1e-5, interleaved=inter, norm=norm, **out)
    return [g if g is None or torch.is_tensor(g) else g.as_torch() for g in got]


AHEAD = [  # type, tokens, q heads, k heads, dim, rotated, interleaved, norm
    ("bfloat16", 4096, 16, 8, 128, 128, False, True), ("float16", 4096, 16, 8, 128, 128, True, True),
    ("bfloat16", 8192, 16, 8, 64, 32, False, True),            # half of a head rotated
    ("float16", 8192, 17, 11, 64, 32, True, True),             # items of fewer heads than the others
    ("bfloat16", 4001, 11, 9, 80, 80, False, True),            # idle lanes
    ("float16", 4001, 11, 9, 80, 40, True, True),
    ("bfloat16", 4001, 11, 9, 72, 48, False, True), ("bfloat16", 4001, 9, 11, 72, 72, True, True),   # an odd number of chunks
    ("float16", 4001, 16, 4, 72, 0, False, True),              # no rotation
    ("bfloat16", 9001, 17, 6, 64, 64, False, True),            # up to 8 heads an item
    ("float32", 4001, 16, 8, 64, 64, False, True), ("float32", 4001, 11, 9, 40, 24, True, True),
    ("float32", 4096, 7, 13, 36, 24, False, True), ("bfloat16", 4001, 11, 9, 80, 32, False, False),
]


@pytest.mark.parametrize("dtype,tokens,qh,kh,dim,rot,inter,norm", AHEAD)
def test_gradient_with_copies_ahead(dtype, tokens, qh, kh, dim, rot, inter, norm):
    plan = Plan(dtype, tokens, (qh, kh), (dim, dim), (rot, rot), inter, backward=True)
    assert plan.ahead and plan.rounds > 2
    rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, "contiguous", "float32" if norm else None, 1)
    dy = [layout(tuple(x.shape), "contiguous", dtype, rng, 0.1) for x in (q, k)]
    if pos is not None:                                        # padding at both ends and in runs
        pos[0] = pos[-1] = -1
        pos[1000:1100] = 61
        pos[2000:2300:3] = -5
        q[1000], k[2000], dy[0][1001], dy[1][2003] = float("nan"), float("inf"), float("nan"), -float("inf")
    got = backward(q, k, qw, kw, cos, sin, pos, dy, inter, norm)
    check_gradient(plan, got, q, k, qw, kw, cos, sin, pos, dy, inter, norm, dtype)
    again = backward(q, k, qw, kw, cos, sin, pos, dy, inter, norm)
    in_place = backward(q, k, qw, kw, cos, sin, pos, dy, inter, norm, dq=dy[0], dk=dy[1])
    assert in_place[0] is dy[0] and in_place[1] is dy[1]
    for a, b, c in zip(got, again, in_place):
        assert a is None or (torch.equal(a, b) and torch.equal(a, c))


NEXT_ROW = [  # sizes whose rows go through registers, several heads an item
    ("bfloat16", 4500, 16, 2, 128, 128, False), ("float16", 4096, 32, 1, 128, 64, True),     # few key heads
    ("float16", 1501, 16, 4, 100, 50, False), ("bfloat16", 3001, 11, 9, 50, 50, True),       # narrow chunks
    ("float32", 1201, 16, 4, 288, 288, False), ("bfloat16", 1201, 16, 4, 576, 64, True),     # several units a lane
    ("float32", 601, 24, 12, 127, 6, False),
]


@pytest.mark.parametrize("dtype,tokens,qh,kh,dim,rot,inter", NEXT_ROW)
def test_gradient_with_the_next_row_in_registers(dtype, tokens, qh, kh, dim, rot, inter):
    plan = Plan(dtype, tokens, (qh, kh), (dim, dim), (rot, rot), inter, backward=True)
    assert not plan.ahead and max(plan.heads_an_item) >= 3
    rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, "contiguous", "float32", 1)
    dy = [layout(tuple(x.shape), "contiguous", dtype, rng, 0.1) for x in (q, k)]
    pos[::7] = -1
    q[0] = float("nan")
    got = backward(q, k, qw, kw, cos, sin, pos, dy, inter)
    check_gradient(plan, got, q, k, qw, kw, cos, sin, pos, dy, inter, True, dtype)


FORWARD = [  # type, tokens, q heads, k heads, dim, rotated, interleaved
    ("bfloat16", 8192, 16, 8, 128, 128, True), ("float16", 8192, 17, 11, 128, 64, False), ("float32", 4096, 17, 11, 64, 64, True),
    ("float32", 4096, 16, 8, 64, 32, False), ("float16", 5001, 20, 20, 80, 40, True), ("bfloat16", 4001, 11, 9, 72, 48, False),
    ("bfloat16", 1501, 17, 11, 100, 50, False), ("float16", 1501, 9, 17, 50, 50, True), ("float32", 1201, 17, 5, 288, 288, False),
    ("bfloat16", 1201, 17, 5, 576, 64, True), ("float16", 601, 24, 11, 127, 6, False),
]


@pytest.mark.parametrize("dtype,tokens,qh,kh,dim,rot,inter", FORWARD)
def test_rotation_of_several_heads_an_item(dtype, tokens, qh, kh, dim, rot, inter):
    plan = Plan(dtype, tokens, (qh, kh), (dim, dim), (rot, rot), inter)
    assert max(plan.heads_an_item) >= 3
    _, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, "contiguous", "float32", 1)
    pos[5::9] = 61
    valid = (pos < 61).cpu()
    qo, ko = torch.full_like(q, 3.0), torch.full_like(k, 3.0)
    headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, 1e-5, inter, q_out=qo, k_out=ko)
    c, s = angles(cos, sin, pos[valid.cuda()])
    for x, w, out in ((q, qw, qo), (k, kw, ko)):
        check(out[valid], *ref.norm_rotate(f64(x[valid]), f64(w), c, s, 1e-5, inter, True), dtype)
        assert (out[~valid] == 3.0).all()


WRITES = [  # type, tokens, heads, dim, v dim, group
    ("bfloat16", 8192, 8, 128, 128, 32),           # scales by shuffles, two a pair of chunks
    ("float16", 4096, 17, 128, 128, 0),            # one scale a head
    ("bfloat16", 4096, 11, 96, 96, 32),            # through shared memory
    ("float32", 4096, 11, 64, 64, 16), ("float16", 2048, 17, 72, 72, 24), ("float32", 1201, 17, 100, 100, 20),
    ("bfloat16", 1201, 11, 576, 576, 0), ("float16", 1201, 11, 576, 576, 64),      # several units a lane
    ("bfloat16", 3001, 8, 33, 33, 0),              # single items
]


@pytest.mark.parametrize("dtype,tokens,heads,dim,v_dim,group", WRITES)
@pytest.mark.parametrize("fmt,scale", [("e4m3", "e8m0"), ("e5m2", "f32")])
def test_write_of_several_heads_an_item(dtype, tokens, heads, dim, v_dim, group, fmt, scale):
    plan = Plan(dtype, tokens, (heads, heads), (dim, v_dim), (0, 0), False)
    assert max(plan.heads_an_item) >= 3
    rng = np.random.default_rng(2)
    x = [layout((tokens, heads, d), "contiguous", dtype, rng, 4.0) for d in (dim, v_dim)]
    # special values behind the first rows of an item
    x[0][3, heads - 1, 1], x[0][4, heads - 2, dim - 1], x[0][5, heads - 1] = float("inf"), -float("inf"), float("nan")
    x[1][6, 2, 0], x[1][7, heads - 1], x[1][8, heads - 1, :3] = float("nan"), 0.0, torch.finfo(TORCH[dtype]).max
    size, pages = 16, -(-tokens // 16) + 3
    groups = [group or d for d in (dim, v_dim)]
    pools = [pool(pages, size, heads, d, g, fmt, scale, rng) for d, g in zip((dim, v_dim), groups)]
    slots = rng.permutation(pages * size)[:tokens]
    slots[rng.random(tokens) < 0.1] = -1
    want = [expected_after_write(v, values(*p, fmt, scale), slots, g, fmt, scale) for v, p, g in zip(x, pools, groups)]
    kvcache.write(*x, *pools[0], *pools[1], torch.tensor(slots).cuda(), format=fmt)
    for p, (codes, scales) in zip(pools, want):
        c, s = values(*p, fmt, scale)
        np.testing.assert_array_equal(s, scales)
        np.testing.assert_array_equal(c, codes)


STEPS = [  # type, tokens, q heads, kv heads, dim, v dim, rotated, interleaved, group
    ("bfloat16", 8192, 16, 8, 128, 128, 128, False, 32), ("float16", 2048, 34, 17, 128, 128, 64, True, 0),
    ("bfloat16", 2048, 22, 11, 96, 96, 48, False, 32), ("float32", 2048, 22, 11, 64, 128, 64, True, 16),
    ("float16", 1201, 17, 17, 100, 100, 50, True, 0), ("bfloat16", 601, 22, 11, 576, 512, 64, False, 64),
]


@pytest.mark.parametrize("dtype,tokens,qh,kh,dim,v_dim,rot,inter,group", STEPS)
@pytest.mark.parametrize("fmt,scale", [("e4m3", "e8m0"), ("e4m3", "f32")])
def test_step_of_several_heads_an_item(dtype, tokens, qh, kh, dim, v_dim, rot, inter, group, fmt, scale):
    plans = Plan.launches(dtype, tokens, (qh, kh, kh), (dim, dim, v_dim), (rot, rot, 0), inter)
    assert all(min(plan.heads_an_item) >= 3 for plan in plans)
    rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, "contiguous", "float32", 1)
    v = layout((tokens, kh, v_dim), "contiguous", dtype, rng)
    groups = [group or d for d in (dim, v_dim)]
    pages = -(-tokens // 16) + 3
    pools = [pool(pages, 16, kh, d, g, fmt, scale, rng) for d, g in zip((dim, v_dim), groups)]
    before = [values(*p, fmt, scale) for p in pools]
    slots = rng.permutation(pages * 16)[:tokens]
    slots[rng.random(tokens) < 0.1] = -1
    pos[::11] = -1
    valid = (pos >= 0).cpu().numpy()
    q_out = torch.full_like(q, 5.0)
    kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools[0], *pools[1], torch.tensor(slots).cuda(), eps=1e-5,
                              interleaved=inter, format=fmt, q_out=q_out)
    at = torch.tensor(valid)
    c, s = angles(cos, sin, pos[at.cuda()])
    check(q_out[at], *ref.norm_rotate(f64(q[at]), f64(qw), c, s, 1e-5, inter, True), dtype)
    assert (q_out[~at] == 5.0).all()
    there = valid & (slots >= 0)
    flat = [[a.reshape(-1, *a.shape[2:])[slots[there]] for a in values(*p, fmt, scale)] for p in pools]
    want, size = ref.norm_rotate(f64(k[at]), f64(kw), c, s, 1e-5, inter, True)
    check_quantised(*flat[0], want[there[valid]], size[there[valid]], groups[0], fmt, scale)
    vc, vs = ref.quantise(f64(v), groups[1], fmt, scale)
    np.testing.assert_array_equal(flat[1][0], vc[there])
    np.testing.assert_array_equal(flat[1][1], vs[there])
    rest = np.setdiff1d(np.arange(pages * 16), slots[there])
    for p, old in zip(pools, before):
        for a, b in zip(values(*p, fmt, scale), old):
            np.testing.assert_array_equal(a.reshape(-1, *a.shape[2:])[rest], b.reshape(-1, *b.shape[2:])[rest])


def test_a_prompt_written_and_read_back():
    """A prompt's step and the read of what it wrote, several heads an item in both."""
    tokens, qh, kh, dim = 4096, 16, 8, 128
    assert min(Plan("bfloat16", tokens, (qh, kh, kh), (dim,) * 3, (dim, dim, 0), False).heads_an_item) >= 3
    rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, dim, "bfloat16", "contiguous", "float32", 1)
    v = layout((tokens, kh, dim), "contiguous", "bfloat16", rng)
    pools = [pool(300, 16, kh, dim, 32, "e4m3", "e8m0", rng) for _ in range(2)]
    pages = rng.permutation(300)[:tokens // 16]
    slots = pages[np.arange(tokens) // 16] * 16 + np.arange(tokens) % 16
    kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools[0], *pools[1], torch.tensor(slots).cuda())
    out = [torch.empty(tokens, kh, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kvcache.read(*pools[0], *pools[1], torch.tensor(pages[None]).cuda(), torch.tensor([0, tokens]).cuda(), *out)
    for o, p in zip(out, pools):
        c, s = values(*p, "e4m3", "e8m0")
        want = ref.dequantise(*(a.reshape(-1, *a.shape[2:])[slots] for a in (c, s)), LIMIT["bfloat16"])
        assert torch.equal(o.cpu(), torch.tensor(want.astype(np.float32)).bfloat16())

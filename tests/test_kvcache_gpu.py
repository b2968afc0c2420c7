"""The quantised paged cache on the GPU.  ``write`` and ``read`` are defined operation by
operation in float32, so they are compared for equality with the definition carried out
in 64 bits and rounded after every operation; the joined step goes by a tolerance."""
import numpy as np
import pytest
import torch

import headwise_ref as ref
import numba_cuda_b200 as cuda
from numba_cuda_b200.kernels import headnorm, kvcache
from test_headnorm_gpu import TORCH, angles, check, f64, layout, setup

pytestmark = pytest.mark.gpu
U = ref.U
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LIMIT = {"float32": 3.4028234663852886e38, "float16": 65504.0, "bfloat16": 3.3895313892515355e38}


def pool(pages, size, heads, dim, group, fmt, scale, rng, how="token"):
    """(codes, scales) with random contents; `how`: place of the head axis in memory, or views of odd strides."""
    lead = (pages, size, heads)

    def lay(shape, dtype):
        if how == "token":
            return torch.empty(shape, dtype=dtype, device="cuda")
        if how == "head":
            return torch.empty((shape[0], shape[2], shape[1], shape[3]), dtype=dtype, device="cuda").transpose(1, 2)
        return torch.empty((shape[0], shape[1], shape[2] + 1, shape[3] + 3), dtype=dtype, device="cuda")[:, :, 1:, 1:-2]

    codes = lay((*lead, dim), torch.uint8)
    codes.copy_(torch.tensor(rng.integers(0, 120, (*lead, dim)) | (rng.integers(0, 2, (*lead, dim)) << 7), dtype=torch.uint8))
    if scale == "f32":
        scales = lay((*lead, dim // group), torch.float32)
        scales.copy_(torch.tensor(rng.uniform(0.001, 0.1, (*lead, dim // group)), dtype=torch.float32))
    else:
        scales = lay((*lead, dim // group), torch.uint8)
        scales.copy_(torch.tensor(rng.integers(110, 135, (*lead, dim // group)), dtype=torch.uint8))
    return codes, scales


def values(codes, scales, fmt, scale):
    c = ref.fp8_values(codes.cpu().numpy(), fmt)
    return c, f64(scales) if scale == "f32" else ref.e8m0_values(scales.cpu().numpy())


def expected_after_write(x, before, slots, group, fmt, scale):
    """64-bit code values and scales of the whole pool."""
    codes, scales = (v.copy() for v in before)
    pages, size = codes.shape[:2]
    new_codes, new_scales = ref.quantise(f64(x), group, fmt, scale)
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * size:
            codes[slot // size, slot % size] = new_codes[t]
            scales[slot // size, slot % size] = new_scales[t]
    return codes, scales


CACHES = [  # tokens, heads, dim, v dim, group (0: whole head), page size, pages, head axis
    (5, 2, 128, 128, 0, 16, 4, "token"), (33, 3, 64, 64, 32, 16, 9, "head"), (1, 1, 1, 1, 0, 1, 3, "token"),
    (70, 2, 96, 48, 16, 7, 30, "odd"), (9, 4, 100, 33, 0, 5, 8, "token"), (12, 2, 256, 512, 64, 64, 2, "head"),
    (3, 1, 576, 576, 0, 3, 40, "token"), (4, 2, 1024, 1024, 16, 16, 2, "token"), (31, 5, 72, 200, 0, 10, 12, "odd"),
    (3500, 2, 128, 33, 0, 16, 230, "token"),      # large, with sides of different chunk widths: a launch each
    (8, 1, 80, 80, 16, 16, 4, "token"), (64, 8, 40, 40, 20, 16, 5, "token"), (6, 2, 1023, 7, 0, 4, 4, "token"),
]


@pytest.mark.parametrize("tokens,heads,dim,v_dim,group,size,pages,how", CACHES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("fmt,scale", [("e4m3", "f32"), ("e4m3", "e8m0"), ("e5m2", "f32"), ("e5m2", "e8m0")])
def test_write(tokens, heads, dim, v_dim, group, size, pages, how, dtype, fmt, scale):
    for seed, lay in enumerate(("contiguous", "packed", "heads first", "odd")):
        rng = np.random.default_rng(seed)
        x = [layout((tokens, heads, d), lay, dtype, rng, 4.0) for d in (dim, v_dim)]
        x[0][0, 0] = 0.0                                            # a row of zeros
        x[1][-1, -1] *= 1e-3
        groups = [group or d if d % (group or d) == 0 else d for d in (dim, v_dim)]
        pools = [pool(pages, size, heads, d, g, fmt, scale, rng, how) for d, g in zip((dim, v_dim), groups)]
        slots = rng.permutation(pages * size)[:tokens]
        slots[rng.random(len(slots)) < 0.2] = -1
        if len(slots) < tokens:
            slots = np.concatenate([slots, np.full(tokens - len(slots), pages * size)])
        at = torch.tensor(slots, dtype=torch.int32 if seed % 2 else torch.int64).cuda()
        want = [expected_after_write(v, values(*p, fmt, scale), slots, g, fmt, scale) for v, p, g in zip(x, pools, groups)]
        kvcache.write(*x, *pools[0], *pools[1], at, format=fmt)
        for p, (codes, scales) in zip(pools, want):
            c, s = values(*p, fmt, scale)
            np.testing.assert_array_equal(s, scales)
            np.testing.assert_array_equal(c, codes)


@pytest.mark.parametrize("fmt,scale", [("e4m3", "f32"), ("e5m2", "e8m0"), ("e4m3", "e8m0")])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_write_special_values(fmt, scale, dtype):
    """Infinities saturate and say nothing about the scale, NaNs stay, the smallest and the
    largest magnitudes keep their scale finite."""
    top = torch.finfo(TORCH[dtype]).max
    x = torch.ones(8, 1, 64, dtype=TORCH[dtype], device="cuda") * 3
    x[0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0])
    x[1] = float("inf")
    x[2] = float("nan")
    x[3] = torch.finfo(TORCH[dtype]).tiny
    x[4] = top
    x[5] = -top
    x[6, 0, 1:] = 0.0
    x[7] = torch.linspace(-1, 1, 64).to(x)
    rng = np.random.default_rng(0)
    for group in (64, 16):
        p = pool(2, 4, 1, 64, group, fmt, scale, rng)
        slots = torch.arange(8, device="cuda").flip(0)
        want = expected_after_write(x, values(*p, fmt, scale), slots.cpu().numpy(), group, fmt, scale)
        kvcache.write(x, None, *p, None, None, slots, format=fmt)
        c, s = values(*p, fmt, scale)
        np.testing.assert_array_equal(s, want[1])
        np.testing.assert_array_equal(c, want[0])
        assert np.isfinite(s).all()


def test_e8m0_scales_and_codes_are_the_casts():
    """With a power-of-two scale of 1 a row's codes are ``casts.cast`` of it, and the scale
    codes are its conversion of the quotients toward +inf."""
    rng = np.random.default_rng(1)
    x = rng.uniform(-448, 448, (300, 2, 64)).astype(np.float32)
    x[..., 0] = 448.0
    p = pool(20, 16, 2, 64, 64, "e4m3", "e8m0", rng)
    kvcache.write(x, None, *p, None, None, np.arange(300))
    got = p[0].flatten(0, 1)[:300].cpu().numpy()
    assert got.tobytes() == cuda.casts.cast(x, "f32", "e4m3").copy_to_host().tobytes()
    assert (p[1].flatten(0, 1)[:300].cpu().numpy() == 127).all()
    x *= np.exp2(rng.uniform(-40, 40, (300, 2, 1))).astype(np.float32)
    kvcache.write(x, None, *p, None, None, np.arange(300))
    q = np.abs(x).max(-1) / np.float32(448)
    want = cuda.casts.cast(q, "f32", "e8m0", rounding=cuda.casts.cudaRoundMode.cudaRoundPosInf).copy_to_host()
    assert (p[1].flatten(0, 1)[:300, :, 0].cpu().numpy() == want).all()


def test_write_row_error_is_half_a_step():
    """Written and read back, an item is off by at most half a step of its code plus the
    roundings of scale and product (3u)."""
    rng = np.random.default_rng(2)
    x = layout((200, 4, 128), "contiguous", "float32", rng, 2.0)
    for fmt, step in (("e4m3", 2.0 ** -4), ("e5m2", 2.0 ** -3)):
        p = pool(13, 16, 4, 128, 128, fmt, "f32", rng)
        kvcache.write(x, None, *p, None, None, torch.arange(200, device="cuda"), format=fmt)
        out = torch.empty_like(x)
        kvcache.read(*p, None, None, torch.arange(13, device="cuda")[None], torch.tensor([0, 200], device="cuda"), out, None, format=fmt)
        scale = np.repeat(f64(p[1].flatten(0, 1)[:200]), 128, -1)
        bits, low, _ = ref.FP8[fmt]
        bound = np.maximum(np.abs(f64(x)) * step, scale * 2.0 ** (low - bits - 1)) * (1 + 1e-6) + 4 * U * np.abs(f64(x))
        assert (np.abs(f64(out) - f64(x)) <= bound).all()


READS = [  # lengths, heads, dim, v dim, group, page size, pages, head axis
    ([5, 0, 17, 1], 2, 128, 128, 0, 16, 6, "token"), ([40], 3, 64, 96, 32, 7, 9, "head"), ([1], 1, 1, 1, 0, 1, 3, "token"),
    ([0, 0], 1, 16, 16, 0, 16, 2, "token"), ([33, 64, 2, 0, 0, 9], 4, 72, 200, 0, 16, 11, "odd"),
    ([100, 3], 1, 576, 576, 64, 64, 3, "token"), ([12, 12], 2, 1024, 1024, 16, 5, 8, "head"), ([9], 5, 100, 33, 0, 4, 5, "token"),
    ([3000, 0, 900], 2, 128, 33, 0, 16, 30, "token"),
    ([31, 30, 29], 2, 80, 40, 0, 10, 7, "token"), ([6, 5], 2, 1023, 8, 0, 3, 9, "odd"), ([200] * 40, 1, 64, 64, 0, 16, 30, "token"),
]


@pytest.mark.parametrize("lengths,heads,dim,v_dim,group,size,pages,how", READS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("fmt,scale", [("e4m3", "f32"), ("e4m3", "e8m0"), ("e5m2", "f32"), ("e5m2", "e8m0")])
def test_read(lengths, heads, dim, v_dim, group, size, pages, how, dtype, fmt, scale):
    for seed, lay in enumerate(("contiguous", "packed", "heads first", "odd")):
        rng = np.random.default_rng(seed)
        groups = [group or d if d % (group or d) == 0 else d for d in (dim, v_dim)]
        pools = [pool(pages, size, heads, d, g, fmt, scale, rng, how) for d, g in zip((dim, v_dim), groups)]
        lead = seed % 2                                                # rows before the first sequence
        offsets = np.cumsum([lead] + lengths)
        rows = int(offsets[-1]) + 3                                    # and behind the last
        width = max(1, -(-max(lengths) // size))
        table = rng.integers(0, pages, (len(lengths), width + 1))
        index = torch.int32 if seed < 2 else torch.int64
        t = torch.tensor(table, dtype=index).cuda()[:, :width]
        out = [layout((rows, heads, d), lay, dtype, rng) for d in (dim, v_dim)]
        before = [f64(o) for o in out]
        got = kvcache.read(*pools[0], *pools[1], t, torch.tensor(offsets, dtype=index).cuda(), *out, format=fmt)
        assert got[0] is out[0] and got[1] is out[1]
        for o, old, p in zip(out, before, pools):
            c, s = values(*p, fmt, scale)
            want = old.copy()
            for b, n in enumerate(lengths):
                at = np.arange(n)
                page, place = table[b, at // size], at % size
                want[offsets[b]:offsets[b + 1]] = ref.dequantise(c[page, place], s[page, place], LIMIT[dtype])
            want = torch.tensor(want.astype(np.float32)).to(TORCH[dtype])
            assert torch.equal(o.cpu(), want)


def test_read_all_codes_and_scales():
    """Every code with every scale code, NaNs and infinities among them: float32 products,
    saturated to the output's range."""
    for fmt in ("e4m3", "e5m2"):
        codes = torch.arange(256, dtype=torch.uint8, device="cuda").expand(16, 16, 1, 256).contiguous()
        scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(16, 16, 1, 1).contiguous()
        table, offsets = torch.arange(16, device="cuda")[None], torch.tensor([0, 256], device="cuda")
        for dtype in TORCH:
            out = torch.empty(256, 1, 256, dtype=TORCH[dtype], device="cuda")
            kvcache.read(codes, scales, None, None, table, offsets, out, None, format=fmt)
            want = ref.dequantise(ref.fp8_values(np.arange(256), fmt)[None, None].repeat(256, 0),
                                  ref.e8m0_values(np.arange(256))[:, None, None], LIMIT[dtype])
            want = torch.tensor(want.astype(np.float32)).to(TORCH[dtype])
            got = out.cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_bad_pages_and_slots():
    """Page numbers that are none give rows of zeros, slots that are none are skipped: the
    index arithmetic itself is tested on the host."""
    rng = np.random.default_rng(0)
    p = pool(5, 4, 2, 64, 64, "e4m3", "f32", rng)
    table = torch.tensor([[0, -1, 4, 5, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    out = torch.full((28, 2, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    kvcache.read(*p, None, None, table, torch.tensor([0, 24], device="cuda"), out, None)
    c, s = values(*p, "e4m3", "f32")
    want = np.zeros((28, 2, 64))
    want[:4] = ref.dequantise(c[0], s[0], LIMIT["bfloat16"])
    want[8:12] = ref.dequantise(c[4], s[4], LIMIT["bfloat16"])
    want[24:] = 9.0
    assert torch.equal(out.cpu(), torch.tensor(want.astype(np.float32)).bfloat16())
    # a table without columns
    kvcache.read(*p, None, None, table[:, :0], torch.tensor([0, 24], device="cuda"), out, None)
    assert not f64(out)[:24].any() and (f64(out)[24:] == 9.0).all()
    before = p[0].clone(), p[1].clone()
    x = torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    kvcache.write(x, None, *p, None, None, torch.tensor([-1, 20, 2 ** 40, -2 ** 63], device="cuda"))
    assert torch.equal(before[0], p[0]) and torch.equal(before[1], p[1])
    kvcache.write(x[:0], None, *p, None, None, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert torch.equal(before[0], p[0])


def test_sequences_share_a_page():
    rng = np.random.default_rng(0)
    p = pool(5, 4, 2, 64, 64, "e4m3", "f32", rng)
    out = torch.empty(12, 2, 64, dtype=torch.float32, device="cuda")
    kvcache.read(*p, None, None, torch.tensor([[3, 1], [3, 2]], device="cuda"), torch.tensor([0, 6, 12], device="cuda"), out, None)
    assert torch.equal(out[:4], out[6:10]) and not torch.equal(out[4:6], out[10:])


def test_typed_codes_tell_the_format():
    rng = np.random.default_rng(0)
    x = layout((6, 2, 64), "contiguous", "bfloat16", rng)
    codes, scales = pool(2, 4, 2, 64, 64, "e5m2", "e8m0", rng)
    slots = torch.arange(6, device="cuda")
    kvcache.write(x, None, codes, scales, None, None, slots, format="e5m2")
    typed = torch.zeros_like(codes).view(torch.float8_e5m2), torch.zeros_like(scales).view(torch.float8_e8m0fnu)
    kvcache.write(x, None, *typed, None, None, slots)
    assert torch.equal(typed[0].view(torch.uint8).flatten(0, 1)[:6], codes.flatten(0, 1)[:6])
    with pytest.raises(TypeError, match="disagree"):
        kvcache.write(x, None, *typed, None, None, slots, format="e4m3")


def test_cache_beyond_32_bits():
    """Slots whose codes lie more than 2^32 bytes into the cache."""
    pages, size, heads, dim = 34000, 16, 8, 1024                   # 4.46e9 codes
    codes = torch.empty(pages, size, heads, dim, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, size, heads, 1, dtype=torch.float32, device="cuda")
    rng = np.random.default_rng(0)
    x = layout((3, heads, dim), "contiguous", "bfloat16", rng)
    far = pages * size - 1
    assert far * heads * dim > 2 ** 32
    kvcache.write(x, None, codes, scales, None, None, torch.tensor([0, far, far - 17], device="cuda"))
    want, s = ref.quantise(f64(x), dim, "e4m3", "f32")
    got = torch.stack([codes[0, 0], codes[-1, -1], codes[-2, -2]])
    np.testing.assert_array_equal(ref.fp8_values(got.cpu().numpy(), "e4m3"), want)
    out = torch.empty(16, heads, dim, dtype=torch.float32, device="cuda")
    kvcache.read(codes, scales, None, None, torch.tensor([[pages - 1]], device="cuda"), torch.tensor([0, 16], device="cuda"), out, None)
    np.testing.assert_array_equal(f64(out[15]), ref.dequantise(want[1], s[1], LIMIT["float32"]))


# ---- the joined step ------------------------------------------------------------------------
STEPS = [  # tokens, q heads, kv heads, dim, v dim, rotated, interleaved, group
    (5, 4, 2, 128, 128, 128, False, 0), (33, 8, 1, 64, 64, 32, True, 32), (1, 1, 1, 80, 80, 80, False, 16),
    (70, 6, 3, 96, 64, 48, False, 0), (9, 3, 3, 100, 33, 50, True, 0), (4, 2, 2, 576, 512, 64, False, 64), (300, 16, 2, 128, 128, 0, False, 32),
]


def check_quantised(codes, scales, want, size, group, fmt, scale):
    """Code values and scales of (tokens, heads, dim) against 64-bit values that are known to 32u of `size`."""
    off = 32 * U * size
    top = ref.FP8[fmt][2]
    amax = np.abs(want).reshape(*want.shape[:-1], -1, group).max(-1)
    slack = off.reshape(*amax.shape, group).max(-1) + 4 * U * amax
    low, high = ref.scale_of(np.maximum(amax - slack, 0), fmt, scale), ref.scale_of(amax + slack, fmt, scale)
    assert ((scales >= low * (1 - 2 * U)) & (scales <= high * (1 + 2 * U))).all()
    s = np.repeat(scales, group, -1)
    bits, lowest, _ = ref.FP8[fmt]
    step = np.maximum(np.abs(want) * 2.0 ** -(bits + 1), s * 2.0 ** (lowest - bits - 1))
    assert (np.abs(codes * s - want) <= step * (1 + 8 * U) + off * (1 + 2.0 ** -bits) + 4 * U * np.abs(want)).all()
    assert (np.abs(codes) <= top).all()


@pytest.mark.parametrize("tokens,qh,kh,dim,v_dim,rot,inter,group", STEPS)
@pytest.mark.parametrize("dtype,wdtype", [("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("fmt,scale", [("e4m3", "f32"), ("e4m3", "e8m0"), ("e5m2", "f32")])
def test_step(tokens, qh, kh, dim, v_dim, rot, inter, group, dtype, wdtype, fmt, scale):
    for seed, how in enumerate(("packed", "contiguous", "odd")):
        rng, q, k, qw, kw, cos, sin, pos = setup(tokens, qh, kh, dim, rot, dtype, how, wdtype, seed)
        v = layout((tokens, kh, v_dim), how, dtype, rng)
        groups = [group or d if d % (group or d) == 0 else d for d in (dim, v_dim)]
        pages = 30 if tokens < 390 else 201
        pools = [pool(pages, 13, kh, d, g, fmt, scale, rng) for d, g in zip((dim, v_dim), groups)]
        before = [values(*p, fmt, scale) for p in pools]
        slots = rng.permutation(pages * 13)[:tokens]
        if tokens > 3:
            slots[2] = -1
        q_out = torch.full((tokens, qh, dim), 5.0, dtype=TORCH[dtype], device="cuda")
        got = kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools[0], *pools[1], torch.tensor(slots).cuda(), eps=1e-5,
                                        interleaved=inter, format=fmt, q_out=q_out)
        assert got is q_out
        c, s = angles(cos, sin, pos)
        check(q_out, *ref.norm_rotate(f64(q), f64(qw), c, s, 1e-5, inter, True), dtype)
        there = slots >= 0
        flat = [[a.reshape(-1, *a.shape[2:])[slots[there]] for a in values(*p, fmt, scale)] for p in pools]
        want, size = ref.norm_rotate(f64(k), f64(kw), c, s, 1e-5, inter, True)
        check_quantised(*flat[0], want[there], size[there], groups[0], fmt, scale)
        vc, vs = ref.quantise(f64(v), groups[1], fmt, scale)                       # values are not computed with: equal
        np.testing.assert_array_equal(flat[1][0], vc[there])
        np.testing.assert_array_equal(flat[1][1], vs[there])
        rest = np.setdiff1d(np.arange(pages * 13), slots)
        for p, old in zip(pools, before):
            for a, b in zip(values(*p, fmt, scale), old):
                np.testing.assert_array_equal(a.reshape(-1, *a.shape[2:])[rest], b.reshape(-1, *b.shape[2:])[rest])


def test_step_with_padding():
    rng, q, k, qw, kw, cos, sin, pos = setup(6, 4, 2, 64, 64, "bfloat16", "packed", "float32", 1)
    v = layout((6, 2, 64), "packed", "bfloat16", rng)
    pools = [pool(4, 4, 2, 64, 64, "e4m3", "f32", rng) for _ in range(2)]
    before = [a.clone() for p in pools for a in p]
    pos[1], pos[4] = -1, 61                                     # no rows of the tables
    slots = torch.tensor([3, 5, -1, 16, 7, 0], device="cuda")
    q_out = torch.full_like(q, 2.0)
    kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools[0], *pools[1], slots, q_out=q_out)
    assert (f64(q_out)[[1, 4]] == 2.0).all()
    ok = torch.tensor([0, 2, 3, 5])
    c, s = angles(cos, sin, pos[ok.cuda()])
    check(q_out[ok], *ref.norm_rotate(f64(q[ok]), f64(qw), c, s, 1e-6, False, True), "bfloat16")
    after = [a for p in pools for a in p]
    changed = [s for s in range(16) if not torch.equal(after[2].flatten(0, 1)[s], before[2].flatten(0, 1)[s])]
    assert changed == [0, 3]
    untouched = [i for i in range(16) if i not in (0, 3)]
    for a, b in zip(after, before):
        assert torch.equal(a.flatten(0, 1)[untouched], b.flatten(0, 1)[untouched])


def test_a_layer_s_passes_together():
    """A prompt in two chunks and then single tokens, as a serving loop would run them: norm,
    rotation and write; at the end the whole sequence is read back.  Chunked and
    token-by-token writes give what one write of everything gives."""
    rng = np.random.default_rng(9)
    tokens, qh, kh, dim, size = 61, 8, 2, 128, 16
    rng, q, k, qw, kw, cos, sin, _ = setup(tokens, qh, kh, dim, 128, "bfloat16", "packed", "bfloat16", 0)
    v = layout((tokens, kh, dim), "packed", "bfloat16", rng)
    pos = torch.arange(tokens, device="cuda")
    pages = torch.tensor([5, 1, 7, 2], device="cuda")
    slots = pages[pos // size] * size + pos % size
    pools = [pool(9, size, kh, dim, 32, "e4m3", "e8m0", rng) for _ in range(2)]
    twin = [tuple(a.clone() for a in p) for p in pools]
    q_out = torch.empty_like(q)
    cuts = [0, 30, 50, *range(51, tokens + 1)]
    for lo, hi in zip(cuts, cuts[1:]):
        kvcache.norm_rotate_write(q[lo:hi], k[lo:hi], v[lo:hi], qw, kw, cos, sin, pos[lo:hi], *pools[0], *pools[1], slots[lo:hi],
                                  q_out=q_out[lo:hi])
    whole = kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *twin[0], *twin[1], slots)
    assert torch.equal(whole.as_torch(), q_out)
    for p, t in zip(pools, twin):
        assert torch.equal(p[0], t[0]) and torch.equal(p[1], t[1])
    out = [torch.empty(tokens, kh, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kvcache.read(*pools[0], *pools[1], pages[None], torch.tensor([0, tokens], device="cuda"), *out)
    # the keys, and the same by separate calls: rounded to bf16 before they are quantised
    want, size_ = ref.norm_rotate(f64(k), f64(kw), f64(cos)[:tokens], f64(sin)[:tokens], 1e-6, False, True)
    scale = ref.scale_of(np.abs(want).reshape(tokens, kh, 4, 32).max(-1), "e4m3", "e8m0")
    step = np.maximum(np.abs(want) * 2.0 ** -4, np.repeat(scale, 32, -1) * 2.0 ** -10)
    # half a step of the code (a scale one power up at most: the 64-bit one may sit on a border) and of bf16
    assert (np.abs(f64(out[0]) - want) <= 2 * step + 2.0 ** -8 * np.abs(want)).all()
    k2 = headnorm.norm_rotate(None, k, None, kw, cos, sin, pos)[1]
    kvcache.write(k2, v, *twin[0], *twin[1], slots)
    assert torch.equal(twin[1][0], pools[1][0]) and torch.equal(twin[1][1], pools[1][1])
    out2 = torch.empty_like(out[0])
    kvcache.read(*twin[0], None, None, pages[None], torch.tensor([0, tokens], device="cuda"), out2, None)
    assert (np.abs(f64(out2) - want) <= 2 * step + 2.0 ** -7 * np.abs(want)).all()


def test_captured_step_follows_its_inputs():
    """A decoding step in a graph: new values in the same memory, slots and positions included."""
    rng, q, k, qw, kw, cos, sin, pos = setup(16, 8, 2, 128, 128, "bfloat16", "contiguous", "bfloat16", 0)
    v = layout((16, 2, 128), "contiguous", "bfloat16", rng)
    pools = [pool(8, 16, 2, 128, 128, "e4m3", "f32", rng) for _ in range(2)]
    slots = torch.arange(16, device="cuda")
    q_out, k_read = torch.empty_like(q), torch.empty(16, 2, 128, dtype=torch.bfloat16, device="cuda")
    table, offsets = torch.zeros(16, 1, dtype=torch.int32, device="cuda"), torch.arange(17, dtype=torch.int32, device="cuda")

    def step(stream):
        kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *pools[0], *pools[1], slots, q_out=q_out, stream=stream)
        kvcache.read(*pools[0], None, None, table, offsets, k_read, None, stream=stream)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(torch.cuda.current_stream())
    for trial in range(3):
        q.copy_(torch.randn(q.shape))
        k.copy_(torch.randn(k.shape))
        slots.copy_(torch.randperm(128)[:16])
        pos.copy_(torch.randint(0, 61, (16,)))
        table.copy_((slots // 16)[:, None])
        g.replay()
        torch.cuda.synchronize()
        got = q_out.clone(), k_read.clone(), pools[0][0].clone()
        step(0)
        torch.cuda.synchronize()
        for a, b in zip(got, (q_out, k_read, pools[0][0])):
            assert torch.equal(a, b)


def test_host_tensors_on_a_stream_of_their_own():
    """What a call copies to the device belongs to the call's stream: work that other
    streams start meanwhile does not get its memory."""
    rng = np.random.default_rng(0)
    x = torch.randn(4000, 4, 128)
    slots = torch.arange(4000)
    want, got = (pool(250, 16, 4, 128, 128, "e4m3", "f32", rng) for _ in range(2))
    kvcache.write(x.cuda(), None, *want, None, None, slots.cuda())
    st = cuda.stream()
    torch.cuda.synchronize()
    for _ in range(5):
        kvcache.write(x, None, *got, None, None, slots, stream=st)
        torch.full((4000, 4, 128), 9.0, device="cuda")            # the default stream takes memory at once
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_streams_of_the_package():
    rng = np.random.default_rng(0)
    x = layout((500, 4, 128), "contiguous", "bfloat16", rng)
    st = cuda.stream()
    a, b = pool(32, 16, 4, 128, 128, "e4m3", "f32", rng), pool(32, 16, 4, 128, 128, "e4m3", "f32", rng)
    slots = torch.arange(500, device="cuda")
    torch.cuda.synchronize()
    kvcache.write(x, None, *a, None, None, slots, stream=st)
    kvcache.write(x, None, *b, None, None, slots)
    torch.cuda.synchronize()
    assert torch.equal(a[0].flatten(0, 1)[:500], b[0].flatten(0, 1)[:500])

"""The extension that makes the head-wise calls for plain tensors: it is there, takes the
common call, gives what the Python code gives, and leaves everything else to it."""
import pytest
import torch

from numba_cuda_b200 import _build, _lib
from numba_cuda_b200.devicearray import from_cuda_array_interface
from numba_cuda_b200.kernels import _operands, headnorm, kvcache
from test_headnorm_gpu import layout, setup

pytestmark = pytest.mark.gpu


class Counted:
    """The extension with a count of the calls it made."""

    def __init__(self, made):
        self.made = made

    def __getattr__(self, name):
        entry = getattr(_operands.fast, name)

        def call(*args):
            status = entry(*args)
            self.made.append((name, status))
            return status
        return call


class Nothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def made(monkeypatch):
    calls = []
    for module in (headnorm, kvcache):
        monkeypatch.setattr(module, "fast", Counted(calls))
    return calls


def slow(monkeypatch):
    for module in (headnorm, kvcache):
        monkeypatch.setattr(module, "fast", Nothing())


def everything(dtype, wdtype, inter, seed, scale, fmt=None):
    """All five calls on one set of tensors; the results."""
    rng, q, k, qw, kw, cos, sin, pos = setup(37, 4, 2, 64, 32, dtype, "packed", wdtype, seed)
    v = layout((37, 2, 96), "packed", dtype, rng)
    slots = torch.randperm(5 * 16, generator=torch.Generator().manual_seed(seed))[:37].cuda()
    slots[3] = -1

    def pools():
        out = []
        for d in (64, 96):
            codes = torch.zeros(5, 16, 2, d, dtype=torch.uint8, device="cuda")
            out.append(codes.view(torch.float8_e4m3fn) if fmt is None else codes)
            s = torch.zeros(5, 16, 2, d // 32, dtype=torch.float32 if scale == "f32" else torch.uint8, device="cuda")
            out.append(s if scale == "f32" or fmt else s.view(torch.float8_e8m0fnu))
        return out

    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, 1e-5, inter, q_out=qo, k_out=ko)
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    dw = [None if w is None else torch.zeros_like(w) for w in (qw, kw)]
    headnorm.norm_rotate_backward(q, k, qw, kw, cos, sin, pos, qo, ko, interleaved=inter, dq=dq, dk=dk, dq_weight=dw[0], dk_weight=dw[1])
    a, b, only = pools(), pools(), pools()
    kvcache.write(ko, v, *a, slots, format=fmt)
    kvcache.write(ko, None, *only[:2], None, None, slots, format=fmt)
    q2 = torch.zeros_like(q)
    kvcache.norm_rotate_write(q, k, v, qw, kw, cos, sin, pos, *b, slots, interleaved=inter, format=fmt, q_out=q2)
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3) % 5
    out = [torch.zeros(80, 2, d, dtype=q.dtype, device="cuda") for d in (64, 96)]
    kvcache.read(*b, table, torch.tensor([0, 30, 77], dtype=torch.int32, device="cuda"), *out, format=fmt)
    results = [qo, ko, dq, dk, *[w for w in dw if w is not None], q2, *a, *b, *only, *out]
    return [r.view(torch.uint8) if r.element_size() == 1 else r for r in results]


@pytest.mark.parametrize("dtype,wdtype,inter,scale,fmt", [
    ("bfloat16", "float32", False, "f32", None), ("float16", None, True, "e8m0", None), ("float32", "float32", True, "f32", None),
    ("bfloat16", "bfloat16", False, "e8m0", "e5m2"), ("float32", None, False, "f32", "e4m3")])
def test_same_results_as_the_python_code(made, monkeypatch, dtype, wdtype, inter, scale, fmt):
    got = everything(dtype, wdtype, inter, 1, scale, fmt)
    assert [name for name, status in made if status == 0] == ["norm_rotate", "norm_rotate_backward", "cache_write",
                                                              "cache_write", "norm_rotate_write", "cache_read"]
    slow(monkeypatch)
    for a, b in zip(got, everything(dtype, wdtype, inter, 1, scale, fmt)):
        assert torch.equal(a, b)


def test_other_arguments_are_left_to_the_python_code(made):
    _, q, k, qw, kw, cos, sin, pos = setup(9, 4, 2, 64, 32, "float32", "contiguous", "float32", 0)
    want = headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos)[0].as_torch()          # no outputs given
    assert made[-1][1] is None
    out = torch.empty_like(q)
    for args in ((from_cuda_array_interface(q), None, qw, None, cos, sin, pos), (q, None, qw.cpu(), None, cos, sin, pos.cpu().numpy()),
                 (torch.nn.Parameter(q, requires_grad=False), None, qw, None, cos, sin, pos)):
        headnorm.norm_rotate(*args, q_out=out)
        assert made[-1][1] is None and torch.equal(out, want)
        out.zero_()
    headnorm.norm_rotate(q, None, qw, None, cos, sin, pos, q_out=out, stream=torch.cuda.current_stream())
    assert made[-1][1] == 0 and torch.equal(out, want)


def test_wrong_arguments_raise_what_the_python_code_raises(made):
    _, q, k, qw, kw, cos, sin, pos = setup(9, 4, 2, 64, 32, "float32", "contiguous", "float32", 0)
    f, qo = headnorm.norm_rotate, torch.empty_like(q)
    half = q.half()
    for error, args, more in (
            (ValueError, (q, k[:5], qw, kw, cos, sin, pos), {}), (ValueError, (q, half, qw, kw, cos, sin, pos), {}),
            (ValueError, (q, k, qw[:63], kw, cos, sin, pos), {}), (TypeError, (q, k, qw.half(), kw, cos, sin, pos), {}),
            (TypeError, (q, k, qw.long(), kw, cos, sin, pos), {}), (ValueError, (q, k, qw, kw, cos, sin[:5], pos), {}),
            (TypeError, (q, k, qw, kw, cos.half(), sin.half(), pos), {}), (TypeError, (q, k, qw, kw, cos, sin, pos.float()), {}),
            (ValueError, (q, k, qw, kw, cos, sin, pos[:3]), {}), (ValueError, (q, k, qw, kw, cos, None, pos), {}),
            (ValueError, (q, k, qw, kw, cos.repeat(1, 3), sin.repeat(1, 3), pos), {}), (ValueError, (None, None), {}),
            (ValueError, (q[0], None), {}), (ValueError, (q.transpose(1, 2), None), {}), (TypeError, (q.long(), None), {}),
            (TypeError, (q.double(), None), {}), (ValueError, (q, None, qw), {"norm": False}),
            (ValueError, (q, None), {"q_out": torch.empty(9, 4, 32, device="cuda")}), (TypeError, (q, None), {"q_out": half}),
            (ValueError, (q, None), {"k_out": k}), (ValueError, (q, None), {"q_out": qo.cpu()}),
            (ValueError, (q, None), {"eps": -1.0}), (ValueError, (q, None), {"q_out": qo[:, :1].expand(9, 4, 64)}),
            (ValueError, (q.detach().requires_grad_(), None), {})):
        with pytest.raises(error):
            f(*args, **{"q_out": qo if args[0] is not None else None, "k_out": torch.empty_like(k) if args[1] is not None else None,
                        **more})
    x = torch.zeros(4, 2, 32, device="cuda")
    codes = torch.zeros(3, 4, 2, 32, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales, slots = torch.zeros(3, 4, 2, 1, device="cuda"), torch.arange(4, device="cuda")
    for error, args in (
            (ValueError, (x, None, codes, None, None, None, slots)), (ValueError, (None, None, codes, scales, None, None, slots)),
            (ValueError, (x[:, :1], None, codes, scales, None, None, slots)), (ValueError, (x, None, codes, scales, None, None, slots[:2])),
            (TypeError, (x, None, codes, scales, None, None, slots.float())), (TypeError, (x, None, codes, scales.half(), None, None, slots)),
            (ValueError, (x, None, codes, scales.repeat(1, 1, 1, 3), None, None, slots)), (ValueError, (x, None, codes[:2], scales, None, None, slots)),
            (ValueError, (x, x, codes, scales, codes[:2], scales[:2], slots)), (ValueError, (x, x[:2], codes, scales, codes, scales, slots)),
            (ValueError, (x, None, codes, scales.repeat(1, 1, 1, 4), None, None, slots)),          # blocks of 8 items
            (TypeError, (x, x, codes, scales, codes.view(torch.uint8).view(torch.float8_e5m2), scales, slots)),
            (TypeError, (x, None, codes, scales, None, None, slots, "e5m2")), (ValueError, (x, None, codes, scales, None, None, slots, "bf16")),
            (TypeError, (x, x, codes, scales, codes, scales.to(torch.uint8), slots))):
        with pytest.raises(error):
            kvcache.write(*args)
    for error, args in (
            (TypeError, (codes, scales, None, None, slots[None].float(), slots[:2], x, None)), (ValueError, (codes, scales, None, None, slots, slots[:2], x, None)),
            (ValueError, (codes, scales, None, None, slots[None], slots, x, None)), (ValueError, (codes, scales, None, None, slots[None], slots[:2], x[:, :, :16], None)),
            (ValueError, (codes, scales, None, None, slots[None], slots[:2], x[:1].expand(4, 2, 32), None))):
        with pytest.raises(error):
            kvcache.read(*args)


def test_references_are_kept_even():
    """Many calls neither leak nor lose a reference to their arguments."""
    import sys
    _, q, k, qw, kw, cos, sin, pos = setup(9, 4, 2, 64, 32, "float32", "contiguous", "float32", 0)
    qo, ko, dw = torch.empty_like(q), torch.empty_like(k), torch.empty_like(qw)
    stream = torch.cuda.Stream()
    args = [q, k, qw, kw, cos, sin, pos, qo, ko, dw, stream, q.dtype, None, True]

    def once():
        headnorm.norm_rotate(q, k, qw, kw, cos, sin, pos, q_out=qo, k_out=ko, stream=stream)
        headnorm.norm_rotate_backward(q, None, qw, None, cos, sin, pos, qo, None, dq=qo, dq_weight=dw, stream=stream)
        _operands.fast.norm_rotate(q, k, qw, kw, cos, None, pos, 1e-6, False, True, qo, ko, 0)       # passed on
        _operands.fast.norm_rotate(q, k, qw, kw, cos, sin, pos, "x", False, True, qo, ko, 0)
        _operands.fast.norm_rotate(q)
    once()
    before = [sys.getrefcount(a) for a in args]
    for _ in range(500):
        once()
    after = [sys.getrefcount(a) for a in args]
    assert [b - a for a, b in zip(before[:-3], after[:-3])] == [0] * (len(args) - 3)
    assert abs(after[-3] - before[-3]) < 50


def test_the_extension_is_built():
    import os
    assert os.path.exists(_build.PYFAST)
    assert _lib.lib().b2k_current_device() == torch.cuda.current_device()

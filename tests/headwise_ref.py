"""The head-wise operators in 64 bits, from their definitions: norm and rotation of
heads, its gradient, and the quantised paged cache.  NumPy only."""
import numpy as np

U = 2.0 ** -24                      # half a step of float32, relative
FP8 = {"e4m3": (3, -6, 448.0), "e5m2": (2, -14, 57344.0)}      # mantissa bits, lowest exponent, largest value


def half_step(name):
    """torch.finfo(t).eps / 2 by type name."""
    return {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[name]


def tiny_step(name):
    """Half a step among the type's subnormal numbers."""
    return {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[name]


def pairs(rot, interleaved):
    if interleaved:
        return np.arange(0, rot, 2), np.arange(1, rot, 2)
    return np.arange(rot // 2), np.arange(rot // 2, rot)


def turn(y, cos, sin, interleaved):
    """(rotated y, the sum of magnitudes behind each item); cos, sin: (tokens, R/2)."""
    rot = 2 * cos.shape[1]
    i, j = pairs(rot, interleaved)
    c, s = cos[:, None], sin[:, None]
    out, size = y.copy(), np.abs(y)
    a, b = y[..., i], y[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    size[..., i], size[..., j] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return out, size


def rms(x, eps):
    return 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def norm_rotate(x, w, cos, sin, eps, interleaved, norm):
    y = x * rms(x, eps) * w if norm else x
    return turn(y, cos, sin, interleaved) if cos is not None else (y, np.abs(y))


def norm_rotate_backward(x, w, cos, sin, dy, eps, interleaved, norm):
    """(dx, magnitude behind dx, dw, magnitude behind dw)."""
    g, size = turn(dy, cos, -sin, interleaved) if cos is not None else (dy, np.abs(dy))
    if not norm:
        return g, size, None, None
    r, d = rms(x, eps), x.shape[-1]
    h, n = g * w, x * r
    dx = r * (h - n * (h * n).mean(-1, keepdims=True))
    big = size * np.abs(w)
    behind = r * (big + np.abs(n) * (big * np.abs(n)).sum(-1, keepdims=True) / d)
    return dx, behind, (g * n).sum((0, 1)), (size * np.abs(n)).sum((0, 1))


def f32(x):
    """Round 64-bit numbers to float32.  One float32 operation is its 64-bit result rounded
    so: 53 bits are enough for the second rounding to be harmless."""
    with np.errstate(over="ignore"):
        return np.asarray(x, dtype=np.float64).astype(np.float32).astype(np.float64)


def nearest_fp8(x, fmt):
    """The nearest value of the format, ties to even, saturating; NaN stays."""
    bits, low, top = FP8[fmt]
    x = np.clip(x, -top, top)
    _, e = np.frexp(np.where(np.isnan(x), 0.0, x))
    step = np.exp2(np.maximum(e - 1, low).astype(np.float64) - bits)
    return np.clip(np.round(x / step) * step, -top, top)


def scale_of(amax, fmt, scale_format):
    s = f32(np.maximum(f32(amax / FP8[fmt][2]), 2.0 ** -126))
    if scale_format == "e8m0":
        m, e = np.frexp(s)
        s = np.exp2(e.astype(np.float64) - (m == 0.5))
    return s


def quantise(x, group, fmt, scale_format):
    """(values of the codes, scales) of x (tokens, heads, dim), every step as in float32."""
    g = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(invalid="ignore", over="ignore"):
        scales = scale_of(np.where(np.isfinite(g), np.abs(g), 0.0).max(-1, initial=0.0), fmt, scale_format)
        by = f32(1.0 / scales)
        codes = nearest_fp8(f32(g * by[..., None]), fmt)
    return codes.reshape(x.shape), scales


def fp8_values(codes, fmt):
    """The numbers that codes (uint8) stand for."""
    codes = np.asarray(codes).astype(np.int64)
    bits, low, top = FP8[fmt]
    mant, exp = codes & ((1 << bits) - 1), (codes & 0x7F) >> bits
    v = np.where(exp == 0, mant * 2.0 ** (low - bits), (1 + mant * 2.0 ** -bits) * np.exp2(exp.astype(np.float64) + low - 1))
    if fmt == "e4m3":
        v = np.where((codes & 0x7F) == 0x7F, np.nan, v)
    else:
        v = np.where((codes & 0x7F) > 0x7C, np.nan, np.where((codes & 0x7F) == 0x7C, np.inf, v))
    return np.where(codes & 0x80, -v, v)


def e8m0_values(codes):
    codes = np.asarray(codes).astype(np.int64)
    return np.where(codes == 255, np.nan, np.exp2(codes.astype(np.float64) - 127))


def dequantise(codes, scales, limit):
    """float32 products of code values and scales, saturated to +-limit (NaN stays)."""
    with np.errstate(invalid="ignore", over="ignore"):
        v = f32(codes * np.repeat(scales, codes.shape[-1] // scales.shape[-1], -1))
    return np.clip(v, -limit, limit)

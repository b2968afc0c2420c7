"""A paged cache of keys and values in 8 bits: quantised as tokens are written
(``write``), read back by page table (``read``), and written straight from the norm and
rotation of a layer's queries and keys (``norm_rotate_write``).

The cache is four arrays the caller owns::

    k_codes  (pages, page_size, heads, dim)     E4M3 or E5M2 codes
    k_scales (pages, page_size, heads, groups)  float32, or E8M0 codes (powers of two)
    v_codes, v_scales                           likewise; heads and dim may differ

of any strides but unit ones in the last axis.  ``dim / groups`` items of a head share a
scale: the whole head (``groups == 1``) or blocks of at least 16 items.  Codes and
scales are the conversions of ``casts``: for a group x,
``scale = max(max|x| / largest, 2**-126)`` over its finite items, with ``largest`` 448
(E4M3) or 57344 (E5M2), rounded up to a power of two for E8M0 scales, and the codes are
``x * (1 / scale)`` to nearest even, saturating; an infinity gets the largest code, a NaN
stays one.  Slot ``page * page_size + place`` is one token's place in the cache.

The reference has the scalar conversion only (numba/cuda/_internal/cuda_fp8.py:3341-3374);
its users write such kernels themselves."""
from __future__ import annotations

from .. import _lib
from ..casts import _format_code
from ..devicearray import stream_ptr
from ._operands import (CACHE, heads, index_bytes, indices, on_one_device, operand, pack_heads)
from .headnorm import result, rotation

_CODES = {_lib.FMT_E4M3, _lib.FMT_E5M2}


def _side(codes, scales, what, written, stream):
    """Checked (codes, scales, heads, dim, group) of keys or values."""
    c = operand(codes, f"{what}_codes", written, stream)
    s = operand(scales, f"{what}_scales", written, stream)
    if len(c.shape) != 4 or len(s.shape) != 4 or c.shape[:3] != s.shape[:3]:
        raise ValueError(f"{what}_codes and {what}_scales must have the axes (pages, page_size, heads, dim) and "
                         "(pages, page_size, heads, groups)")
    if (c.shape[3] > 1 and c.strides[3] != 1) or (s.shape[3] > 1 and s.strides[3] != 1):
        raise ValueError(f"{what}_codes and {what}_scales must have unit stride in their last axis")
    if c.format not in _CODES and c.format != _lib.FMT_U8:
        raise TypeError(f"{what}_codes must be fp8 codes (uint8, float8_e4m3fn or float8_e5m2)")
    if s.format not in (_lib.FMT_F32, _lib.FMT_U8, _lib.FMT_E8M0):
        raise TypeError(f"{what}_scales must be float32 or E8M0 codes (uint8, float8_e8m0fnu)")
    groups = s.shape[3]
    if groups < 1 or c.shape[3] % groups:
        raise ValueError(f"{what}_scales: the groups must divide the head")
    return c, s


def cache(k_codes, k_scales, v_codes, v_scales, format, written, stream):
    """Check the cache's arrays: (k codes operand, v codes operand, operands, packed b2k_cache)."""
    if (k_codes is None) != (k_scales is None) or (v_codes is None) != (v_scales is None):
        raise ValueError("codes and scales go together")
    sides = [None if k_codes is None else _side(k_codes, k_scales, "k", written, stream),
             None if v_codes is None else _side(v_codes, v_scales, "v", written, stream)]
    there = [x for x in sides if x is not None]
    if not there:
        raise ValueError("neither a key nor a value cache is given")
    if any(c.shape[:2] != there[0][0].shape[:2] for c, _ in there):
        raise ValueError("the key and the value cache must have the same pages")
    told = {c.format for c, _ in there} - {_lib.FMT_U8}
    code = _format_code(format) if format is not None else None
    if code is not None and code not in _CODES:
        raise ValueError("format must be e4m3 or e5m2")
    if len(told) > 1 or (told and code is not None and code not in told):
        raise TypeError("the codes' types and format disagree")
    if code is None:
        code = told.pop() if told else _lib.FMT_E4M3
    scale = {_lib.FMT_F32 if s.format == _lib.FMT_F32 else _lib.FMT_E8M0 for _, s in there}
    if len(scale) > 1:
        raise TypeError("the key and the value scales must have the same type")
    values = [code, scale.pop(), there[0][0].shape[0], there[0][0].shape[1]]
    for side in sides:
        if side is None:
            values += [0] * 11
        else:
            c, s = side
            values += [c.ptr, *c.strides[:3], s.ptr, *s.strides[:3], c.shape[2], c.shape[3], c.shape[3] // s.shape[3]]
    return (sides[0][0] if sides[0] else None, sides[1][0] if sides[1] else None,
            [op for side in there for op in side], CACHE.pack(*values))


def _fits(x, codes, what):
    if (x is None) != (codes is None):
        raise ValueError(f"{what} and its cache go together")
    if x is not None and x.shape[1:] != codes.shape[2:]:
        raise ValueError(f"{what} has heads of the shape {x.shape[1:]}, its cache {codes.shape[2:]}")


def write(k, v, k_codes, k_scales, v_codes, v_scales, slots, format=None, stream=0):
    """Quantise the tokens of ``k`` and ``v`` into the cache in one launch.

    :param k, v: (tokens, heads, dim) arrays of one type, float32, float16 or bfloat16, as
                 for ``headnorm.norm_rotate``; either may be ``None``, with its cache.
    :param slots: one int32 or int64 per token; a slot outside the cache (-1, say) skips its
                 token.  The valid slots of one call must be distinct: which token's codes
                 and scales a slot gets is not defined when two share it.
    :param format: ``"e4m3"`` (the default for untyped codes) or ``"e5m2"``.
    """
    k = heads(k, "k", stream=stream) if k is not None else None
    v = heads(v, "v", stream=stream) if v is not None else None
    kc, vc, ops, packed = cache(k_codes, k_scales, v_codes, v_scales, format, True, stream)
    _fits(k, kc, "k")
    _fits(v, vc, "v")
    first = k if k is not None else v
    if k is not None and v is not None and (k.shape[0] != v.shape[0] or k.format != v.format):
        raise ValueError("k and v must have the same number of tokens and the same type")
    at = indices(slots, "slots", first.shape[0], stream)
    on_one_device([k, v, at, *ops])
    _lib.check(_lib.lib().b2k_cache_write(packed, first.format, first.shape[0], pack_heads(k), pack_heads(v), at.ptr,
                                          index_bytes(at), stream_ptr(stream)))


def read(k_codes, k_scales, v_codes, v_scales, page_table, offsets, k_out, v_out, format=None, stream=0):
    """Read sequences back into ``k_out`` and ``v_out`` in one launch; returns both.

    :param page_table: (sequences, width) int32 or int64 page numbers, unit stride along a
                 sequence.  A number that is no page, or a place beyond the width, gives a
                 row of zeros.
    :param offsets: sequences + 1 int32 or int64 row numbers that do not decrease: rows
                 ``offsets[b] .. offsets[b + 1]`` of the outputs are sequence ``b`` from its
                 first place on.  Rows outside all sequences are left as they were.
    :param k_out, v_out: (rows, heads, dim) arrays, float32, float16 or bfloat16; either may
                 be ``None``, with its cache.  Values beyond the type's range saturate.
    """
    ko = heads(k_out, "k_out", True, stream) if k_out is not None else None
    vo = heads(v_out, "v_out", True, stream) if v_out is not None else None
    kc, vc, ops, packed = cache(k_codes, k_scales, v_codes, v_scales, format, False, stream)
    _fits(ko, kc, "k_out")
    _fits(vo, vc, "v_out")
    first = ko if ko is not None else vo
    if ko is not None and vo is not None and (ko.shape[0] != vo.shape[0] or ko.format != vo.format):
        raise ValueError("k_out and v_out must have the same number of rows and the same type")
    table = operand(page_table, "page_table", stream=stream)
    if table.format not in (_lib.FMT_I32, _lib.FMT_I64):
        raise TypeError("page_table must be int32 or int64")
    if len(table.shape) != 2 or (table.shape[1] > 1 and table.strides[1] != 1):
        raise ValueError("page_table must be 2-D, (sequences, width), with unit stride in its last axis")
    at = indices(offsets, "offsets", table.shape[0] + 1, stream)
    on_one_device([ko, vo, table, at, *ops])
    _lib.check(_lib.lib().b2k_cache_read(packed, first.format, first.shape[0], pack_heads(ko), pack_heads(vo), table.ptr,
                                         table.strides[0], table.shape[1], index_bytes(table), at.ptr, table.shape[0],
                                         index_bytes(at), stream_ptr(stream)))
    return k_out, v_out


def norm_rotate_write(q, k, v, q_weight, k_weight, cos, sin, positions, k_codes, k_scales, v_codes, v_scales, slots,
                      eps=1e-6, interleaved=False, norm=True, format=None, q_out=None, stream=0):
    """A serving step between a layer's projection and its attention, in one launch: ``q``
    is normalised and rotated into ``q_out`` (returned), ``k`` is normalised, rotated and
    quantised into the cache without being rounded in between, ``v`` is quantised
    beside it.  Arguments as for ``headnorm.norm_rotate`` and ``write``; a token whose
    position is no row of the tables is skipped altogether, one whose slot is outside
    the cache writes its row of ``q_out`` only."""
    q, k, ops, packed = rotation(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, stream)
    v = heads(v, "v", stream=stream) if v is not None else None
    q_out, qo = result(q_out, q, "q_out", stream)
    kc, vc, more, packed_cache = cache(k_codes, k_scales, v_codes, v_scales, format, True, stream)
    _fits(k, kc, "k")
    _fits(v, vc, "v")
    first = q if q is not None else k
    if v is not None and (v.shape[0] != first.shape[0] or v.format != first.format):
        raise ValueError("v must have the tokens and the type of q and k")
    at = indices(slots, "slots", first.shape[0], stream)
    on_one_device([*ops, v, qo, at, *more])
    _lib.check(_lib.lib().b2k_norm_rotate_write(packed, pack_heads(v), pack_heads(qo), packed_cache, at.ptr,
                                                index_bytes(at), stream_ptr(stream)))
    return q_out


__all__ = ["write", "read", "norm_rotate_write"]

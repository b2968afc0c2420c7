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
from ._operands import CACHE, INDEX_FORMATS, fast, heads, index_bytes, indices, on_one_device, operand, pack_heads, written
from .headnorm import result, rotation

_CODES = (_lib.FMT_E4M3, _lib.FMT_E5M2)
_CODE_TYPES = (_lib.FMT_E4M3, _lib.FMT_E5M2, _lib.FMT_U8)
_SCALE_TYPES = (_lib.FMT_F32, _lib.FMT_E8M0, _lib.FMT_U8)
_NO_SIDE = (0,) * 11


def _side(codes, scales, what, written, stream):
    """Checked operands of keys' or values' codes and scales, and the members of b2k_pages."""
    c = operand(codes, what + "_codes", written, stream)
    s = operand(scales, what + "_scales", written, stream)
    c_ptr, c_shape, c_strides, c_type, _, _ = c
    s_ptr, s_shape, s_strides, s_type, _, _ = s
    if len(c_shape) != 4 or len(s_shape) != 4 or c_shape[:3] != s_shape[:3]:
        raise ValueError(f"{what}_codes and {what}_scales must have the axes (pages, page_size, heads, dim) and "
                         "(pages, page_size, heads, groups)")
    _, _, n, dim = c_shape
    groups = s_shape[3]
    if (c_strides[3] != 1 and dim > 1) or (s_strides[3] != 1 and groups > 1):
        raise ValueError(f"{what}_codes and {what}_scales must have unit stride in their last axis")
    if c_type not in _CODE_TYPES:
        raise TypeError(f"{what}_codes must be fp8 codes (uint8, float8_e4m3fn or float8_e5m2)")
    if s_type not in _SCALE_TYPES:
        raise TypeError(f"{what}_scales must be float32 or E8M0 codes (uint8, float8_e8m0fnu)")
    if groups < 1 or dim % groups:
        raise ValueError(f"{what}_scales: the groups must divide the head")
    return c, s, (c_ptr, c_strides[0], c_strides[1], c_strides[2], s_ptr, s_strides[0], s_strides[1], s_strides[2], n, dim,
                  dim // groups)


def cache(k_codes, k_scales, v_codes, v_scales, format, written, stream):
    """Check the cache's arrays: (shape of k_codes, of v_codes, operands, packed b2k_cache)."""
    if (k_codes is None) != (k_scales is None) or (v_codes is None) != (v_scales is None):
        raise ValueError("codes and scales go together")
    code = None
    if format is not None:
        code = _format_code(format)
        if code not in _CODES:
            raise ValueError("format must be e4m3 or e5m2")
    k_shape = v_shape = pages = scale = None
    k_members = v_members = _NO_SIDE
    ops = []
    if k_codes is not None:
        c, s, k_members = _side(k_codes, k_scales, "k", written, stream)
        ops += [c, s]
        k_shape = c[1]
    if v_codes is not None:
        c, s, v_members = _side(v_codes, v_scales, "v", written, stream)
        ops += [c, s]
        v_shape = c[1]
    for at in range(0, len(ops), 2):
        told, kind = ops[at][3], ops[at + 1][3]
        if told != _lib.FMT_U8:
            if code is not None and code != told:
                raise TypeError("the codes' types and format disagree")
            code = told
        kind = _lib.FMT_F32 if kind == _lib.FMT_F32 else _lib.FMT_E8M0
        if scale is not None and scale != kind:
            raise TypeError("the key and the value scales must have the same type")
        scale = kind
        if pages is not None and pages != ops[at][1][:2]:
            raise ValueError("the key and the value cache must have the same pages")
        pages = ops[at][1][:2]
    if not ops:
        raise ValueError("neither a key nor a value cache is given")
    return k_shape, v_shape, ops, CACHE.pack(_lib.FMT_E4M3 if code is None else code, scale, *pages, *k_members, *v_members)


def _fits(op, shape, what):
    if (op is None) != (shape is None):
        raise ValueError(f"{what} and its cache go together")
    if op is not None and op[1][1:] != shape[2:]:
        raise ValueError(f"{what} has heads of the shape {tuple(op[1][1:])}, its cache {tuple(shape[2:])}")


def _pair(k, v, what):
    """The number of tokens (rows) and the type of k and v, of which one may be missing."""
    first = k if k is not None else v
    if k is not None and v is not None and (k[1][0] != v[1][0] or k[3] != v[3]):
        raise ValueError(f"{what} and the same type")
    return first[1][0], first[3]


def write(k, v, k_codes, k_scales, v_codes, v_scales, slots, format=None, stream=0):
    """Quantise the tokens of ``k`` and ``v`` into the cache in one launch.

    :param k, v: (tokens, heads, dim) arrays of one type, float32, float16 or bfloat16, as
                 for ``headnorm.norm_rotate``; either may be ``None``, with its cache.
    :param slots: one int32 or int64 per token; a slot outside the cache (-1, say) skips its
                 token.  The valid slots of one call must be distinct: which token's codes
                 and scales a slot gets is not defined when two share it.
    :param format: ``"e4m3"`` (the default for untyped codes) or ``"e5m2"``.
    """
    status = fast.cache_write(k, v, k_codes, k_scales, v_codes, v_scales, slots, format, stream)
    if status is not None:
        return _lib.check(status)
    k = heads(k, "k", stream=stream) if k is not None else None
    v = heads(v, "v", stream=stream) if v is not None else None
    kc, vc, ops, packed = cache(k_codes, k_scales, v_codes, v_scales, format, True, stream)
    _fits(k, kc, "k")
    _fits(v, vc, "v")
    tokens, fmt = _pair(k, v, "k and v must have the same number of tokens")
    at = indices(slots, "slots", tokens, stream)
    on_one_device((k, v, at, *ops))
    _lib.check(_lib.lib().b2k_cache_write(packed, fmt, tokens, pack_heads(k), pack_heads(v), at[0], index_bytes(at),
                                          stream_ptr(stream)))
    written(k_codes, k_scales, v_codes, v_scales)


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
    status = fast.cache_read(k_codes, k_scales, v_codes, v_scales, page_table, offsets, k_out, v_out, format, stream)
    if status is not None:
        _lib.check(status)
        return k_out, v_out
    ko = heads(k_out, "k_out", True, stream) if k_out is not None else None
    vo = heads(v_out, "v_out", True, stream) if v_out is not None else None
    kc, vc, ops, packed = cache(k_codes, k_scales, v_codes, v_scales, format, False, stream)
    _fits(ko, kc, "k_out")
    _fits(vo, vc, "v_out")
    rows, fmt = _pair(ko, vo, "k_out and v_out must have the same number of rows")
    table = operand(page_table, "page_table", stream=stream)
    if table[3] not in INDEX_FORMATS:
        raise TypeError("page_table must be int32 or int64")
    if len(table[1]) != 2 or (table[2][1] != 1 and table[1][1] > 1):
        raise ValueError("page_table must be 2-D, (sequences, width), with unit stride in its last axis")
    sequences, width = table[1]
    at = indices(offsets, "offsets", sequences + 1, stream)
    on_one_device((ko, vo, table, at, *ops))
    _lib.check(_lib.lib().b2k_cache_read(packed, fmt, rows, pack_heads(ko), pack_heads(vo), table[0], table[2][0], width,
                                         index_bytes(table), at[0], sequences, index_bytes(at), stream_ptr(stream)))
    written(k_out, v_out)
    return k_out, v_out


def norm_rotate_write(q, k, v, q_weight, k_weight, cos, sin, positions, k_codes, k_scales, v_codes, v_scales, slots,
                      eps=1e-6, interleaved=False, norm=True, format=None, q_out=None, stream=0):
    """A serving step between a layer's projection and its attention, in one launch: ``q``
    is normalised and rotated into ``q_out`` (returned), ``k`` is normalised, rotated and
    quantised into the cache without being rounded in between, ``v`` is quantised
    beside it.  Arguments as for ``headnorm.norm_rotate`` and ``write``; a token whose
    position is no row of the tables is skipped altogether, one whose slot is outside
    the cache writes its row of ``q_out`` only."""
    status = fast.norm_rotate_write(q, k, q_weight, k_weight, cos, sin, positions, v, k_codes, k_scales, v_codes, v_scales,
                                    slots, eps, interleaved, norm, format, q_out, stream)
    if status is not None:
        _lib.check(status)
        return q_out
    q, k, ops, packed = rotation(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, stream)
    v = heads(v, "v", stream=stream) if v is not None else None
    q_out, qo = result(q_out, q, "q_out", stream)
    kc, vc, more, packed_cache = cache(k_codes, k_scales, v_codes, v_scales, format, True, stream)
    _fits(k, kc, "k")
    _fits(v, vc, "v")
    first = q if q is not None else k
    if v is not None and (v[1][0] != first[1][0] or v[3] != first[3]):
        raise ValueError("v must have the tokens and the type of q and k")
    at = indices(slots, "slots", first[1][0], stream)
    on_one_device((*ops, v, qo, at, *more))
    _lib.check(_lib.lib().b2k_norm_rotate_write(packed, pack_heads(v), pack_heads(qo), packed_cache, at[0], index_bytes(at),
                                                stream_ptr(stream)))
    written(q_out, k_codes, k_scales, v_codes, v_scales)
    return q_out


__all__ = ["write", "read", "norm_rotate_write"]

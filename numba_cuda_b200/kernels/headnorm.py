"""Norm and rotation of a transformer layer's queries and keys, head by head, in one
pass over the data: ``norm_rotate`` and its gradient ``norm_rotate_backward``.

For a head ``x`` of a token at position ``p``::

    y = x / sqrt(mean(x**2) + eps) * weight
    (y[i], y[j]) -> (y[i] cos - y[j] sin, y[j] cos + y[i] sin),   cos = cos[p, i], sin = sin[p, i]

over the pairs ``(i, j) = (i, i + R/2)`` of the first ``R`` items, or ``(2i, 2i + 1)`` with
``interleaved``; the remaining items are not rotated.  All arithmetic is in float32,
rounded once when a result is stored.

The reference's users write this over their own last-axis reductions: its library
reduce stops at one axis (numba/cuda/kernels/reduction.py:217-218).  ``kernels.kvcache``
has the form that writes the keys straight into a quantised cache."""
from __future__ import annotations

from .. import _lib
from ..devicearray import stream_ptr
from ._operands import (HEAD_FORMATS, ROTATION, fast, heads, index_bytes, indices, like, on_one_device, operand, pack_heads,
                        vector, workspace, written)


def _table(x, what, stream):
    op = operand(x, what, stream=stream)
    if op[3] != _lib.FMT_F32:
        raise TypeError(f"{what} must be float32")
    if len(op[1]) != 2 or (op[2][1] != 1 and op[1][1] > 1):
        raise ValueError(f"{what} must be 2-D, (positions, half the rotated items), with unit stride in its last axis")
    return op


_NO_ANGLES = (0, 0, 0, 0, 0, 0, 0, 8)
_NO_ARRAY = (0, 0, 0, 0, 0)


def rotation(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, stream):
    """Check the arguments that all calls share: (q, k, all operands, packed b2k_rotation)."""
    given = []                           # (operand, members of b2k_heads, its weight's operand)
    for x, w, what in ((q, q_weight, "q"), (k, k_weight, "k")):
        if x is None:
            given.append((None, _NO_ARRAY, None))
            continue
        op = heads(x, what, stream=stream)
        ptr, (_, n, dim), (token, head, _), _, _, _ = op
        if w is not None:
            if not norm:
                raise ValueError("weights belong to the norm: norm=False takes none")
            w = vector(w, what + "_weight", dim, HEAD_FORMATS, "float32, float16 or bfloat16", False, stream)
        given.append((op, (ptr, token, head, n, dim), w))
    (q, q_members, qw), (k, k_members, kw) = given
    first = q if q is not None else k
    if first is None:
        raise ValueError("neither q nor k is given")
    tokens, fmt = first[1][0], first[3]
    if k is not None and (k[1][0] != tokens or k[3] != fmt):
        raise ValueError("q and k must have the same number of tokens and the same type")
    weight = qw if qw is not None else kw
    if kw is not None and kw[3] != weight[3]:
        raise TypeError("q_weight and k_weight must have the same type")
    ops = [q, k, qw, kw]
    rotary, *angles = _NO_ANGLES
    if cos is not None or sin is not None or positions is not None:
        if cos is None or sin is None or positions is None:
            raise ValueError("cos, sin and positions go together")
        c, s = _table(cos, "cos", stream), _table(sin, "sin", stream)
        if c[1] != s[1]:
            raise ValueError("cos and sin must have the same shape")
        rows, half = c[1]
        at = indices(positions, "positions", tokens, stream)
        ops += [c, s, at]
        rotary = 2 * half
        if (q is not None and rotary > q_members[4]) or (k is not None and rotary > k_members[4]):
            raise ValueError("cos and sin rotate more items than a head has")
        angles = c[0], s[0], c[2][0], s[2][0], rows, at[0], index_bytes(at)
    packed = ROTATION.pack(fmt, tokens, *q_members, *k_members, 1 if norm else 0, float(eps), qw[0] if qw is not None else 0,
                           kw[0] if kw is not None else 0, weight[3] if weight is not None else _lib.FMT_F32, rotary,
                           1 if interleaved else 0, *angles)
    return q, k, ops, packed


def result(out, source, what, stream):
    """(array to return, operand) of an optional output with an input's shape and type."""
    if source is None:
        if out is not None:
            raise ValueError(f"{what} is given without its input")
        return None, None
    if out is None:
        out = like(source, stream)
    op = operand(out, what, True, stream)
    if op[1] != source[1]:
        raise ValueError(f"{what} must have the shape {tuple(source[1])}")
    if op[3] != source[3]:
        raise TypeError(f"{what} must have its input's type")
    if op[2][2] != 1 and op[1][2] > 1:
        raise ValueError(f"{what} must have unit stride in its last axis")
    return out, op


def norm_rotate(q, k, q_weight=None, k_weight=None, cos=None, sin=None, positions=None, eps=1e-6, interleaved=False,
                norm=True, q_out=None, k_out=None, stream=0):
    """Normalise and rotate the heads of ``q`` and ``k`` in one launch; returns
    ``(q_out, k_out)``.

    :param q, k: (tokens, heads, dim) arrays of one type, float32, float16 or bfloat16
                 (``uint16`` items are bfloat16 bits), unit stride in ``dim``, any other
                 strides -- views of one projection's output, or of a heads-first array.
                 Either may be ``None``; their head counts and sizes (up to 1024) may differ.
    :param q_weight, k_weight: ``dim`` items each, shared by all heads; ``None`` for ones.
    :param cos, sin: float32 tables (positions, R/2); ``None`` (with ``positions``) to
                 leave the rotation out.
    :param positions: one int32 or int64 per token.  A token whose position is not a row of
                 the tables is padding: its rows of the outputs are left as they were.
    :param norm: ``False`` leaves the norm out.
    :param q_out, k_out: outputs; new arrays when not given (padding rows are then not
                 set).  An output may be its own input's memory; it must not overlap an
                 input in any other way, nor another output.
    :param stream: stream of the launch (0 = the default stream); arrays that other streams
                 produce must be complete or ordered before it, and arrays stay in use until
                 the launch has run, as everywhere here.

    Squares are summed in float32: a head whose squares add up to more than 3.4e38 gives
    zeros (NaN where an item itself is infinite).  The calls are not recorded for autograd:
    tensors that require grad or carry a forward tangent are refused, and the version
    counters of the tensors that a call has written rise.
    """
    status = fast.norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, q_out, k_out, stream)
    if status is not None:
        _lib.check(status)
        return q_out, k_out
    q, k, ops, packed = rotation(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, stream)
    q_out, qo = result(q_out, q, "q_out", stream)
    k_out, ko = result(k_out, k, "k_out", stream)
    on_one_device([*ops, qo, ko])
    _lib.check(_lib.lib().b2k_norm_rotate(packed, pack_heads(qo), pack_heads(ko), stream_ptr(stream)))
    written(q_out, k_out)
    return q_out, k_out


def norm_rotate_backward(q, k, q_weight, k_weight, cos, sin, positions, q_grad, k_grad, eps=1e-6, interleaved=False,
                         norm=True, dq=None, dk=None, dq_weight=None, dk_weight=None, stream=0):
    """Gradients of ``norm_rotate``: for the gradients ``q_grad``, ``k_grad`` of its outputs
    returns ``(dq, dk, dq_weight, dk_weight)``, with ``None`` where an input was ``None``.

    The weights' gradients are sums over all tokens and heads, accumulated in float32 in
    an order that depends on the shapes only, and are stored in the weights' type.  A
    padding token has zero gradients and adds nothing to the sums, whatever the weights are; so
    has a head whose squares add up to more than 3.4e38.  The sum of gradient x weight x item over
    a head is taken in float32 too.  ``dq`` and ``dk`` may be the memory of ``q_grad`` and
    ``k_grad``."""
    status = fast.norm_rotate_backward(q, k, q_weight, k_weight, cos, sin, positions, q_grad, k_grad, eps, interleaved,
                                       norm, dq, dk, dq_weight, dk_weight, stream)
    if status is not None:
        _lib.check(status)
        return dq, dk, dq_weight, dk_weight
    q, k, ops, packed = rotation(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, stream)
    grads, outs, weights = [], [], []
    for grad, x, what in ((q_grad, q, "q_grad"), (k_grad, k, "k_grad")):
        if (grad is None) != (x is None):
            raise ValueError(f"{what} and its input go together")
        op = heads(grad, what, stream=stream) if x is not None else None
        if op is not None and (op[1] != x[1] or op[3] != x[3]):
            raise ValueError(f"{what} must have its input's shape and type")
        grads.append(op)
    for out, x, what in ((dq, q, "dq"), (dk, k, "dk")):
        outs.append(result(out, x, what, stream))
    for out, w, what in ((dq_weight, ops[2], "dq_weight"), (dk_weight, ops[3], "dk_weight")):
        if w is None:
            if out is not None:
                raise ValueError(f"{what} is given without its weight")
            weights.append((None, None))
            continue
        if out is None:
            out = like(w, stream)
        weights.append((out, vector(out, what, w[1][0], (w[3],), "of its weight's type", True, stream)))
    on_one_device([*ops, *grads, *(op for _, op in outs), *(op for _, op in weights)])
    L = _lib.lib()
    scratch, need = None, 0
    if ops[2] is not None or ops[3] is not None:
        need = int(L.b2k_norm_rotate_backward_scratch_bytes(packed))
        scratch = workspace(need, stream)
    _lib.check(L.b2k_norm_rotate_backward(
        packed, pack_heads(grads[0]), pack_heads(grads[1]), pack_heads(outs[0][1]), pack_heads(outs[1][1]),
        weights[0][1][0] if weights[0][1] is not None else None,
        weights[1][1][0] if weights[1][1] is not None else None,
        scratch.data_ptr() if scratch is not None else None, need, stream_ptr(stream)))
    written(dq, dk, dq_weight, dk_weight)
    return outs[0][0], outs[1][0], weights[0][0], weights[1][0]


__all__ = ["norm_rotate", "norm_rotate_backward"]

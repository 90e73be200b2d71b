"""Routing to experts and the rows of the grouped GEMMs (device pointers, stream-ordered).

    route_device            logits -> expert ids and weights of every token
    dispatch_device         ids -> rows sorted by expert: offsets and maps
    gather_i8_device        token rows -> int8 rows of the experts (or gather_bf16_device)
    gemm.I8Plan.grouped     the experts' products, offsets read on the device
    combine_device          experts' rows -> weighted sum per token

and the gradients of a router that is trained through them: combine_backward_device,
route_backward_device.  Arguments are device buffers (anything with ``data_ptr()``, or a raw
address); nothing synchronises, allocates or computes on the host, so the chain can be captured in
a CUDA graph.  The calls go through ``smb_call_words``, since a decode step makes many of them.
"""
from __future__ import annotations

import struct

from . import capi
from .gemm import _addr, _stream_ptr

_ROUTE = struct.Struct("@10qd3q").pack
_ROUTE_BACKWARD = struct.Struct("@9qd3q").pack
_DISPATCH = struct.Struct("@11q").pack
_GATHER_BF16 = struct.Struct("@10q").pack
_GATHER_I8 = struct.Struct("@11q").pack
_COMBINE = struct.Struct("@11q").pack
_COMBINE_BACKWARD = struct.Struct("@14q").pack

# Element types by name: those that say what a buffer holds, and integers, which may be the bits of anything (16-bit
# ones are taken for bf16 unless the caller says otherwise).
_FLOATS = {"float32": capi.DTYPE_F32, "bfloat16": capi.DTYPE_BF16}
_BITS = {"uint16": capi.DTYPE_BF16, "int16": capi.DTYPE_BF16}
_kind_of_type: dict = {}   # type -> (DTYPE_*, whether the type itself says so); DTYPE_* None: no logits


def _kind_of(own):
    name = str(own).removeprefix("torch.")
    if "float" in name or "complex" in name:
        return _FLOATS.get(name), True
    return _BITS.get(name, capi.DTYPE_F32), False


def _kind(x, dtype: int | None) -> int:
    """DTYPE_* of a buffer: its own type where that is a floating one, which has to agree with `dtype`; else (integers,
    raw addresses) `dtype`, or fp32."""
    own = getattr(x, "dtype", None)
    if own is None:
        return capi.DTYPE_F32 if dtype is None else dtype
    try:
        kind, certain = _kind_of_type[own]
    except KeyError:
        kind, certain = _kind_of_type[own] = _kind_of(own)
    if kind is None:
        raise ValueError(f"logits and their gradient are fp32 or bf16, not {own}")
    if dtype is None:
        return kind
    if certain and dtype != kind:
        raise ValueError(f"dtype {dtype} does not agree with a buffer of {own}")
    return dtype


def route_device(logits, ids, weights, tokens: int, experts: int, top_k: int, dtype: int | None = None, bias=None,
                 n_groups: int = 1, top_groups: int = 1, flags: int = 0, scale: float = 1.0, ld: int | None = None,
                 stream=None) -> None:
    """ids [tokens, top_k] int32 and weights [tokens, top_k] fp32 from logits [tokens, experts]; closed
    slots hold id -1, weight 0.  `flags`: capi.ROUTE_*.  The logits are fp32 or bf16; `dtype` (capi.DTYPE_*) says
    which where the buffer does not (a raw address, integers; default fp32), and has to agree with it where it does."""
    capi.call_words(capi.CALL_MOE_ROUTE, _ROUTE(
        _addr(logits), _kind(logits, dtype), experts if ld is None else ld, _addr(bias), tokens, experts, top_k, n_groups,
        top_groups, flags, scale, _addr(ids), _addr(weights), _stream_ptr(stream)), 14)


def route_backward_device(logits, ids, grad_weights, grad_logits, tokens: int, experts: int, top_k: int,
                          dtype: int | None = None, flags: int = 0, scale: float = 1.0, ld: int | None = None,
                          ld_grad: int | None = None, stream=None) -> None:
    """grad_logits [tokens, experts], in the logits' type, for the ids of the forward pass.  `dtype` as above."""
    kind = _kind(logits, dtype)
    if getattr(grad_logits, "dtype", None) is not None:
        _kind(grad_logits, kind)
    capi.call_words(capi.CALL_MOE_ROUTE_BACKWARD, _ROUTE_BACKWARD(
        _addr(logits), kind, experts if ld is None else ld, _addr(ids), _addr(grad_weights), tokens, experts, top_k, flags,
        scale, _addr(grad_logits), experts if ld_grad is None else ld_grad, _stream_ptr(stream)), 13)


def max_rows(tokens: int, top_k: int, groups: int, align: int = 1) -> int:
    """Rows the sorted buffers must have room for."""
    return int(capi.lib().smb_moe_max_rows(tokens, top_k, groups, align))


def dispatch_device(ids, offsets, row_of_slot, slot_of_row, tokens: int, top_k: int, groups: int, max_rows: int,
                    align: int = 1, mtile_group=None, stream=None) -> None:
    """Stable sort of the slots by expert: offsets [groups + 1], row_of_slot [tokens, top_k], slot_of_row
    [max_rows], and with align = 256 the tile map of Bf16Plan.grouped."""
    capi.call_words(capi.CALL_MOE_DISPATCH, _DISPATCH(
        _addr(ids), tokens, top_k, groups, align, max_rows, _addr(offsets), _addr(row_of_slot), _addr(slot_of_row),
        _addr(mtile_group), _stream_ptr(stream)), 11)


def gather_bf16_device(x, row_of_slot, out, tokens: int, top_k: int, width: int, max_rows: int, ld_x: int | None = None,
                       ld_out: int | None = None, stream=None) -> None:
    """Row row_of_slot[t, j] of `out` [max_rows, width] becomes row t of x."""
    capi.call_words(capi.CALL_MOE_GATHER_BF16, _GATHER_BF16(
        _addr(x), width if ld_x is None else ld_x, _addr(row_of_slot), tokens, top_k, width, max_rows, _addr(out),
        width if ld_out is None else ld_out, _stream_ptr(stream)), 10)


def gather_i8_device(x, row_of_slot, codes, scales, tokens: int, top_k: int, width: int, max_rows: int,
                     ld_x: int | None = None, ld_bytes: int | None = None, stream=None) -> None:
    """The same with the rows quantised: int8 codes [max_rows, width] and scales [max_rows]."""
    capi.call_words(capi.CALL_MOE_GATHER_I8, _GATHER_I8(
        _addr(x), width if ld_x is None else ld_x, _addr(row_of_slot), tokens, top_k, width, max_rows, _addr(codes),
        width if ld_bytes is None else ld_bytes, _addr(scales), _stream_ptr(stream)), 11)


def combine_device(rows, row_of_slot, weights, y, tokens: int, top_k: int, width: int, max_rows: int,
                   ld_rows: int | None = None, ld_y: int | None = None, stream=None) -> None:
    """y[t] = sum_j weights[t, j] * rows[row_of_slot[t, j]]; weights None: plain sum (the gradient of a gather)."""
    capi.call_words(capi.CALL_MOE_COMBINE, _COMBINE(
        _addr(rows), width if ld_rows is None else ld_rows, _addr(row_of_slot), _addr(weights), tokens, top_k, width, max_rows,
        _addr(y), width if ld_y is None else ld_y, _stream_ptr(stream)), 11)


def combine_backward_device(grad_y, rows, row_of_slot, weights, grad_rows, grad_weights, tokens: int, top_k: int,
                            width: int, max_rows: int, ld_grad_y: int | None = None, ld_rows: int | None = None,
                            ld_grad_rows: int | None = None, stream=None) -> None:
    """Gradients of combine_device: of the rows (those that a slot names) and, unless None, of the weights."""
    capi.call_words(capi.CALL_MOE_COMBINE_BACKWARD, _COMBINE_BACKWARD(
        _addr(grad_y), width if ld_grad_y is None else ld_grad_y, _addr(rows), width if ld_rows is None else ld_rows,
        _addr(row_of_slot), _addr(weights), tokens, top_k, width, max_rows, _addr(grad_rows),
        width if ld_grad_rows is None else ld_grad_rows, _addr(grad_weights), _stream_ptr(stream)), 14)

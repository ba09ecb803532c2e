"""Rotary positions with one or several axes, and the write of the turned rows into a paged cache (gfx950): one launch
between the fused query/key/value projection of a layer and its attention (kernels/paged_attention.py)."""
from __future__ import annotations

import struct

import torch

from .. import _lib
from .paged_attention import Plans, TYPES, check_batch, check_cache, check_device, check_rows, strides

# ssmoe_rope_append_args
_ARGS = struct.Struct("@3P6qPPq7Pq12if0q")


def pack_args(q=0, k=0, v=0, q_row=0, q_head=0, k_row=0, k_head=0, v_row=0, v_head=0, q_out=0, positions=0, pos_stride=0,
              inv_freq=0, axis=0, k_pages=0, v_pages=0, cu_rows=0, kv_len=0, table=0, n_pages=0, rows=0, seqs=0, max_rows=0,
              heads=0, kv_heads=0, dim=0, page=0, width=0, rot=0, axes=0, adjacent=0, type=0, factor=1.0) -> bytes:
    """The C struct of a call, which the library reads during the call only."""
    return _ARGS.pack(q, k, v, q_row, q_head, k_row, k_head, v_row, v_head, q_out, positions, pos_stride, inv_freq, axis,
                      k_pages, v_pages, cu_rows, kv_len, table, n_pages, rows, seqs, max_rows, heads, kv_heads, dim, page,
                      width, rot, axes, adjacent, type, factor)


_plans = Plans()


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, cu_rows: torch.Tensor, kv_len: torch.Tensor,
                table: torch.Tensor, max_rows: int, axis: torch.Tensor | None = None, adjacent: bool = False,
                factor: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q [rows, heads, dim] and k [rows, kv_heads, dim] by their rows' positions, writes k and v [rows, kv_heads,
    dim] into the cache at their sequence's places (row i of n at token kv_len - n + i) and returns the turned q.

    positions int32 [rows] or [axes, rows]; inv_freq fp64 [rot / 2]; the angle of frequency i is positions[axis[i], row] *
    inv_freq[i], axis int32 [rot / 2] (None: axis 0; an entry outside [0, axes) raises SSMOE_ERR_BATCH in the device status). The pair turned by it is (i, i + rot / 2), or (2 i, 2 i + 1) with
    `adjacent`; elements from rot on are copied. cos and sin are multiplied by `factor`. q, k and v may be views into
    one projection (strides multiples of 8 elements); `out` may be q itself where q is contiguous; else it and the pages overlap
    each other and the inputs nowhere. Rows past cu_rows[-1] are left as they were."""
    max_rows = int(max_rows)
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, positions.shape,
           positions.dtype, positions.is_contiguous(), inv_freq.shape, inv_freq.dtype, inv_freq.is_contiguous(), k_pages.shape,
           k_pages.dtype, k_pages.is_contiguous(), v_pages.shape, v_pages.dtype, v_pages.is_contiguous(), cu_rows.shape,
           cu_rows.stride(), cu_rows.dtype, kv_len.shape, kv_len.stride(), kv_len.dtype, table.shape, table.dtype,
           table.is_contiguous(), max_rows, None if axis is None else (axis.shape, axis.stride(), axis.dtype), factor)
    plan = _plans.get(key)
    if plan is None:
        if not abs(factor) < 1e30:
            raise ValueError("factor must be finite and below 1e30")
        plan = _plans.keep(key, _plan(q, k, v, positions, inv_freq, k_pages, v_pages, cu_rows, kv_len, table, max_rows, axis))
    row_strides, sizes, rot, axes, kind, shape = plan
    dev = check_device(q, k, v, positions, inv_freq, k_pages, v_pages, cu_rows, kv_len, table, axis, out)
    q_at, k_at, v_at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (q_at | k_at | v_at) % 16:
        raise ValueError("q, k and v need 16-byte alignment")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {q.dtype} {tuple(shape)}")
    args = _ARGS.pack(q_at, k_at, v_at, *row_strides, out.data_ptr(), positions.data_ptr(), shape[0], inv_freq.data_ptr(),
                      0 if axis is None else axis.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), cu_rows.data_ptr(),
                      kv_len.data_ptr(), table.data_ptr(), *sizes, rot, axes, 1 if adjacent else 0, kind, float(factor))
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ssmoe_rope_append(args, _lib.raw_stream(dev)))
    return out


def _plan(q, k, v, positions, inv_freq, k_pages, v_pages, cu_rows, kv_len, table, max_rows, axis):
    """Checks a call's shapes, types and strides: (strides, sizes, rot, axes, type, shape of out)."""
    n_pages, kv_heads, page, dim = check_cache(k_pages, v_pages)
    seqs, width = check_batch(cu_rows, kv_len, table, max_rows)
    dtype = k_pages.dtype
    check_rows("q", q, None, dim, dtype)
    check_rows("k", k, kv_heads, dim, dtype)
    check_rows("v", v, kv_heads, dim, dtype)
    rows, heads = q.shape[0], q.shape[1]
    if k.shape[0] != rows or v.shape[0] != rows:
        raise ValueError(f"q, k and v must have the same rows, got {rows}, {k.shape[0]} and {v.shape[0]}")
    if heads < 1 or heads % kv_heads:
        raise ValueError(f"q has {heads} heads, not a positive multiple of the cache's {kv_heads}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous fp64 [rot / 2]")
    rot = 2 * inv_freq.numel()
    if rot < 16 or rot % 16 or rot > dim:
        raise ValueError(f"rot must be a multiple of 16 in [16, {dim}], got {rot}")
    if positions.dtype != torch.int32 or positions.dim() not in (1, 2) or positions.shape[-1] != rows \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int32 [{rows}] or [axes, {rows}]")
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    if axes < 1:
        raise ValueError("positions must have at least one axis")
    if axis is not None and (axis.dtype != torch.int32 or tuple(axis.shape) != (rot // 2,) or not axis.is_contiguous()):
        raise ValueError(f"axis must be contiguous int32 [{rot // 2}]")
    return ((*strides(q), *strides(k), *strides(v)),
            (n_pages, rows, seqs, max_rows, heads, kv_heads, dim, page, width), rot, axes, TYPES[dtype], q.shape)

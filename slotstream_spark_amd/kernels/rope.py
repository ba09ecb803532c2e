"""Rotary positions with one or several axes, and the write of the turned rows into a paged cache (gfx950): one launch
between the fused query/key/value projection of a layer and its attention (kernels/paged_attention.py)."""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .paged_attention import TYPES, check_batch, check_cache, check_device, check_rows, strides

_P, _I, _I64, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class _Args(ctypes.Structure):
    _fields_ = ([(n, _P) for n in ("q", "k", "v")]
                + [(n, _I64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")]
                + [("q_out", _P), ("positions", _P), ("pos_stride", _I64)]
                + [(n, _P) for n in ("inv_freq", "axis", "k_pages", "v_pages", "cu_rows", "kv_len", "table")]
                + [("n_pages", _I64)]
                + [(n, _I) for n in ("rows", "seqs", "max_rows", "heads", "kv_heads", "dim", "page", "width", "rot", "axes",
                                     "adjacent", "type")]
                + [("factor", _F)])


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, cu_rows: torch.Tensor, kv_len: torch.Tensor,
                table: torch.Tensor, max_rows: int, axis: torch.Tensor | None = None, adjacent: bool = False,
                factor: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q [rows, heads, dim] and k [rows, kv_heads, dim] by their rows' positions, writes k and v [rows, kv_heads,
    dim] into the cache at their sequence's places (row i of n at token kv_len - n + i) and returns the turned q.

    positions int32 [rows] or [axes, rows]; inv_freq fp64 [rot / 2]; the angle of frequency i is positions[axis[i], row] *
    inv_freq[i], axis int32 [rot / 2] (None: axis 0). The pair turned by it is (i, i + rot / 2), or (2 i, 2 i + 1) with
    `adjacent`; elements from rot on are copied. cos and sin are multiplied by `factor`. q, k and v may be views into
    one projection (strides multiples of 8 elements); `out` may be q itself where q is contiguous. Rows past
    cu_rows[-1] are left as they were."""
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
    dev = check_device(q, k, v, positions, inv_freq, k_pages, v_pages, cu_rows, kv_len, table, axis, out)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=dtype, device=dev)
    elif out.dtype != dtype or tuple(out.shape) != (rows, heads, dim) or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {(rows, heads, dim)}")
    a = _Args(q.data_ptr(), k.data_ptr(), v.data_ptr(), *strides(q), *strides(k), *strides(v), out.data_ptr(),
              positions.data_ptr(), rows, inv_freq.data_ptr(), _lib.ptr(axis), k_pages.data_ptr(), v_pages.data_ptr(),
              cu_rows.data_ptr(), kv_len.data_ptr(), table.data_ptr(), n_pages, rows, seqs, int(max_rows), heads, kv_heads,
              dim, page, width, rot, axes, int(bool(adjacent)), TYPES[dtype], float(factor))
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().ssmoe_rope_append(ctypes.byref(a), _lib.stream_of(q)))
    return out

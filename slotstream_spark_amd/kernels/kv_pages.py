"""Moving pages of a key-value cache (gfx950): the copies of a fork and the moves of a compaction. memory/kv_pages.py
keeps the pages' owners and calls this."""
from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import check_device


def move_pages(k: torch.Tensor, v: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               table: torch.Tensor | None = None) -> None:
    """Page dst[i] := page src[i] of every layer; k and v are [layers, n_pages, ...] of the same bytes a page. src and dst
    int32 [n] on the GPU. Entries of `table` (int32, any shape) that name src[i] name dst[i] afterwards. No page may be twice
    in dst, nor in both src and dst (its contents would be undefined); k, v and the table overlap each other, src and dst nowhere; ids outside the cache are skipped and raise
    SSMOE_ERR_PAGE in the device status."""
    if k.dim() < 3 or k.shape[:2] != v.shape[:2] or k.dtype != v.dtype or k.numel() != v.numel():
        raise ValueError("k and v must be [layers, n_pages, ...] of one type and size")
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("k and v must be contiguous")
    for name, t in (("src", src), ("dst", dst)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [n]")
    if src.numel() != dst.numel():
        raise ValueError(f"src and dst must have the same length, got {src.numel()} and {dst.numel()}")
    if table is not None and (table.dtype != torch.int32 or not table.is_contiguous()):
        raise ValueError("table must be a contiguous int32 tensor")
    layers, n_pages = k.shape[:2]
    if layers < 1 or n_pages < 1:
        raise ValueError("the cache holds no page")
    page_bytes = k.numel() // (layers * n_pages) * k.element_size()
    if page_bytes < 2048 or page_bytes % 2048:
        raise ValueError(f"a page must have a positive multiple of 2048 bytes, got {page_bytes}")
    dev = check_device(k, v, src, dst, table)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ssmoe_move_pages(k.data_ptr(), v.data_ptr(), layers, n_pages, page_bytes, src.data_ptr(),
                                               dst.data_ptr(), src.numel(), _lib.ptr(table),
                                               0 if table is None else table.numel(), _lib.raw_stream(dev)))

"""Attention of a batch's new rows over a paged key-value cache (gfx950), from one decoded token to prompt chunks.

    out_i = sum_j softmax_j(scale q_i . k_j) v_j    over the tokens j <= p of the row's sequence, p the row's position;
                                                    under a window those with p - j < window or j < sinks

The cache of a layer is k_pages [n_pages, kv_heads, page, dim] and v_pages [n_pages, kv_heads, dim, page] (a dimension's
tokens side by side). The batch is described by three int32 GPU tensors that the kernels read, so that a captured call
follows their contents: cu_rows [seqs + 1] (the rows of sequence s), kv_len [seqs] (its tokens in the cache, the new rows the
last of them) and table [seqs, width] (its pages; -1 where none is held). memory/kv_pages.py keeps such a cache.

Pages may be of e4m3 numbers (torch.float8_e4m3fn) with `scales` uint8 [n_pages, kv_heads, 2, page], as rope_append writes them: a
token's keys are their numbers times 2^(scales[.., 0, t] - 127), its values times 2^(scales[.., 1, t] - 127). q is bf16 then.
Rows may be those of a tree of drafts, `tree` int64 [rows] saying which of its sequence's rows each one sees (kernels/tree.py).

The reference's attention (QSA over its own caches, kernels/vendored.py:105-118) has no counterpart here; this is
the plain causal form a layer or the draft head (engine/mtp.py:209-227) can be given instead.
"""
from __future__ import annotations

import math
import struct

import torch

from .. import _lib

TYPES = {torch.bfloat16: 0, torch.float16: 1}
E4M3 = torch.float8_e4m3fn
TREE_ROWS = 64   # rows of one sequence's tree
PAGES = (16, 32, 64, 128, 256)
DIMS = (64, 128, 256)

# ssmoe_paged_attention_args: 3 + 8 pointers and strides, 2 int64, 11 int, a float (padded to 8 bytes)
_ARGS = struct.Struct("@Pqq8Pqq11if0q")


def pack_args(q=0, q_row=0, q_head=0, k_pages=0, v_pages=0, cu_rows=0, kv_len=0, table=0, out=0, lse=0, ws=0, ws_bytes=0,
              n_pages=0, rows=0, seqs=0, max_rows=0, heads=0, kv_heads=0, dim=0, page=0, width=0, window=0, sinks=0, type=0,
              scale=0.0) -> bytes:
    """The C struct of a call, which the library reads during the call only."""
    return _ARGS.pack(q, q_row, q_head, k_pages, v_pages, cu_rows, kv_len, table, out, lse, ws, ws_bytes, n_pages, rows,
                      seqs, max_rows, heads, kv_heads, dim, page, width, window, sinks, type, scale)


class Plans(dict):
    """What the checks of a call's shapes, types and strides found, by those: nothing of the tensors themselves is kept.
    Emptied when it holds many (a serving loop meets a few)."""

    def keep(self, key, plan):
        if len(self) >= 4096:
            self.clear()
        self[key] = plan
        return plan


_plans = Plans()


def check_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor | None = None) -> tuple[int, int, int, int]:
    """(n_pages, kv_heads, page, dim) of a layer's cache, with `scales` of one in e4m3."""
    if k_pages.dim() != 4 or v_pages.dim() != 4:
        raise ValueError("k_pages must be [n_pages, kv_heads, page, dim] and v_pages [n_pages, kv_heads, dim, page]")
    n, h, page, dim = k_pages.shape
    if tuple(v_pages.shape) != (n, h, dim, page):
        raise ValueError(f"v_pages must be {(n, h, dim, page)}, got {tuple(v_pages.shape)}")
    if page not in PAGES or dim not in DIMS:
        raise ValueError(f"pages hold 16, 32, 64, 128 or 256 tokens of 64, 128 or 256 dimensions, got {page} of {dim}")
    if scales is not None:
        if k_pages.dtype != E4M3 or v_pages.dtype != E4M3:
            raise ValueError(f"scales belong to k_pages and v_pages of {E4M3}, got {k_pages.dtype} and {v_pages.dtype}")
        if scales.dtype != torch.uint8 or tuple(scales.shape) != (n, h, 2, page) or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous uint8 {(n, h, 2, page)}")
    elif k_pages.dtype not in TYPES or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"k_pages and v_pages must both be bf16 or fp16 (or {E4M3} with scales), got {k_pages.dtype} and "
                         f"{v_pages.dtype}")
    if not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise ValueError("k_pages and v_pages must be contiguous")
    if n < 1:
        raise ValueError("the cache holds no page")
    return n, h, page, dim


def check_batch(cu_rows: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor, max_rows: int) -> tuple[int, int]:
    """(seqs, width) of a batch."""
    for name, t in (("cu_rows", cu_rows), ("kv_len", kv_len), ("table", table)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError("table must be [seqs, width]")
    seqs = table.shape[0]
    if tuple(cu_rows.shape) != (seqs + 1,) or tuple(kv_len.shape) != (seqs,):
        raise ValueError(f"cu_rows must be [{seqs + 1}] and kv_len [{seqs}], got {tuple(cu_rows.shape)} and "
                         f"{tuple(kv_len.shape)}")
    if not 1 <= max_rows < 1 << 31:
        raise ValueError("max_rows must be >= 1 and below 2^31")
    return seqs, table.shape[1]


def check_rows(name: str, t: torch.Tensor, heads: int | None, dim: int, dtype) -> None:
    """t [rows, heads, dim], its dimensions contiguous and its strides multiples of 8 elements."""
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {dim}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} like the cache, got {t.dtype}")
    if t.numel() and (t.stride(2) != 1 or (t.shape[0] > 1 and t.stride(0) % 8) or (t.shape[1] > 1 and t.stride(1) % 8)):
        raise ValueError(f"{name} needs contiguous dimensions and strides that are multiples of 8 elements")


def strides(t: torch.Tensor) -> tuple[int, int]:
    """Row and head stride of a [rows, heads, dim] tensor (0 where there is one only)."""
    return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def check_device(*tensors) -> int:
    """The index of the GPU that all of them (None apart) are on."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != dev or dev < 0):
            raise ValueError("all tensors must be on the same GPU")
    return dev


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, cu_rows: torch.Tensor,
                    kv_len: torch.Tensor, table: torch.Tensor, max_rows: int, window: int = 0, sinks: int = 0,
                    scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    scales: torch.Tensor | None = None, tree: torch.Tensor | None = None) -> torch.Tensor:
    """q [rows, heads, dim] -> [rows, heads, dim] of q's type. `max_rows` bounds the rows of one sequence. window 0: every
    token up to the row's own; else the last `window` of them and the first `sinks`. scale: 1 / sqrt(dim) unless given. One kernel
    for the call: that of few rows up to a max_rows of 8 (over e4m3 pages and for trees also where max_rows times the heads of a key head is
    small or the table short), else that of many: single tokens in a batch with a prompt go through the prompt's, without
    the split over their length and the bits of a call of few rows. Two calls over one q and `out`, with cu_rows[:m + 1] and
    cu_rows[m:], serve them apart (rows outside a call's cu_rows are left alone).
    `lse` fp32 [rows, heads] receives ln sum_j exp(scale q_i . k_j). A row that sees nothing is 0, its lse -inf; rows past
    cu_rows[-1] are left as they were in `out` and `lse`, which must not overlap each other nor anything that the call reads.
    `scales`: the pages are of e4m3 numbers. `tree`: row i sees the tokens before its sequence's rows and the rows j of it with bit j
    of tree[i] (tree_masks' words: itself and its ancestors), at most 64 rows a sequence; its position under a window, which must be
    at least max_rows, is that of as many rows as it sees, one at least. A tree's rows have no bits of their own: the order of its sums goes by where
    its tokens lie, so a row of a tree and the same token decoded alone agree as far as fp32 sums do.
    Capturable; workspaces come from torch's allocator at each call, so calls and captured graphs never share one."""
    max_rows, window, sinks = int(max_rows), int(window), int(sinks)
    key = (q.shape, q.stride(), q.dtype, k_pages.shape, k_pages.dtype, k_pages.is_contiguous(), v_pages.shape, v_pages.dtype,
           v_pages.is_contiguous(), cu_rows.shape, cu_rows.stride(), cu_rows.dtype, kv_len.shape, kv_len.stride(), kv_len.dtype,
           table.shape, table.dtype, table.is_contiguous(), max_rows, window, sinks, scale)
    ext = scales is not None or tree is not None
    if ext:
        key += (scales is not None and (scales.shape, scales.dtype, scales.is_contiguous()),
                tree is not None and (tree.shape, tree.dtype, tree.is_contiguous()))
    plan = _plans.get(key)
    if plan is None:
        plan = _plans.keep(key, _plan(q, k_pages, v_pages, cu_rows, kv_len, table, max_rows, window, sinks, scale, scales, tree))
    head, sizes, tail, nb, shape = plan
    dev = check_device(q, k_pages, v_pages, cu_rows, kv_len, table, out, lse)
    if ext:
        check_device(q, scales, tree)
    q_at = q.data_ptr()
    if q_at % 16:
        raise ValueError("q needs 16-byte alignment")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {q.dtype} {tuple(shape)}")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != shape[:2] or not lse.is_contiguous()):
        raise ValueError(f"lse must be contiguous fp32 {tuple(shape[:2])}")
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb else None
    args = _ARGS.pack(q_at, *head, k_pages.data_ptr(), v_pages.data_ptr(), cu_rows.data_ptr(), kv_len.data_ptr(),
                      table.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if ws is None else ws.data_ptr(),
                      nb, *sizes, *tail)
    with _lib.on_device(dev):
        if ext:
            _lib.check(_lib.lib().ssmoe_paged_attention_ext(args, _lib.ptr(scales), _lib.ptr(tree), _lib.raw_stream(dev)))
        else:
            _lib.check(_lib.lib().ssmoe_paged_attention(args, _lib.raw_stream(dev)))
    return out


def _plan(q, k_pages, v_pages, cu_rows, kv_len, table, max_rows, window, sinks, scale, scales=None, tree=None):
    """Checks a call's shapes, types and strides: (strides of q, sizes, mask and scale, workspace bytes, shape of out)."""
    n_pages, kv_heads, page, dim = check_cache(k_pages, v_pages, scales)
    seqs, width = check_batch(cu_rows, kv_len, table, max_rows)
    check_rows("q", q, None, dim, k_pages.dtype if scales is None else torch.bfloat16)
    if tree is not None:
        if tree.dtype != torch.int64 or tuple(tree.shape) != (q.shape[0],) or not tree.is_contiguous():
            raise ValueError(f"tree must be contiguous int64 [{q.shape[0]}]")
        if max_rows > TREE_ROWS:
            raise ValueError(f"a tree has at most {TREE_ROWS} rows of a sequence, max_rows is {max_rows}")
        if 0 < window < max_rows:
            raise ValueError(f"with a tree the window must hold max_rows rows: {window} of {max_rows}")
    rows, heads = q.shape[0], q.shape[1]
    if heads < 1 or heads % kv_heads:
        raise ValueError(f"q has {heads} heads, not a positive multiple of the cache's {kv_heads}")
    head = strides(q)
    sizes = (n_pages, rows, seqs, max_rows, heads, kv_heads, dim, page, width)
    tail = (window, sinks, TYPES[q.dtype], 1.0 / math.sqrt(dim) if scale is None else float(scale))
    if not 0 <= window < 1 << 31 or not 0 <= sinks < 1 << 31 or not 0 < tail[3] < 1e30:
        raise ValueError("need 0 <= window, sinks < 2^31 and 0 < scale < 1e30")
    L = _lib.lib()
    nb = L.ssmoe_paged_attention_ext_workspace_bytes(_ARGS.pack(0, *head, *(0,) * 8, 0, *sizes, *tail), scales is not None,
                                                     tree is not None)
    if nb < 0:
        raise ValueError(L.ssmoe_last_error().decode(errors="replace"))
    return head, sizes, tail, nb, q.shape

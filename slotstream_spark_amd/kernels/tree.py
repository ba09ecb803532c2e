"""Trees of drafted tokens over a paged cache (gfx950): which rows a row sees, the greedy round of a tree, and the move of the
accepted branch in the cache.

A round with a tree, for each of a batch's sequences: row 0 is the pending token, every other row a draft behind its parent among the
rows before it, at most 64 rows. The rows are written behind the cache in their order (rope_append, with positions that go by
depth), each sees the cache, its ancestors and itself (paged_attention with `tree`), the target's choices decide how far a branch is
followed, and that branch's keys and values move up to where its tokens belong.

    masks, positions = tree_masks(parents, cu_rows, kv_len, max_rows)
    q = rope_append(q, k, v, positions, ...);  o = paged_attention(q, ..., tree=masks)            (every layer)
    accepted = accept_tree(logits, tokens, parents, cu_rows, max_rows)
    keep_rows(k, v, cu_rows, kv_len, table, accepted)                                            (all layers at once)

The reference verifies chains (engine/generate.py:208-229); a chain is the tree in which every row's parent is the row before it.
"""
from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import DIMS, E4M3, PAGES, TREE_ROWS, TYPES, Plans, check_batch, check_device

_plans = Plans()


def _check_tree(rows: int, cu_rows: torch.Tensor, max_rows: int, **ints) -> int:
    for name, t in ints.items():
        if t.dtype != torch.int32 or tuple(t.shape) != (rows,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [{rows}]")
    if cu_rows.dtype != torch.int32 or cu_rows.dim() != 1 or cu_rows.numel() < 1 or not cu_rows.is_contiguous():
        raise ValueError("cu_rows must be contiguous int32 [seqs + 1]")
    if not 1 <= max_rows <= TREE_ROWS:
        raise ValueError(f"a tree has 1 to {TREE_ROWS} rows of a sequence, max_rows is {max_rows}")
    return cu_rows.numel() - 1


def tree_masks(parents: torch.Tensor, cu_rows: torch.Tensor, kv_len: torch.Tensor, max_rows: int,
               masks: torch.Tensor | None = None, positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """parents int32 [rows] (a row's parent among its sequence's rows, before it; of a first row not read) -> (masks int64 [rows],
    positions int32 [rows]): bit j of a row's word says that it sees row j of its sequence, its position is kv_len - rows + its depth.
    A parent that is no earlier row is taken as none and raises SSMOE_ERR_BATCH in the device status. Rows past cu_rows[-1] are left
    as they were (zero in new tensors). Capturable."""
    max_rows, rows = int(max_rows), parents.shape[0] if parents.dim() == 1 else -1
    seqs = _check_tree(rows, cu_rows, max_rows, parents=parents)
    if kv_len.dtype != torch.int32 or tuple(kv_len.shape) != (seqs,) or not kv_len.is_contiguous():
        raise ValueError(f"kv_len must be contiguous int32 [{seqs}]")
    masks = torch.zeros(rows, dtype=torch.int64, device=parents.device) if masks is None else masks
    positions = torch.zeros(rows, dtype=torch.int32, device=parents.device) if positions is None else positions
    for name, t, kind in (("masks", masks, torch.int64), ("positions", positions, torch.int32)):
        if t.dtype != kind or tuple(t.shape) != (rows,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {kind} [{rows}]")
    dev = check_device(parents, cu_rows, kv_len, masks, positions)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ssmoe_tree_masks(parents.data_ptr(), cu_rows.data_ptr(), kv_len.data_ptr(), masks.data_ptr(),
                                               positions.data_ptr(), rows, seqs, max_rows, _lib.raw_stream(dev)))
    return masks, positions


def accept_tree(target: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_rows: torch.Tensor, max_rows: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The greedy round: target fp32 [rows, vocab], tokens int32 [rows] (a row's own token), parents as tree_masks takes them ->
    int32 [seqs, 4 + 2 max_rows] on the device: n_accept, n_emit, 0, flags, the chosen tokens [max_rows], the branch's rows [max_rows],
    -1 where there is none.

    From row 0 on, a row's choice is the first maximum of its logits, and the branch goes on to the first row behind it whose token is that
    choice. A row with a logit that is not finite ends it before its choice (flag 1). Workspaces come from torch's allocator at each call.
    `out` overlaps nothing that the call reads. Capturable."""
    max_rows = int(max_rows)
    key = (target.shape, target.dtype, target.is_contiguous(), tokens.shape, tokens.dtype, tokens.is_contiguous(), parents.shape,
           parents.dtype, parents.is_contiguous(), cu_rows.shape, cu_rows.dtype, cu_rows.is_contiguous(), max_rows)
    plan = _plans.get(key)
    if plan is None:
        plan = _plans.keep(key, _accept_plan(target, tokens, parents, cu_rows, max_rows))
    rows, vocab, seqs, nb, shape = plan
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=target.device)
    elif out.dtype != torch.int32 or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous int32 {tuple(shape)}")
    dev = check_device(target, tokens, parents, cu_rows, out)
    ws = torch.empty(nb, dtype=torch.uint8, device=target.device) if nb else None
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ssmoe_accept_tree(target.data_ptr(), tokens.data_ptr(), parents.data_ptr(), cu_rows.data_ptr(), rows, seqs,
                                                max_rows, vocab, _lib.ptr(ws), nb, out.data_ptr(), _lib.raw_stream(dev)))
    return out


def _accept_plan(target, tokens, parents, cu_rows, max_rows):
    """Checks a call's shapes and types: (rows, vocab, seqs, workspace bytes, shape of out)."""
    if target.dim() != 2 or target.dtype != torch.float32 or not target.is_contiguous() or target.shape[1] < 1:
        raise ValueError("target must be contiguous fp32 [rows, vocab]")
    rows, vocab = target.shape
    seqs = _check_tree(rows, cu_rows, max_rows, tokens=tokens, parents=parents)
    L = _lib.lib()
    nb = L.ssmoe_accept_tree_workspace_bytes(rows, seqs, max_rows, vocab)
    if nb < 0:
        raise ValueError(L.ssmoe_last_error().decode(errors="replace"))
    return rows, vocab, seqs, nb, torch.Size((seqs, 4 + 2 * max_rows))


def keep_rows(k: torch.Tensor, v: torch.Tensor, cu_rows: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor,
              accepted: torch.Tensor, scales: torch.Tensor | None = None) -> None:
    """Token kv_len - rows + d of every sequence := its token kv_len - rows + path[d], for d up to n_accept, in all layers: k [layers,
    n_pages, kv_heads, page, dim], v [layers, n_pages, kv_heads, dim, page], of e4m3 with scales uint8 [layers, n_pages, kv_heads, 2,
    page]. cu_rows, kv_len and table are the round's (cu_rows[m:], kv_len[m:] and table[m:] of a larger batch among them); accepted int32
    [seqs, 4 + 2 max_rows] is accept_tree's result. What lies behind the moved tokens is not to be read any more. Rows of pages that others
    hold too are not to be moved (KVPages.extend copies those); values are written in whole pieces of 8 tokens, the others of a piece as
    they were, so nothing else may write to these pages meanwhile.
    A path that does not rise, or names no row of the sequence, is followed up to there and raises SSMOE_ERR_BATCH in the device
    status. Capturable."""
    if k.dim() != 5 or v.dim() != 5:
        raise ValueError("k must be [layers, n_pages, kv_heads, page, dim] and v [layers, n_pages, kv_heads, dim, page]")
    layers, n, h, page, dim = k.shape
    if tuple(v.shape) != (layers, n, h, dim, page):
        raise ValueError(f"v must be {(layers, n, h, dim, page)}, got {tuple(v.shape)}")
    if page not in PAGES or dim not in DIMS or min(layers, n, h) < 1:
        raise ValueError(f"pages hold 16, 32, 64, 128 or 256 tokens of 64, 128 or 256 dimensions, got {tuple(k.shape)}")
    if v.dtype != k.dtype or (k.dtype != E4M3 if scales is not None else k.dtype not in TYPES):
        raise ValueError(f"k and v must both be bf16 or fp16, or {E4M3} with scales, got {k.dtype} and {v.dtype}")
    if scales is not None and (scales.dtype != torch.uint8 or tuple(scales.shape) != (layers, n, h, 2, page)
                               or not scales.is_contiguous()):
        raise ValueError(f"scales must be contiguous uint8 {(layers, n, h, 2, page)}")
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("k and v must be contiguous")
    seqs, width = check_batch(cu_rows, kv_len, table, 1)
    if accepted.dtype != torch.int32 or accepted.dim() != 2 or accepted.shape[0] != seqs or not accepted.is_contiguous() \
            or accepted.shape[1] % 2 or not 6 <= accepted.shape[1] <= 4 + 2 * TREE_ROWS:
        raise ValueError(f"accepted must be contiguous int32 [{seqs}, 4 + 2 max_rows]")
    max_rows = (accepted.shape[1] - 4) // 2
    most = 2 ** 31 - 1   # rows of the call: nothing is at a row's number, and the views cu_rows[m:] of a batch begin anywhere
    dev = check_device(k, v, cu_rows, kv_len, table, accepted, scales)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ssmoe_keep_rows(
            k.data_ptr(), v.data_ptr(), _lib.ptr(scales), layers, n, h, page, dim, k.element_size(), cu_rows.data_ptr(),
            kv_len.data_ptr(), table.data_ptr(), width, accepted.data_ptr(), most, seqs, max_rows, _lib.raw_stream(dev)))

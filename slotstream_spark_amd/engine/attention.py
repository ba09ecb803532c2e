"""One attention layer over a paged key-value cache, and a sequence's place in it.

AttentionLayer is the segment between the norm before an attention layer and its residual: the fused query/key/value
projection, optional per-head norms of q and k, rotary positions with the cache write (ssmoe_rope_append), the attention of the
new rows over the pages (ssmoe_paged_attention) and the output projection. Calls of up to FEW_ROWS rows project on the
GEMV (each row with the bits it has alone, as the verify layer's rows), longer ones on the bf16 GEMM. It stands where the
reference runs QSA (seg_attn, model/layers.py; the head's, engine/mtp.py:209-227), with plain causal attention, a sliding
window with first tokens that stay visible, and one or several position axes.

SeqCache is one sequence of a KVPages as an engine loop holds it: `pos` and `last` are what rollback() sets on the caches of a
SeqState (engine/rollback.py:26-41), and the batch tensors stay in place, so that a captured step follows them. A MoEStack keeps
`pos` at its own position; the draft head, whose forks have positions of their own, keeps them in MTPState.
"""
from __future__ import annotations

import torch

from ..kernels.head_ops import lin_epi, rmsnorm
from ..kernels.paged_attention import paged_attention
from ..kernels.rope import rope_append
from ..kernels.router import gemm_bf16
from ..memory.kv_pages import KVPages

FEW_ROWS = 8


class AttentionLayer:
    """wqkv bf16 [(heads + 2 kv_heads) dim, H] (query, key and value rows in that order), wo bf16 [H, heads dim]; inv_freq fp64
    [rot / 2]; q_norm, k_norm bf16 [dim] or None; axis, adjacent and factor as rope_append takes them; window, sinks and scale
    as paged_attention does."""

    def __init__(self, wqkv: torch.Tensor, wo: torch.Tensor, heads: int, kv_heads: int, dim: int, inv_freq: torch.Tensor,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                 axis: torch.Tensor | None = None, adjacent: bool = False, factor: float = 1.0, window: int = 0,
                 sinks: int = 0, scale: float | None = None):
        if wqkv.dim() != 2 or wqkv.shape[0] != (heads + 2 * kv_heads) * dim:
            raise ValueError(f"wqkv must be [{(heads + 2 * kv_heads) * dim}, H], got {tuple(wqkv.shape)}")
        H = wqkv.shape[1]
        if tuple(wo.shape) != (H, heads * dim):
            raise ValueError(f"wo must be [{H}, {heads * dim}], got {tuple(wo.shape)}")
        if H % 256 or heads * dim % 256:
            raise ValueError("the hidden size and heads * dim must be multiples of 256")
        if (q_norm is None) != (k_norm is None):
            raise ValueError("q_norm and k_norm come together")
        for name, t, shape in (("wqkv", wqkv, wqkv.shape), ("wo", wo, wo.shape), ("q_norm", q_norm, (dim,)),
                               ("k_norm", k_norm, (dim,))):
            if t is not None and (t.dtype != torch.bfloat16 or tuple(t.shape) != tuple(shape) or not t.is_contiguous()):
                raise ValueError(f"{name} must be contiguous bf16 {tuple(shape)}")
        self.hidden, self.heads, self.kv_heads, self.dim = H, heads, kv_heads, dim
        self.wqkv, self.wo, self.inv_freq, self.axis, self.eps = wqkv, wo, inv_freq, axis, float(eps)
        self.adjacent, self.factor, self.window, self.sinks, self.scale = adjacent, factor, window, sinks, scale
        # The norms act on query and key heads only: those rows are then a projection of their own.
        self.n_qk = (heads + kv_heads) * dim
        self.qk_norm = None if q_norm is None else torch.cat([q_norm.repeat(heads), k_norm.repeat(kv_heads)]).contiguous()

    def _lin(self, x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        return lin_epi(x, w, out=out) if x.shape[0] <= FEW_ROWS else gemm_bf16(x, w, out=out)

    def append(self, x: torch.Tensor, positions, k_pages, v_pages, cu_rows, kv_len, table, max_rows: int,
               scales: torch.Tensor | None = None) -> torch.Tensor:
        """Projects x bf16 [R, H], writes its key and value rows into the cache, returns the turned queries [R, heads, dim]."""
        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != self.hidden or not x.is_contiguous():
            raise ValueError(f"x must be a contiguous bf16 [R, {self.hidden}] tensor")
        R, h, kv, d = x.shape[0], self.heads, self.kv_heads, self.dim
        if self.qk_norm is None:
            qkv = self._lin(x, self.wqkv).view(R, h + 2 * kv, d)
            q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        else:
            qk = rmsnorm(self._lin(x, self.wqkv[:self.n_qk]), self.qk_norm, self.eps, group=d).view(R, h + kv, d)
            q, k, v = qk[:, :h], qk[:, h:], self._lin(x, self.wqkv[self.n_qk:]).view(R, kv, d)
        return rope_append(q, k, v, positions, self.inv_freq, k_pages, v_pages, cu_rows, kv_len, table, max_rows,
                           axis=self.axis, adjacent=self.adjacent, factor=self.factor, scales=scales)

    def __call__(self, x: torch.Tensor, positions, k_pages, v_pages, cu_rows, kv_len, table, max_rows: int,
                 out: torch.Tensor | None = None, scales: torch.Tensor | None = None,
                 tree: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [R, H] (normalised rows of the batch) -> bf16 [R, H]; the batch, the scales of e4m3 pages and the words of a tree's
        rows as rope_append and paged_attention take them."""
        q = self.append(x, positions, k_pages, v_pages, cu_rows, kv_len, table, max_rows, scales)
        o = paged_attention(q, k_pages, v_pages, cu_rows, kv_len, table, max_rows, window=self.window, sinks=self.sinks,
                            scale=self.scale, scales=scales, tree=tree)
        return self._lin(o.view(x.shape[0], self.heads * self.dim), self.wo, out)


class SeqCache:
    """One sequence of `pages`, with text positions (a row's position is its token's place). Beside the pages it holds 12 bytes for each
    token that the table covers."""

    def __init__(self, pages: KVPages):
        self.pages, self.pos, self.last = pages, 0, None
        dev, most = pages.k.device, pages.width * pages.page
        self.kv_len = torch.zeros(1, dtype=torch.int32, device=dev)
        self._cu = torch.zeros((most + 1, 2), dtype=torch.int32, device=dev)   # cu_rows of n rows: [0, n]
        self._cu[:, 1] = torch.arange(most + 1, dtype=torch.int32, device=dev)
        self._positions = torch.zeros(most, dtype=torch.int32, device=dev)
        self.seq = pages.new()
        self.table = pages.table[self.seq:self.seq + 1]

    def rows(self, n: int):
        """(cu_rows, kv_len, table, positions) of `n` rows: tensors that stay in place; place() sets the contents of kv_len and
        positions, which are those of the call that it named last."""
        if not 0 <= n < self._cu.shape[0]:
            raise ValueError(f"{n} rows exceed the table's {self._cu.shape[0] - 1}")
        return self._cu[n], self.kv_len, self.table, self._positions[:n]

    def room(self, pos: int, n: int) -> None:
        """Pages that the tokens pos .. pos + n - 1 may be written to: what the sequence held from `pos` on (rows taken back, drafts) is
        given up, and a page that a fork holds too is copied first. Nothing changes where it is refused."""
        at = min(pos, self.pages.length[self.seq])
        self.pages.rewrite(self.seq, at, pos + n - at)

    def place(self, pos: int, n: int) -> None:
        """The next call's rows are the tokens pos .. pos + n - 1: their pages are there, the tensors of rows(n) say so."""
        self.room(pos, n)
        self.point(pos, n)

    def point(self, pos: int, n: int) -> None:
        """place() where room() has been called for these tokens, others behind them among them."""
        self.kv_len.fill_(pos + n)
        torch.add(self._cu[:n, 1], pos, out=self._positions[:n])

    def reset(self) -> None:
        self.pos, self.last = 0, None
        self.pages.truncate(self.seq, 0)

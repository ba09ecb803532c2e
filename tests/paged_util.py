"""A small paged cache with its batch, and the operators on it in 64 bits (not collected: no test_ prefix)."""
import math

import numpy as np
import torch


class Batch:
    """`rows[s]` new rows and `lens[s]` cached tokens of each sequence (the new rows last), pages dealt at random from a
    cache with `spare` more; what the cache holds past a sequence's tokens is `tail` (default: large values)."""

    def __init__(self, rows, lens, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=0, spare=2, tail=3e4, width=None):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.heads, self.kv_heads, self.dim, self.page, self.dtype = (
            list(rows), list(lens), heads, kv_heads, dim, page, dtype)
        need = [-(-n // page) for n in self.lens]
        w = max(need + [1]) if width is None else width
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g)
        self.table = torch.full((len(self.rows), w), -1, dtype=torch.int32)
        self.k = torch.full((n_pages, kv_heads, page, dim), tail).to(dtype)
        self.v = torch.full((n_pages, kv_heads, dim, page), tail).to(dtype)
        at = 0
        for s, n in enumerate(need):
            mine = ids[at:at + n]
            at += n
            self.table[s, :n] = mine.to(torch.int32)
            for j, p in enumerate(mine.tolist()):
                t = min(page, self.lens[s] - j * page)
                self.k[p, :, :t] = torch.randn(kv_heads, t, dim, generator=g).to(dtype)
                self.v[p, :, :, :t] = torch.randn(kv_heads, dim, t, generator=g).to(dtype)
        self.total = sum(self.rows)
        self.q = (torch.randn(self.total, heads, dim, generator=g) * 1.5).to(dtype)
        self.cu = torch.tensor([0] + list(np.cumsum(self.rows)), dtype=torch.int32)
        self.kv_len = torch.tensor(self.lens, dtype=torch.int32)
        self.max_rows = max(self.rows + [1])

    def args(self, device="cuda"):
        """(q, k_pages, v_pages, cu_rows, kv_len, table, max_rows) on the device."""
        return [t.to(device) for t in (self.q, self.k, self.v, self.cu, self.kv_len, self.table)] + [self.max_rows]


def attention64(b: Batch, window=0, sinks=0, scale=None, absolute=False):
    """(out, lse) of every row in 64 bits; `absolute`: sum_j p_j |v_j| in the place of out. A token in a page that the table
    does not hold is not there."""
    scale = 1.0 / math.sqrt(b.dim) if scale is None else scale
    group = b.heads // b.kv_heads
    out = torch.zeros(b.total, b.heads, b.dim, dtype=torch.float64)
    lse = torch.full((b.total, b.heads), -math.inf, dtype=torch.float64)
    r = 0
    for s, n in enumerate(b.rows):
        held = [j for j in range(b.lens[s]) if 0 <= int(b.table[s, j // b.page]) < b.k.shape[0]]
        ids = b.table[s].long()[[j // b.page for j in held]]
        off = torch.tensor([j % b.page for j in held], dtype=torch.long)
        k, v = b.k[ids, :, off].double(), b.v[ids, :, :, off].double()   # [tokens, kv_heads, dim]
        at = torch.tensor(held, dtype=torch.long)
        for i in range(n):
            p = b.lens[s] - n + i
            see = at <= p
            if window:
                see &= (p - at < window) | (at < sinks)
            if see.any():
                x = torch.einsum("hd,thd->ht", b.q[r].double(), k[see].repeat_interleave(group, 1)) * scale
                lse[r] = torch.logsumexp(x, 1)
                vv = v[see].repeat_interleave(group, 1)
                out[r] = torch.einsum("ht,thd->hd", torch.softmax(x, 1), vv.abs() if absolute else vv)
            r += 1
    return out, lse


def half_step(dtype) -> float:
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def attention_bound(b: Batch, **mask):
    """How far an output may be from attention64's: the result is rounded once (u |out|) and every probability once before
    its product (u sum p |v|); fp32 scores of `dim` terms at values of a few units, the exponential and the sums add
    less than 2^-16 relative to sum p |v|."""
    u = half_step(b.dtype)
    out, _ = attention64(b, **mask)
    mass, _ = attention64(b, absolute=True, **mask)
    return u * out.abs() + (u + 2.0 ** -16) * mass + 1e-7


def rope64(x, positions, inv_freq, axis=None, adjacent=False, factor=1.0):
    """x [rows, heads, dim] turned in 64 bits by positions [axes, rows]."""
    x = x.double().clone()
    half = inv_freq.numel()
    for i in range(half):
        a = positions[int(axis[i]) if axis is not None else 0].double() * inv_freq[i].double()
        i0, i1 = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        c, s = (a.cos() * factor)[:, None], (a.sin() * factor)[:, None]
        p, q = x[:, :, i0].clone(), x[:, :, i1].clone()
        x[:, :, i0], x[:, :, i1] = p * c - q * s, q * c + p * s
    return x

"""Paged caches in 8 bits and trees of drafts in 64 bits, for the tests of their operators (not collected: no test_ prefix)."""
import math

import torch

from tests.paged_util import Batch, half_step

E4M3 = torch.float8_e4m3fn


def quantise64(x):
    """(codes e4m3, bytes uint8) of the vectors x [..., dim] in 64 bits: the least exponent e >= -126 with max |x| <= 448 2^e, codes
    of x 2^-e; what is not finite is left out of the maximum and NaN."""
    fine = torch.isfinite(x)
    m, e = torch.frexp(torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1) / 448.0)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(-126, 127)
    y = torch.where(fine, torch.ldexp(x, -e[..., None]), torch.full_like(x, math.nan))
    return y.float().to(E4M3), (e + 127).to(torch.uint8)


def values64(codes, scales, keys):
    """What pages of codes stand for: keys [.., page, dim] by scales[.., 0, :], values [.., dim, page] by scales[.., 1, :]."""
    e = torch.exp2(scales.double() - 127)
    return codes.double() * (e[..., 0, :, None] if keys else e[..., 1, None, :])


class Batch8(Batch):
    """A Batch whose pages are e4m3 numbers: k8, v8, scales; k and v are what they stand for, in 64 bits. Where a sequence holds
    nothing the pages have `tail` (a code) and the exponent byte `tail_exp`."""

    def __init__(self, rows, lens, heads, kv_heads, dim, page, seed=0, tail=0x7E, tail_exp=127, spread=6, **kw):
        super().__init__(rows, lens, heads, kv_heads, dim, page, torch.bfloat16, seed=seed, tail=math.inf, **kw)
        n = self.k.shape[0]
        g = torch.Generator().manual_seed(seed + 1)
        # every token's own power of two
        kf = self.k.double() * torch.exp2(torch.randint(-1, 2, (n, kv_heads, page, 1), generator=g).double())
        vf = self.v.double() * torch.exp2(torch.randint(-spread, spread + 1, (n, kv_heads, 1, page), generator=g).double())
        none = torch.isinf(self.k[:, 0, :, 0])                       # [n, page]
        kc, ke = quantise64(kf)
        vc, ve = quantise64(vf.transpose(2, 3))
        self.k8, self.v8 = kc, vc.transpose(2, 3).contiguous()
        self.scales = torch.stack([ke, ve], 2).contiguous()
        held = none[:, None, :, None].expand(n, kv_heads, page, dim)
        self.k8.view(torch.uint8)[held] = tail
        self.v8.view(torch.uint8)[held.transpose(2, 3)] = tail
        self.scales[none[:, None, None, :].expand(n, kv_heads, 2, page)] = tail_exp
        self.widen()

    def widen(self):
        self.k, self.v = values64(self.k8, self.scales, True), values64(self.v8, self.scales, False)

    def args(self, device="cuda"):
        return [t.to(device) for t in (self.q, self.k8, self.v8, self.cu, self.kv_len, self.table)] + [self.max_rows]


def random_parents(n, seed):
    """A tree of n rows in which every row's parent is an earlier one."""
    g = torch.Generator().manual_seed(seed)
    return [-1] + [int(torch.randint(max(0, i - 1 - i // 2), i, (1,), generator=g)) for i in range(1, n)]


def masks_of(parents):
    """Words (Python ints) of one sequence's rows."""
    out = []
    for i, p in enumerate(parents):
        out.append((1 << i) | (out[p] if 0 <= p < i else 0))
    return out


def as_int64(words):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64)


def tree64(b, words, window=0, sinks=0, scale=None, absolute=False):
    """(out, lse) in 64 bits of rows that see the tokens before their sequence's rows and the rows of their words."""
    scale = 1.0 / math.sqrt(b.dim) if scale is None else scale
    group = b.heads // b.kv_heads
    out = torch.zeros(b.total, b.heads, b.dim, dtype=torch.float64)
    lse = torch.full((b.total, b.heads), -math.inf, dtype=torch.float64)
    r = 0
    for s, n in enumerate(b.rows):
        base = b.lens[s] - n
        held = [j for j in range(b.lens[s]) if 0 <= int(b.table[s, j // b.page]) < b.k.shape[0]]
        at = torch.tensor(held, dtype=torch.long)
        ids, off = b.table[s].long()[at // b.page], at % b.page
        k, v = b.k[ids, :, off].double(), b.v[ids, :, :, off].double()
        for i in range(n):
            word = words[r] & ((1 << n) - 1)
            p = base + max(bin(word).count("1"), 1) - 1
            see = torch.tensor([(t < base and (not window or p - t < window or t < sinks))
                                or (t >= base and (word >> (t - base)) & 1 == 1) for t in held], dtype=torch.bool)
            if see.any():
                x = torch.einsum("hd,thd->ht", b.q[r].double(), k[see].repeat_interleave(group, 1)) * scale
                lse[r] = torch.logsumexp(x, 1)
                vv = v[see].repeat_interleave(group, 1)
                out[r] = torch.einsum("ht,thd->hd", torch.softmax(x, 1), vv.abs() if absolute else vv)
            r += 1
    return out, lse


def tree_bound(b, words, **mask):
    """As paged_util.attention_bound: one rounding of the result, one of every probability (with e4m3 pages after its token's power
    of two, which changes no relative error), fp32 scores, exponentials and sums."""
    u = half_step(b.dtype)
    out, _ = tree64(b, words, **mask)
    mass, _ = tree64(b, words, absolute=True, **mask)
    return u * out.abs() + (u + 2.0 ** -16) * mass + 1e-7


def accept64(target, tokens, parents, cu, max_rows):
    """accept_tree's result by the loop that it stands for."""
    out = torch.full((len(cu) - 1, 4 + 2 * max_rows), -1, dtype=torch.int32)
    for s, (lo, hi) in enumerate(zip(cu, cu[1:])):
        row, path, toks, flags = 0, [], [], 0
        while lo < hi:
            path.append(row)
            x = target[lo + row]
            if not torch.isfinite(x).all():
                flags = 1
                break
            t = int(torch.nonzero(x == x.max())[0])
            toks.append(t)
            nxt = [i for i in range(1, hi - lo) if parents[lo + i] == row and 0 <= parents[lo + i] < i and tokens[lo + i] == t]
            if not nxt:
                break
            row = nxt[0]
        out[s, :4] = torch.tensor([max(len(path) - 1, 0), len(toks), 0, flags])
        out[s, 4:4 + len(toks)] = torch.tensor(toks, dtype=torch.int32)
        out[s, 4 + max_rows:4 + max_rows + len(path)] = torch.tensor(path, dtype=torch.int32)
    return out

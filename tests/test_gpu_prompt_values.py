"""The many-row attention where its tiles are handled apart, for every page size's kernel: non-finite values at places that some rows
see and others do not, scores that raise the running maximum, batches of prompts beside single tokens, tables far wider than the
sequences. Against 64 bits with the bounds of tests/paged_util.py."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from tests.paged_util import Batch, attention64, attention_bound
from tests.test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.int16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_unseen_places(page, dim, bad, dtype):
    """Past the tokens, before the window, in pages not held, at later rows' tokens, with and without the split over the length."""
    for n in (150, 2500):
        b = Batch([40, 12], [n, 205], 4, 2, dim, page, dtype, tail=bad, seed=3)
        b.table[1, 1:128 // page] = -1                        # tokens page .. 127 are not held: the windows begin at 134 and later
        check(b, window=60, sinks=16)
        b = Batch([40], [n], 4, 2, dim, page, dtype, seed=4)
        want = check(b)
        at = n - 10                                           # the token of row 30: seen by it and the rows behind it
        p, off = int(b.table[0, at // page]), at % page
        k = b.k.clone()
        b.k[p, :, off] = bad
        got = paged_attention(*b.args())
        assert torch.equal(bits(got[:30]), bits(want[:30])) and torch.isnan(got[30:]).all()
        b.k = k
        b.v[p, 1, 7, off] = bad
        got = paged_attention(*b.args())
        keep = torch.ones(4, dim, dtype=torch.bool, device="cuda")
        keep[2:, 7] = False
        assert torch.equal(bits(got[:30]), bits(want[:30])) and torch.equal(bits(got[30:][:, keep]), bits(want[30:][:, keep]))
        seen = got[30:, 2:, 7].float()
        assert torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_first_tokens_under_a_window(page, dim):
    """The first tokens' tile is seen in part by every row: an infinity there reaches all rows, one behind the first tokens those
    alone whose window holds it."""
    b = Batch([70], [300], 4, 2, dim, page, seed=5)
    want = check(b, window=90, sinks=6)
    for token, rows in ((3, slice(0, 70)), (6, slice(0, 0)), (200, slice(0, 60))):   # row i is token 230 + i
        v = b.v.clone()
        b.v[int(b.table[0, token // page]), :, 9, token % page] = math.inf
        got = paged_attention(*b.args(), window=90, sinks=6)
        b.v = v
        keep = [d for d in range(dim) if d != 9]
        assert torch.equal(bits(got[..., keep]), bits(want[..., keep]))
        hit = torch.zeros(70, dtype=torch.bool)
        hit[rows] = True
        assert (got[hit][:, :, 9] == math.inf).all() and torch.equal(bits(got[~hit]), bits(want[~hit]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_large_scores(page, dim, dtype):
    """Scores of some hundreds: the running maximum is raised by far more than 2^8 in tiles behind the first, for many rows."""
    b = Batch([40, 150], [600, 150], 4, 2, dim, page, dtype, seed=10)
    b.q *= 20
    lse = torch.empty(b.total, b.heads, device="cuda")
    got = paged_attention(*b.args(), lse=lse).double().cpu()
    want, want_lse = attention64(b)
    # The largest sum of |q k| of any row and token, from which an fp32 score of `dim` products in any order is off by at most
    # dim 2^-24 of it, and by 2^-22 more for its scale and the subtraction of the maximum: `off`. A probability then is off
    # by 2 off relative, as its sum is too.
    top, raised, r = 0.0, 0, 0
    for s, n in enumerate(b.rows):
        t = torch.arange(b.lens[s])
        k = b.k[b.table[s].long()[t // page], :, t % page].double().repeat_interleave(2, 1)
        for i in range(n):
            x = torch.einsum("hd,thd->ht", b.q[r].double(), k) / math.sqrt(dim)
            a = torch.einsum("hd,thd->ht", b.q[r].double().abs(), k.abs()) / math.sqrt(dim)
            p = b.lens[s] - n + i + 1
            top = max(top, float(a[:, :p].max()))
            raised += int((x[:, :p].amax(1) > x[:, :min(p, 64)].amax(1) + 10 * math.log(2)).sum())
            r += 1
    assert raised > 100                                       # of 760 rows and heads: the case is there, 194 at the fewest
    off = top * (dim * 2.0 ** -24 + 2.0 ** -22)
    assert ((got - want).abs() <= attention_bound(b) + 2.5 * off * attention64(b, absolute=True)[0]).all()
    assert ((lse.double().cpu() - want_lse).abs() <= off + 1e-5 * (1 + want_lse.abs())).all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(8, 2, 128, 64, torch.bfloat16), (4, 4, 64, 16, torch.float16),
                                                          (6, 1, 256, 32, torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_prompts_beside_single_tokens(heads, kv_heads, dim, page, dtype, window, sinks):
    """One prompt chunk, single tokens over long contexts, a verify round and a sequence without rows in one call."""
    check(Batch([200, 1, 1, 3, 0, 1], [260, 5000, 3001, 2000, 50, 1], heads, kv_heads, dim, page, dtype, seed=dim), window, sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_table_far_wider_than_its_sequences(dim):
    """Tables of 131,072 tokens, as a KVPages of the default size has them: prompts from nothing and behind a context."""
    check(Batch([100, 33, 1], [100, 3333, 700], 4, 2, dim, 64, seed=dim, width=2048))
    check(Batch([1, 3], [777, 1500], 4, 2, dim, 64, seed=dim, width=2048))

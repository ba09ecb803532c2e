"""Prompts over e4m3 pages and trees in the many-row form, against their definitions in 64 bits. Short tables and few packed rows take the few-row
form (they are in test_gpu_e4m3_cache.py and test_gpu_tree.py), so here the tables are wide and every call has 72 packed rows or more."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from tests import test_gpu_e4m3_cache as causal, test_gpu_tree as tree
from tests.test_gpu_tree import ERR_PAGE, KINDS, as_int64, masks_of, trees
from tests.tree_util import Batch8

pytestmark = pytest.mark.gpu


def make(kind, rows, lens, dim, page, heads=8, kv_heads=1, **kw):
    return tree.make(kind, rows, lens, heads, kv_heads, dim, page, width=4160 // page + 1, **kw)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (18, 2)])
def test_prompts_by_pages(page, dim, heads, kv_heads):
    causal.check(make("e4m3", [9, 1, 20, 70, 0, 33], [9, 40, 333, 700, 12, 65], dim, page, heads, kv_heads, seed=page + dim))


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_of_more_pages_than_a_register_holds(page, dim):
    """The table's entries are read 64 at a time."""
    causal.check(make("e4m3", [40, 1], [2600, 1090], dim, page, seed=dim))


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (33, 0), (64, 17), (100, 200), (1500, 3)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 32), (128, 64), (256, 16)])
def test_prompts_by_windows(window, sinks, dim, page):
    causal.check(make("e4m3", [30, 1, 12], [30, 129, 2400], dim, page, seed=window), window, sinks)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 32), (128, 64), (256, 16), (256, 32)])
@pytest.mark.parametrize("tail,tail_exp", [(0x7F, 127), (0xFF, 254), (0x7E, 255), (0x7F, 255), (0xFE, 0)])
def test_unseen_places_do_not_matter(dim, page, tail, tail_exp):
    b = make("e4m3", [20, 1], [90, 405], dim, page, tail=tail, tail_exp=tail_exp, seed=3)
    causal.check(b)
    b.table[1, 1:320 // page] = -1
    causal.check(b, window=60, sinks=16)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 32), (128, 64), (256, 16)])
def test_a_token_of_nan(dim, page):
    b = make("e4m3", [20], [90], dim, page, seed=4)
    want = causal.check(b)
    p, off = int(b.table[0, 89 // page]), 89 % page
    b.v8.view(torch.uint8)[p, :, 5, off] = 0xFF
    got = paged_attention(*b.args(), scales=b.scales.cuda())
    assert torch.equal(got[:-1].view(torch.int16), want[:-1].view(torch.int16))
    assert torch.isnan(got[-1, :, 5]).all()
    keep = [d for d in range(dim) if d != 5]
    assert torch.equal(got[-1][:, keep], want[-1][:, keep])
    b.k8.view(torch.uint8)[p, :, off] = 0x7F
    b.scales[p, :, :, off] = 255
    got = paged_attention(*b.args(), scales=b.scales.cuda())
    assert torch.equal(got[:-1].view(torch.int16), want[:-1].view(torch.int16))
    assert torch.isnan(got[-1]).all()


@pytest.mark.parametrize("page", [16, 32])
def test_missing_pages_of_prompts(page):
    b = make("e4m3", [20, 12], [700, 1300], 128, page, seed=3)
    for bad in (-1, 10 ** 6):
        b.table[0, 128 // page] = bad
        b.table[1, 1152 // page] = bad
        paged_attention(*b.args(), scales=b.scales.cuda())
        torch.cuda.synchronize()
        assert _lib.device_error() == ERR_PAGE
        held = Batch8.__new__(Batch8)
        held.__dict__.update(b.__dict__)
        held.table = torch.where(b.table < b.k8.shape[0], b.table, torch.full_like(b.table, -1))
        want, _ = causal.attention64(held)
        out = paged_attention(*b.args(), scales=b.scales.cuda())
        assert _lib.device_error() == ERR_PAGE
        assert ((out.double().cpu() - want).abs() <= causal.attention_bound(held)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_trees_by_pages(kind, page, dim):
    b = make(kind, [12, 1, 64, 30, 0, 64], [12, 70, 64, 333, 5, 1200], dim, page, seed=page)
    tree.check(b, trees(b))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [9, 50])
def test_any_words(kind, rows):
    b = make(kind, [rows, rows], [rows, 200], 128, 16, seed=8)
    g = torch.Generator().manual_seed(5)
    words = [int(torch.randint(0, 1 << 32, (1,), generator=g)) << 32 | int(torch.randint(0, 1 << 32, (1,), generator=g))
             for _ in range(2 * rows)]
    words[0], words[1], words[2], words[rows] = 0, (1 << 64) - 1, 1 << 63, 0
    tree.check(b, words)
    tree.check(b, words, window=77, sinks=9)


@pytest.mark.parametrize("kind", KINDS)
def test_windows_of_trees_that_begin_at_the_edges_of_tiles(kind):
    rows, window = 20, 70
    lens = [rows + window + d for d in (30, 31, 32, 33, 62, 63, 64, 65, 66, 127, 128, 129)]
    b = make(kind, [rows] * len(lens), lens, 64, 16, seed=rows)
    words = trees(b)
    for s in range(len(lens)):
        words[s * rows + 2] = 0
        b.table[s, :(lens[s] - rows - window + 1) // 16] = -1
    tree.check(b, words, window=window)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
def test_what_other_branches_hold_does_not_matter(kind, page):
    rows = 30
    b = make(kind, [rows], [rows + 50], 128, page, seed=2)
    words = masks_of([-1, 0, 0] + [1 + i % 2 if i < 3 else i - 2 for i in range(1, rows - 2)])
    want = tree.check(b, words)
    bad = 2
    p, off = int(b.table[0, 52 // page]), 52 % page
    if kind == "e4m3":
        b.k8.view(torch.uint8)[p, :, off] = 0x7F
        b.v8.view(torch.uint8)[p, :, :, off] = 0xFF
        b.scales[p, :, :, off] = 255
    else:
        b.k[p, :, off] = math.inf
        b.v[p, :, :, off] = math.nan
    got = paged_attention(*b.args(), scales=b.scales.cuda() if kind == "e4m3" else None, tree=as_int64(words).cuda())
    for i, w in enumerate(words):
        if w >> bad & 1:
            assert torch.isnan(got[i]).all()
        else:
            assert torch.equal(got[i].view(torch.int16), want[i].view(torch.int16))


@pytest.mark.parametrize("page", [16, 64])
def test_missing_pages_of_trees(page):
    b = make("bf16", [20], [700], 64, page, seed=3)
    for bad in (-1, 10 ** 6):
        b.table[0, 256 // page] = bad
        tree.check(b, trees(b), error=ERR_PAGE)


@pytest.mark.parametrize("page", [16, 64])
def test_a_captured_call_follows_lengths_and_tables(page):
    b = make("e4m3", [40, 12], [1500, 300], 128, page, seed=6)
    q, k, v, cu, kv_len, table, rows = b.args()
    sc, out = b.scales.cuda(), torch.zeros_like(b.q.cuda())
    paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc, out=out)
    for n0, n1 in ((1500, 300), (1100, 17), (40, 12), (1499, 260)):
        kv_len.copy_(torch.tensor([n0, n1]))
        table[0, :4] = table[0, :4].flip(0)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc))
        torch.cuda.synchronize()

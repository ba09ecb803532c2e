"""Trees of drafts over a paged cache against their definitions (tests/tree_util.py): masks, the attention of their rows over pages of 16
bits and of e4m3, the greedy round and the move of the accepted branch. Bounds count the roundings."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.kernels.tree import accept_tree, keep_rows, tree_masks
from tests.paged_util import Batch, attention64, attention_bound
from tests.tree_util import Batch8, accept64, as_int64, masks_of, random_parents, tree64, tree_bound

pytestmark = pytest.mark.gpu

ERR_PAGE, ERR_BATCH = 32, 64


def trees(b, seed=0):
    return [w for s, n in enumerate(b.rows) for w in masks_of(random_parents(n, seed + s) if n else [])]


def check(b, words, window=0, sinks=0, error=0):
    print(f"[tree] {type(b).__name__} rows={b.rows[:6]} lens={b.lens[:6]} heads={b.heads}/{b.kv_heads} dim={b.dim} page={b.page} "
          f"window={window}", flush=True)
    lse = torch.full((b.total, b.heads), 7.0, device="cuda")
    sc = b.scales.cuda() if isinstance(b, Batch8) else None
    out = paged_attention(*b.args(), window=window, sinks=sinks, lse=lse, scales=sc, tree=as_int64(words).cuda())
    torch.cuda.synchronize()
    assert _lib.device_error() == error
    want, want_lse = tree64(b, words, window, sinks)
    err = (out.double().cpu() - want).abs()
    bound = tree_bound(b, words, window=window, sinks=sinks)
    assert (err <= bound).all(), f"off by {(err / bound).max():.2f} of what the roundings allow"
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse.cpu()), empty)
    assert (out.cpu()[empty] == 0).all()
    assert ((lse.double().cpu() - want_lse).abs()[~empty] <= 1e-5 * (1 + want_lse.abs()[~empty])).all()
    return out


def make(kind, *args, **kw):
    if kind == "e4m3":
        return Batch8(*args, **kw)
    return Batch(*args, dtype={"bf16": torch.bfloat16, "fp16": torch.float16}[kind], **kw)


KINDS = ["bf16", "fp16", "e4m3"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (7, 1), (12, 4), (16, 1)])
def test_head_layouts(kind, dim, heads, kv_heads):
    for rows in ([1, 3, 8], [12, 2, 33]):
        b = make(kind, rows, [max(rows[0], 1), 70, 333], heads, kv_heads, dim, 32, seed=heads * dim)
        check(b, trees(b))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("rows", [5, 26, 64])
def test_pages_and_lengths(kind, page, rows):
    """The rows begin at every place of a tile: at the cache's first token, inside a page, across pages."""
    lens = [rows, rows + 1, rows + 7, rows + 8, rows + 31, rows + 60, rows + 64, rows + 130, rows + 511]
    b = make(kind, [rows] * len(lens), lens, 4, 2, 64, page, seed=page)
    check(b, trees(b))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(64, 0), (64, 5), (100, 200), (300, 16), (5000, 3)])
@pytest.mark.parametrize("rows", [6, 40])
def test_window_and_first_tokens(kind, window, sinks, rows):
    b = make(kind, [rows] * 4, [rows, rows + 60, 329, 700], 6, 2, 128, 16, seed=window + rows)
    check(b, trees(b), window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [7, 50])
def test_any_words(kind, rows):
    """Words that are no tree's: rows after their own, none, all, bits of rows that are not there."""
    b = make(kind, [rows, rows], [rows, 200], 4, 1, 128, 16, seed=8)
    g = torch.Generator().manual_seed(5)
    words = [int(torch.randint(0, 1 << 32, (1,), generator=g)) << 32 | int(torch.randint(0, 1 << 32, (1,), generator=g))
             for _ in range(2 * rows)]
    words[0], words[1], words[2], words[rows] = 0, (1 << 64) - 1, 1 << 63, 0      # row 0 of the first sees nothing at all
    check(b, words)
    check(b, words, window=77, sinks=9)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [4, 40])
def test_windows_that_begin_at_the_edges_of_tiles(kind, rows):
    """The first token in sight is the last of a tile of 32 or 64, the first of the next, or beside them; rows that see none of the tree
    among the others; pages before the window are not held, and nothing is raised for them."""
    window = 70
    lens = [rows + window + d for d in (30, 31, 32, 33, 62, 63, 64, 65, 66, 127, 128, 129)]
    b = make(kind, [rows] * len(lens), lens, 4, 2, 64, 16, seed=rows)
    words = trees(b)
    for s in range(len(lens)):
        words[s * rows + 2] = 0
        first = lens[s] - rows - window + 1                      # the first token that row 0 (and a row without bits) sees
        b.table[s, :first // 16] = -1
    check(b, words, window=window)


def test_a_chain_is_the_causal_rows():
    """In a chain every row sees what a causal row sees. Its values agree with the causal call's to the roundings of both."""
    for dim, rows in ((64, 5), (128, 20), (256, 8)):
        b = Batch([rows] * 2, [rows + 500, 64], 8, 2, dim, 32, seed=dim)
        words = [(2 << i) - 1 for i in range(rows)] * 2
        out = check(b, words)
        causal = paged_attention(*b.args())
        assert ((out.double() - causal.double()).abs().cpu() <= 2 * tree_bound(b, words)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_long_cache_in_many_chunks(kind):
    b = make(kind, [8, 26, 64], [9001, 5000, 2000], 8, 2, 128, 64, seed=5, width=400)
    check(b, trees(b))
    check(b, trees(b), window=3000, sinks=70)
    b = make(kind, [8, 3], [9001, 5000], 8, 2, 128, 64, seed=6, width=400)
    check(b, trees(b))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("seqs", [3, 64, 65, 130])
def test_many_sequences_share_the_chunks(kind, seqs):
    """Rows and lengths of every size, none among them: the chunks are shared by all sequences' own."""
    g = torch.Generator().manual_seed(seqs)
    rows = [int(torch.randint(0, 21, (1,), generator=g)) for _ in range(seqs)]
    rows[1] = 20
    lens = [int(torch.randint(0, 700, (1,), generator=g)) if i % 5 else i % 40 for i in range(seqs)]
    b = make(kind, rows, lens, 2, 1, 64, 16, seed=seqs)
    check(b, trees(b))
    if kind == "e4m3":                                            # and those of causal rows
        out = paged_attention(*b.args(), scales=b.scales.cuda())
        want, _ = attention64(b)
        assert ((out.double().cpu() - want).abs() <= attention_bound(b)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_shared_chunks_in_a_graph_follow_the_lengths(kind):
    b = make(kind, [30, 12, 9], [2000, 900, 640], 8, 1, 64, 16, seed=12)
    q, k, v, cu, kv_len, table, most = b.args()
    sc = b.scales.cuda() if kind == "e4m3" else None
    tree, out = as_int64(trees(b)).cuda(), torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, cu, kv_len, table, most, scales=sc, tree=tree, out=out)
    for lens in ([2000, 900, 640], [30, 900, 9], [0, 0, 0], [2000, 12, 640]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, k, v, cu, kv_len, table, most, scales=sc, tree=tree))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [6, 30])
def test_what_other_branches_hold_does_not_matter(kind, rows):
    """Rows beside a row's branch hold infinities and NaN; the rows that see them get them."""
    b = make(kind, [rows], [rows + 50], 4, 2, 128, 16, seed=2)
    parents = [-1, 0, 0] + [1 + i % 2 if i < 3 else i - 2 for i in range(1, rows - 2)]
    words = masks_of(parents)
    want = check(b, words)
    bad = 2                                                     # the second child's branch
    t = 50 + bad
    page, off = int(b.table[0, t // 16]), t % 16
    if kind == "e4m3":
        b.k8.view(torch.uint8)[page, :, off] = 0x7F
        b.v8.view(torch.uint8)[page, :, :, off] = 0xFF
        b.scales[page, :, :, off] = 255
    else:
        b.k[page, :, off] = math.inf
        b.v[page, :, :, off] = math.nan
    sc = b.scales.cuda() if kind == "e4m3" else None
    got = paged_attention(*b.args(), scales=sc, tree=as_int64(words).cuda())
    for i, w in enumerate(words):
        if w >> bad & 1:
            assert torch.isnan(got[i]).all()
        else:
            assert torch.equal(got[i].view(torch.int16), want[i].view(torch.int16))


def test_missing_pages_are_raised_and_skipped():
    for rows in (5, 20):
        b = Batch([rows], [200], 4, 2, 64, 16, seed=3)
        b.table[0, 4] = -1
        check(b, trees(b), error=ERR_PAGE)
        b.table[0, 4] = 10 ** 6
        check(b, trees(b), error=ERR_PAGE)


def test_padding_strides_streams_and_graphs():
    b = Batch([3, 30], [40, 300], 8, 2, 128, 32, seed=9)
    q, k, v, cu, kv_len, table, rows = b.args()
    words = trees(b)
    tree = torch.zeros(36, dtype=torch.int64, device="cuda")
    tree[:33] = as_int64(words).cuda()
    wide = torch.zeros(36, 12, 128, dtype=torch.bfloat16, device="cuda")
    wide[:33, 2:10] = q
    want = paged_attention(q, k, v, cu, kv_len, table, rows, tree=tree[:33].contiguous())
    out = torch.full((36, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        paged_attention(wide[:, 2:10], k, v, cu, kv_len, table, rows, tree=tree, out=out)
    st.synchronize()
    assert torch.equal(out[:33], want) and (out[33:] == 5).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(wide[:, 2:10], k, v, cu, kv_len, table, rows, tree=tree, out=out)
    for n in (300, 290, 40):
        kv_len[1] = n
        tree[5:20] = tree[5:20].flip(0)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:33], paged_attention(wide[:, 2:10], k, v, cu, kv_len, table, rows, tree=tree)[:33])


# ---------------------------------------------------------------- masks
@pytest.mark.parametrize("rows", [[1], [64], [3, 0, 17, 64, 1, 33]])
def test_masks_and_positions(rows):
    parents = [random_parents(n, 3 + n) for n in rows if n]
    flat = torch.tensor(sum(parents, []), dtype=torch.int32)
    cu = torch.tensor([0] + list(torch.tensor(rows).cumsum(0)), dtype=torch.int32)
    kv_len = torch.tensor([n + 10 * s for s, n in enumerate(rows)], dtype=torch.int32)
    masks, pos = tree_masks(flat.cuda(), cu.cuda(), kv_len.cuda(), 64)
    words = sum((masks_of(p) for p in parents), [])
    assert torch.equal(masks.cpu(), as_int64(words))
    base = sum(([10 * s] * n for s, n in enumerate(rows)), [])
    assert pos.cpu().tolist() == [t + bin(w).count("1") - 1 for t, w in zip(base, words)]
    assert _lib.device_error() == 0


def test_masks_of_bad_parents_and_padding():
    parents = torch.tensor([9, 0, 2, 7, 1, -1, 5], dtype=torch.int32, device="cuda")
    cu, kv_len = torch.tensor([0, 6], dtype=torch.int32, device="cuda"), torch.tensor([6], dtype=torch.int32, device="cuda")
    masks = torch.full((7,), 77, dtype=torch.int64, device="cuda")
    m, _ = tree_masks(parents, cu, kv_len, 6, masks=masks)
    assert m.cpu().tolist() == [1, 3, 4, 8, 19, 32, 77]
    assert _lib.device_error() == ERR_BATCH
    cu[1] = 7                                                     # more rows than max_rows
    tree_masks(parents, cu, kv_len, 6, masks=masks)
    assert _lib.device_error() == ERR_BATCH and masks[6] == 77


# ---------------------------------------------------------------- the greedy round
def round_of(rows, vocab, seed, follow=0.7):
    g = torch.Generator().manual_seed(seed)
    parents = [random_parents(n, seed + s) if n else [] for s, n in enumerate(rows)]
    total = sum(rows)
    cu = [0] + list(int(x) for x in torch.tensor(rows).cumsum(0))
    target = torch.randn(total, vocab, generator=g)
    tokens = torch.randint(0, vocab, (total,), generator=g)
    for s, p in enumerate(parents):
        for i in range(1, len(p)):
            if float(torch.rand(1, generator=g)) < follow:
                tokens[cu[s] + i] = target[cu[s] + p[i]].argmax()
    return target, tokens.to(torch.int32), torch.tensor(sum(parents, []), dtype=torch.int32), cu


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 255, 1001, 4099, 32003])
@pytest.mark.parametrize("rows", [[1], [64], [5, 0, 33, 64, 2]])
def test_accept(vocab, rows):
    target, tokens, parents, cu = round_of(rows, vocab, vocab)
    got = accept_tree(target.cuda(), tokens.cuda(), parents.cuda(), torch.tensor(cu, dtype=torch.int32).cuda(), 64)
    assert torch.equal(got.cpu(), accept64(target, tokens, parents, cu, 64))
    assert _lib.device_error() == 0


def test_accept_ties_and_non_finite_rows():
    rows, vocab = [40] * 6, 2003
    target, tokens, parents, cu = round_of(rows, vocab, 3, follow=0.0)
    target = (target * 2).round()                                 # many equal maxima
    target[0, 1500] = target[0].max()
    for s in range(6):
        for i in range(1, 40):
            tokens[cu[s] + i] = int(torch.nonzero(target[cu[s] + parents[cu[s] + i]] == target[cu[s] + parents[cu[s] + i]].max())[0])
    target[0] = -0.0
    target[0, 700:] = 0.0                                         # all equal: the first one
    want = accept64(target, tokens, parents, cu, 40)
    for s, bad in ((1, math.nan), (2, math.inf), (3, -math.inf)):
        d = int(want[s, 0]) // 2
        target[cu[s] + int(want[s, 4 + 40 + d]), 1999 + s] = bad
    target[cu[4]] = math.nan
    want = accept64(target, tokens, parents, cu, 40)
    assert want[:, 3].tolist() == [0, 1, 1, 1, 1, 0] and want[4, 1] == 0
    got = accept_tree(target.cuda(), tokens.cuda(), parents.cuda(), torch.tensor(cu, dtype=torch.int32).cuda(), 40)
    assert torch.equal(got.cpu(), want)


def test_accept_in_a_graph_and_another_stream():
    target, tokens, parents, cu = (x.cuda() if isinstance(x, torch.Tensor) else x for x in round_of([20, 9], 5001, 8))
    dcu = torch.tensor(cu, dtype=torch.int32).cuda()
    out = torch.zeros(2, 44, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        accept_tree(target, tokens, parents, dcu, 20, out=out)
    for seed in (8, 9, 10):
        t, k, p, _ = round_of([20, 9], 5001, seed)
        target.copy_(t)
        tokens.copy_(k)
        parents.copy_(p)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), accept64(t, k, p, cu, 20))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = accept_tree(target, tokens, parents, dcu, 20)
    st.synchronize()
    assert torch.equal(got, out)


# ---------------------------------------------------------------- the accepted branch in the cache
def check_keep(kind, rows, lens, kv_heads, dim, page, layers, seed=0, paths=None, error=0):
    print(f"[keep] {kind} rows={rows[:5]} lens={lens[:5]} {kv_heads}x{dim} page={page}", flush=True)
    b = make(kind, rows, lens, kv_heads, kv_heads, dim, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    n, most = b.k.shape[0], max(rows)
    bits = torch.uint8 if kind == "e4m3" else torch.int16
    k = torch.randint(0, 250, (layers, n, kv_heads, page, dim), generator=g).to(bits)
    v = torch.randint(0, 250, (layers, n, kv_heads, dim, page), generator=g).to(bits)
    sc = torch.randint(0, 250, (layers, n, kv_heads, 2, page), generator=g).to(torch.uint8) if kind == "e4m3" else None
    took = torch.full((len(rows), 4 + 2 * most), -1, dtype=torch.int32)
    for s, m in enumerate(rows):
        if paths is not None:
            path = paths[s]
        else:
            parents, i, path = random_parents(m, seed + s) if m else [], m - 1, []
            while i >= 0:
                path.insert(0, i)
                i = parents[i]
        took[s, 0] = max(len(path) - 1, 0)
        took[s, 4 + most:4 + most + len(path)] = torch.tensor(path, dtype=torch.int32)
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}[kind]
    dk, dv = k.cuda().view(dtype), v.cuda().view(dtype)
    ds = sc.cuda() if sc is not None else None
    keep_rows(dk, dv, b.cu.cuda(), b.kv_len.cuda(), b.table.cuda(), took.cuda(), scales=ds)
    torch.cuda.synchronize()
    assert _lib.device_error() == error
    k0, v0, s0 = k.clone(), v.clone(), sc.clone() if sc is not None else None
    for s, m in enumerate(rows):
        base, before = b.lens[s] - m, -1
        for d in range(int(took[s, 0]) + 1):
            p = int(took[s, 4 + most + d])
            if not before < p < m:
                break
            before = p
            x, y = base + p, base + d
            if x < 0 or y < 0:
                continue
            (xp, xo), (yp, yo) = ((int(b.table[s, t // page]), t % page) for t in (x, y))
            k[:, yp, :, yo] = k0[:, xp, :, xo]
            v[:, yp, :, :, yo] = v0[:, xp, :, :, xo]
            if sc is not None:
                sc[:, yp, :, :, yo] = s0[:, xp, :, :, xo]
    assert torch.equal(dk.view(bits).cpu(), k) and torch.equal(dv.view(bits).cpu(), v)
    assert sc is None or torch.equal(ds.cpu(), sc)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (3, 128), (2, 256)])
def test_keep(kind, page, kv_heads, dim):
    check_keep(kind, [1, 64, 5, 30, 12], [1, 64, 20, 300, 77], kv_heads, dim, page, 3, seed=page)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_keep_paths(kind):
    """Branches that overlap their own places, long ones, rows that stay, no rows, rows before the cache."""
    paths = [[0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19], [0, 1, 2, 3], [0], [], [1, 3], [0, 2]]
    check_keep(kind, [20, 5, 1, 0, 4, 6], [33, 40, 9, 12, 60, 4], 2, 64, 16, 2, paths=paths)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_keep_from_every_place(kind, page):
    """Long branches (every other row, all but one, the last ones) that begin at each of eight places beside each other."""
    paths = [list(range(0, 64, 2)), [0, 1, 2] + list(range(4, 64)), [0] + list(range(50, 64)), list(range(0, 40, 3))] * 2
    check_keep(kind, [64, 64, 64, 40] * 2, [64 + 250 + i for i in range(8)], 1, 64, page, 2, paths=paths)


def test_keep_follows_a_bad_path_up_to_its_fault():
    check_keep("bf16", [6, 6, 6], [20, 20, 20], 1, 64, 16, 1, paths=[[0, 2, 2, 4], [0, 3, 9], [0, 4, 1]], error=ERR_BATCH)


def test_keep_in_a_graph():
    b = Batch([6], [30], 2, 2, 64, 16)
    k = torch.randn(2, b.k.shape[0], 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.randn(2, b.k.shape[0], 2, 64, 16, dtype=torch.bfloat16, device="cuda")
    took = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
    cu, kv_len, table = b.cu.cuda(), b.kv_len.cuda(), b.table.cuda()
    took[0, 0] = 0
    took[0, 10] = 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep_rows(k, v, cu, kv_len, table, took)
    for path, n in (([0, 2, 5], 30), ([0, 1, 4, 5], 29), ([0, 3], 17)):
        kv_len[0] = n
        took[0, 0] = len(path) - 1
        took[0, 10:] = -1
        took[0, 10:10 + len(path)] = torch.tensor(path, dtype=torch.int32)
        k1, v1 = k.clone(), v.clone()
        keep_rows(k1, v1, cu, kv_len, table, took)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, k1) and torch.equal(v, v1)


# ---------------------------------------------------------------- a round
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_round_equals_its_branch_written_plainly(kind):
    """Rows of a tree written, attended, accepted and moved: the cache then holds what the accepted branch's rows written one after the
    other leave, bit for bit, and the rows' attention is that of the branch to the roundings."""
    from slotstream_spark_amd.kernels.rope import rope_append
    n, base, heads, kv, dim, page, vocab = 20, 45, 8, 2, 128, 16, 997
    b = make(kind, [n], [base + n], heads, kv, dim, page, seed=21)
    pages = (b.k8, b.v8) if kind == "e4m3" else (b.k, b.v)
    k, v = (t.cuda()[None].contiguous() for t in pages)
    sc = b.scales.cuda()[None].contiguous() if kind == "e4m3" else None
    one = lambda t: None if t is None else t[0]
    parents = torch.tensor(random_parents(n, 4), dtype=torch.int32, device="cuda")
    cu, kv_len, table = b.cu.cuda(), b.kv_len.cuda(), b.table.cuda()
    g = torch.Generator().manual_seed(22)
    qkv = torch.randn(n, heads + 2 * kv, dim, generator=g).to(torch.bfloat16).cuda()
    inv = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).cuda()
    masks, pos = tree_masks(parents, cu, kv_len, n)
    k1, v1, sc1 = k.clone(), v.clone(), None if sc is None else sc.clone()
    q = rope_append(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], pos, inv, k[0], v[0], cu, kv_len, table, n, scales=one(sc))
    out = paged_attention(q, k[0], v[0], cu, kv_len, table, n, scales=one(sc), tree=masks)
    target, tokens, _, _ = round_of([n], vocab, 23, follow=0.0)
    i, up = n - 1, parents.tolist()
    while i > 0:                                                # the branch of the last row is the target's choice
        tokens[i] = target[up[i]].argmax()
        i = up[i]
    took = accept_tree(target.cuda(), tokens.cuda(), parents, cu, n)
    keep_rows(k, v, cu, kv_len, table, took, scales=sc)
    path = [p for p in took[0, 4 + n:].tolist() if p >= 0]
    assert len(path) > 3 and path != list(range(len(path)))
    at = torch.tensor(path, device="cuda")
    m = len(path)
    cu1, len1 = torch.tensor([0, m], dtype=torch.int32).cuda(), torch.tensor([base + m], dtype=torch.int32).cuda()
    rows = qkv[at].contiguous()
    plain = torch.arange(base, base + m, dtype=torch.int32, device="cuda")
    q1 = rope_append(rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], plain, inv, k1[0], v1[0], cu1, len1, table, m, scales=one(sc1))
    assert torch.equal(q1, q[at])
    for t in range(base + m):
        p, o = int(table[0, t // page]), t % page
        for x, y in ((k, k1), (v.transpose(3, 4), v1.transpose(3, 4))):
            assert torch.equal(x[0, p, :, o].float(), y[0, p, :, o].float())
        assert sc is None or torch.equal(sc[0, p, :, :, o], sc1[0, p, :, :, o])
    out1 = paged_attention(q1, k1[0], v1[0], cu1, len1, table, m, scales=one(sc1))
    # both are a rounding of bf16 and of the probabilities away from one another's exact value: values of a few units
    assert (out[at].float() - out1.float()).abs().max() <= 2 * 2.0 ** -7 * out1.float().abs().max()
    assert _lib.device_error() == 0

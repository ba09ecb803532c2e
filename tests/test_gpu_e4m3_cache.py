"""A paged cache in 8 bits against its definition in 64 bits (tests/tree_util.py): the rows that rope_append writes as e4m3 numbers with
a power of two each, and the attention of few and of many rows over such pages. Bounds count the roundings."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.kv_pages import move_pages
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.kernels.rope import rope_append
from tests.paged_util import Batch, attention64, attention_bound, rope64
from tests.tree_util import E4M3, Batch8, quantise64, values64

pytestmark = pytest.mark.gpu


def check(b, window=0, sinks=0, **kw):
    print(f"[e4m3] rows={b.rows[:6]} lens={b.lens[:6]} heads={b.heads}/{b.kv_heads} dim={b.dim} page={b.page} window={window}", flush=True)
    lse = torch.full((b.total, b.heads), 7.0, device="cuda")
    out = paged_attention(*b.args(), window=window, sinks=sinks, lse=lse, scales=b.scales.cuda(), **kw)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    want, want_lse = attention64(b, window, sinks)
    err = (out.double().cpu() - want).abs()
    bound = attention_bound(b, window=window, sinks=sinks)
    assert (err <= bound).all(), f"off by {(err / bound).max():.2f} of what the roundings allow"
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse.cpu()), empty)
    assert (out.cpu()[empty] == 0).all()
    assert ((lse.double().cpu() - want_lse).abs()[~empty] <= 1e-5 * (1 + want_lse.abs()[~empty])).all()
    return out


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (7, 1), (12, 4), (16, 1), (9, 3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_head_layouts(heads, kv_heads, dim):
    check(Batch8([1, 3, 2], [1, 70, 333], heads, kv_heads, dim, 32, seed=heads * dim))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_sizes_and_lengths(page, dim):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513]
    check(Batch8([1] * len(lens), lens, 4, 2, dim, page, seed=page + dim))


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 33, 70])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 16), (64, 32), (128, 32), (256, 64), (64, 64), (128, 64), (128, 256)])
def test_rows_of_a_sequence(rows, dim, page):
    check(Batch8([rows, 1, rows], [rows, 40, 200], 8, 2, dim, page, seed=rows))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (64, 17), (100, 200), (5000, 3)])
@pytest.mark.parametrize("rows", [1, 4, 21])
def test_window_and_first_tokens(window, sinks, rows):
    for dim, page in ((64, 16), (128, 64)):
        check(Batch8([rows] * 4, [rows, 60, 129, 700], 6, 2, dim, page, seed=window + rows), window, sinks)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (16, 2), (5, 1)])
def test_prompts_over_short_tables(dim, page, heads, kv_heads):
    check(Batch8([300, 1, 80], [300, 33, 200], heads, kv_heads, dim, page, seed=dim + page))
    check(Batch8([500], [500], heads, kv_heads, dim, page, seed=dim))


def test_sequences_without_rows_or_tokens():
    b = Batch8([0, 2, 1, 0, 3], [0, 50, 0, 20, 2], 4, 2, 64, 16)
    out = check(b)
    assert (out[2] == 0).all() and (out[3] == 0).all() and (out[4] != 0).any()


def test_long_cache_in_many_chunks():
    b = Batch8([1, 2], [9001, 5000], 8, 2, 128, 64, seed=5, width=400)
    check(b)
    check(b, window=3000, sinks=70)
    check(Batch8([20, 9], [3001, 1500], 16, 1, 128, 64, seed=6))      # many rows, split over their tokens


def test_a_row_alone_equals_the_row_in_a_round():
    for dim, heads, kv_heads, window, sinks in ((64, 8, 2, 0, 0), (128, 8, 1, 0, 0), (256, 8, 2, 0, 0), (128, 6, 2, 300, 5)):
        b = Batch8([4, 4], [1030, 77], heads, kv_heads, dim, 16, seed=dim)
        q, k, v, cu, kv_len, table, _ = b.args()
        sc = b.scales.cuda()
        whole = paged_attention(q, k, v, cu, kv_len, table, 4, window, sinks, scales=sc)
        one = torch.arange(3, dtype=torch.int32, device="cuda")
        for i in range(4):
            got = paged_attention(q[i::4].contiguous(), k, v, one, kv_len - 3 + i, table, 1, window, sinks, scales=sc)
            assert torch.equal(got.view(torch.int16), whole[i::4].contiguous().view(torch.int16))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [3, 20])
@pytest.mark.parametrize("tail,tail_exp", [(0x7F, 127), (0xFF, 254), (0x7E, 255), (0x7F, 255), (0xFE, 0)])
def test_unseen_places_do_not_matter(dim, rows, tail, tail_exp):
    """NaN codes, the largest codes and exponents (255 is none) past the tokens, before the window and in pages not held."""
    b = Batch8([rows, 1], [90, 205], 4, 2, dim, 16, tail=tail, tail_exp=tail_exp, seed=3)
    b.table[1, 1:9] = -1
    check(b, window=60, sinks=16)


@pytest.mark.parametrize("rows", [3, 20])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_token_of_nan(dim, rows):
    """A later row's own token is not seen by the rows before it, whatever it holds; a NaN value reaches those that see it alone,
    in its dimension."""
    b = Batch8([rows], [90], 4, 2, dim, 16, seed=4)
    want = check(b)
    page, off = int(b.table[0, 89 // 16]), 89 % 16
    b.v8.view(torch.uint8)[page, :, 5, off] = 0xFF
    got = paged_attention(*b.args(), scales=b.scales.cuda())
    assert torch.equal(got[:-1].view(torch.int16), want[:-1].view(torch.int16))
    assert torch.isnan(got[-1, :, 5]).all()
    keep = [d for d in range(dim) if d != 5]
    assert torch.equal(got[-1][:, keep], want[-1][:, keep])
    b.k8.view(torch.uint8)[page, :, off] = 0x7F
    b.scales[page, :, :, off] = 255
    got = paged_attention(*b.args(), scales=b.scales.cuda())
    assert torch.equal(got[:-1].view(torch.int16), want[:-1].view(torch.int16))
    assert torch.isnan(got[-1]).all()


def test_strided_queries_streams_and_graphs():
    b = Batch8([2, 30], [40, 300], 8, 2, 128, 32, seed=9)
    q, k, v, cu, kv_len, table, rows = b.args()
    sc = b.scales.cuda()
    wide = torch.zeros(32, 12, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10] = q
    want = paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = paged_attention(wide[:, 2:10], k, v, cu, kv_len, table, rows, scales=sc)
        out = torch.zeros_like(q)
        paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc, out=out)
    st.synchronize()
    assert torch.equal(got, want) and torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc, out=out)
    for n in (300, 290, 40):
        kv_len[1] = n
        sc[0, 0, 0, 0] = 100 + n % 7
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, k, v, cu, kv_len, table, rows, scales=sc))


# ---------------------------------------------------------------- the cache write
def turned_bound(x, want, factor=1.0):
    """fp32 products of one rounding each and a sum, of angles within 2^-22 of a turn."""
    return 2.0 ** -21 * abs(factor) * x.double().abs().amax(-1, keepdim=True) * 2


def check_append(rows, lens, heads, kv_heads, dim, page, rot, adjacent=False, axes=1, factor=1.0, seed=0, big=None):
    print(f"[append] rows={rows[:6]} lens={lens[:6]} heads={heads}/{kv_heads} dim={dim} page={page} rot={rot} {adjacent} {axes}", flush=True)
    b = Batch(rows, lens, heads, kv_heads, dim, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 7)
    qkv = torch.randn(b.total + 2, heads + 2 * kv_heads, dim, generator=g).to(torch.bfloat16)     # two rows of padding
    qkv[:, heads:] *= torch.exp2(torch.randint(-9, 10, (b.total + 2, 2 * kv_heads, 1), generator=g)).to(torch.bfloat16)
    if big is not None:
        big(qkv)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    inv = 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    pos = torch.randint(0, 100000, (axes, b.total + 2), generator=g).to(torch.int32)
    axis = torch.arange(rot // 2, dtype=torch.int32) % axes if axes > 1 else None
    n = b.k.shape[0]
    k8 = torch.full((n, kv_heads, page, dim), 0x55, dtype=torch.uint8)
    v8 = torch.full((n, kv_heads, dim, page), 0x55, dtype=torch.uint8)
    sc = torch.full((n, kv_heads, 2, page), 77, dtype=torch.uint8)
    dk, dv, ds = k8.cuda().view(E4M3), v8.cuda().view(E4M3), sc.cuda()
    dq = qkv.cuda()
    out = rope_append(dq[:, :heads], dq[:, heads:heads + kv_heads], dq[:, heads + kv_heads:], pos.cuda(), inv.cuda(), dk, dv,
                      b.cu.cuda(), b.kv_len.cuda(), b.table.cuda(), b.max_rows, axis=None if axis is None else axis.cuda(),
                      adjacent=adjacent, factor=factor, scales=ds)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    turned = rope64(k, pos, inv, axis, adjacent, factor)
    tq = rope64(q, pos, inv, axis, adjacent, factor)[:b.total]
    fine = torch.isfinite(tq)
    assert ((out[:b.total].double().cpu() - tq).abs() <= 2.0 ** -8 * tq.abs() + turned_bound(q[:b.total], tq, factor))[fine].all()
    got_k, got_v, got_s = dk.view(torch.uint8).cpu(), dv.view(torch.uint8).cpu(), ds.cpu()
    # untouched places
    r = 0
    seen = torch.zeros(n, page, dtype=torch.bool)
    for s, m in enumerate(b.rows):
        for i in range(m):
            t = b.lens[s] - m + i
            if t >= 0:
                p, o = int(b.table[s, t // page]), t % page
                seen[p, o] = True
                for kind, x, raw in ((0, turned[r], got_k[p, :, o]), (1, v[r].double(), got_v[p, :, :, o])):
                    e = got_s[p, :, kind, o].double() - 127
                    codes = raw.contiguous().view(E4M3).double()
                    bad = ~torch.isfinite(x)
                    assert torch.equal(torch.isnan(codes), bad)
                    x, codes = torch.where(bad, 0.0, x), torch.where(bad, 0.0, codes)
                    by = torch.exp2(e)[:, None]
                    off = turned_bound(k[r], x, factor) if kind == 0 else torch.zeros(kv_heads, 1, dtype=torch.float64)
                    off = torch.where(torch.isfinite(off), off, torch.full_like(off, math.inf))
                    top = x.abs().amax(1, keepdim=True)
                    # the exponent is the least that holds the maximum (or one beside it where the maximum is that near to the border)
                    assert ((top <= 448 * by + off) & ((top > 224 * by - off) | (e[:, None] == -126))).all()
                    # one rounding: 2^-4 of the value, or half of the least step
                    assert ((codes * by - x).abs() <= (2.0 ** -4 * x.abs()).maximum(2.0 ** -10 * by) * (1 + 2.0 ** -20) + off).all()
                    if kind == 1:
                        want, byte = quantise64(v[r].double())
                        assert torch.equal(got_s[p, :, 1, o], byte)
                        assert torch.equal(torch.nan_to_num(raw.contiguous().view(E4M3).float()), torch.nan_to_num(want.float()))
            r += 1
    free = ~seen
    assert (got_k.transpose(1, 2)[free] == 0x55).all() and (got_v.permute(0, 3, 1, 2)[free] == 0x55).all()
    assert (got_s.permute(0, 3, 1, 2)[free] == 77).all()


@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 16), (128, 128), (128, 48), (256, 256), (256, 64), (256, 16)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append(dim, rot, page):
    check_append([1, 3, 9, 40], [1, 20, 9, 133], 4, 2, dim, page, rot, seed=dim + rot)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (7, 7), (32, 8), (16, 1)])
def test_append_head_layouts(heads, kv_heads):
    check_append([1, 1, 17], [1, 64, 31], heads, kv_heads, 128, 16, 128, seed=heads)


def test_append_variants():
    check_append([5, 0, 2, 3], [3, 0, 64, 90], 4, 2, 128, 32, 64, adjacent=True, axes=3, factor=0.25, seed=1)   # two rows too many
    check_append([1] * 30, list(range(1, 31)), 4, 4, 64, 16, 32, axes=3, seed=2)
    check_append([200], [777], 8, 2, 256, 64, 64, axes=3, seed=3)


def test_append_values_at_the_edges():
    """Vectors of zeros, of one value on a border, subnormal and very large ones, infinities and NaN."""
    def big(qkv):
        qkv[0, 4:] = 0
        qkv[1, 4:] = 0
        qkv[1, 4:, 3] = 448.0 * 4
        qkv[2, 4:] = 2.0 ** -133
        qkv[3, 6:] *= 2.0 ** 118
        qkv[4, 4:, 7] = math.inf
        qkv[5, 6:, 9] = math.nan
        qkv[5, 6:, 10] = -math.inf
        qkv[6, 6:] = math.nan
        qkv[7, 4:, :] = 1.875
    check_append([9], [20], 4, 2, 64, 16, 16, seed=4, big=big)


@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (3, 64, 16), (2, 128, 64), (1, 256, 256)])
def test_pages_move_with_their_scales(kv_heads, dim, page):
    """Pages of one KB and of an odd number of them, ids outside the cache, a table that follows."""
    g = torch.Generator().manual_seed(dim)
    n, layers = 23, 3
    k, v, sc = (torch.randint(0, 256, s, generator=g, dtype=torch.uint8) for s in (
        (layers, n, kv_heads, page, dim), (layers, n, kv_heads, dim, page), (layers, n, kv_heads, 2, page)))
    perm = torch.randperm(n, generator=g)
    src, dst = perm[:9].to(torch.int32), perm[9:18].to(torch.int32)
    table = torch.randint(-1, n, (5, 40), generator=g).to(torch.int32)
    dk, dv, ds, dt = k.cuda().view(E4M3), v.cuda().view(E4M3), sc.cuda(), table.cuda()
    move_pages(dk, dv, src.cuda(), dst.cuda(), dt, scales=ds)
    to = {int(a): int(b) for a, b in zip(src, dst)}
    for t, d in ((k, dk.view(torch.uint8)), (v, dv.view(torch.uint8)), (sc, ds)):
        t[:, dst.long()] = t[:, src.long()].clone()
        assert torch.equal(t, d.cpu())
    assert torch.equal(dt.cpu(), torch.tensor([[to.get(p, p) for p in row] for row in table.tolist()], dtype=torch.int32))
    assert _lib.device_error() == 0
    move_pages(dk, dv, torch.tensor([n, 1], dtype=torch.int32).cuda(), torch.tensor([0, -1], dtype=torch.int32).cuda(), scales=ds)
    assert _lib.device_error() == 32
    assert torch.equal(sc, ds.cpu()) and torch.equal(k, dk.view(torch.uint8).cpu())


def test_written_rows_are_read_back():
    """A prompt and single tokens through the write and the attention, against the attention of the rows as they were."""
    b = Batch([40, 1], [40, 1], 8, 2, 128, 32, seed=11)
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(41, h, 128, generator=g).to(torch.bfloat16).cuda() for h in (8, 2, 2))
    n = b.k.shape[0]
    k8 = torch.zeros(n, 2, 32, 128, dtype=torch.uint8, device="cuda").view(E4M3)
    v8 = torch.zeros(n, 2, 128, 32, dtype=torch.uint8, device="cuda").view(E4M3)
    sc = torch.zeros(n, 2, 2, 32, dtype=torch.uint8, device="cuda")
    inv = torch.tensor([1.0] * 8, dtype=torch.float64, device="cuda")
    pos = torch.zeros(41, dtype=torch.int32, device="cuda")
    args = (b.cu.cuda(), b.kv_len.cuda(), b.table.cuda(), 40)
    q = rope_append(q, k, v, pos, inv, k8, v8, *args, scales=sc)
    out = paged_attention(q, k8, v8, *args, scales=sc)
    b.q = q.cpu()
    b.k, b.v = values64(k8.cpu(), sc.cpu(), True), values64(v8.cpu(), sc.cpu(), False)
    want, _ = attention64(b)
    assert ((out.double().cpu() - want).abs() <= attention_bound(b)).all()

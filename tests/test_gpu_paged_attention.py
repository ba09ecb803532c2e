"""Attention over a paged cache against its definition in 64 bits (tests/paged_util.py): head layouts, types, page sizes,
lengths from nothing to several chunks, windows with first tokens, rows that see nothing, what the cache holds at places
that no row sees, strides, streams and captured graphs. Tolerances count the roundings (paged_util.attention_bound)."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from tests.paged_util import Batch, attention64, attention_bound

pytestmark = pytest.mark.gpu

ERR_PAGE, ERR_BATCH = 32, 64


def check(b, window=0, sinks=0, **kw):
    args = b.args()
    lse = torch.full((b.total, b.heads), 7.0, device="cuda")
    out = paged_attention(*args, window=window, sinks=sinks, lse=lse, **kw)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    want, want_lse = attention64(b, window, sinks)
    err = (out.double().cpu() - want).abs()
    bound = attention_bound(b, window=window, sinks=sinks)
    assert (err <= bound).all(), f"off by {(err / bound).max():.2f} of what the roundings allow"
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse.cpu()), empty)
    assert (out.cpu()[empty] == 0).all()
    # fp32 scores of `dim` products of values up to a few units, and a sum of their exponentials
    assert ((lse.double().cpu() - want_lse).abs()[~empty] <= 1e-5 * (1 + want_lse.abs()[~empty])).all()
    return out


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (7, 1), (12, 4), (16, 1), (9, 3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_layouts(heads, kv_heads, dim, dtype):
    check(Batch([1, 3, 2], [1, 70, 333], heads, kv_heads, dim, 32, dtype, seed=heads * dim))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_sizes_and_lengths(page, dim):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513]
    check(Batch([1] * len(lens), lens, 4, 2, dim, page, seed=page + dim))


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 33])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_a_sequence(rows, dim):
    check(Batch([rows, 1, rows], [rows, 40, 200], 8, 2, dim, 16, seed=rows))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (64, 17), (100, 200), (5000, 3)])
@pytest.mark.parametrize("rows", [1, 4, 21])
def test_window_and_first_tokens(window, sinks, rows):
    for dim, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        check(Batch([rows] * 4, [rows, 60, 129, 700], 6, 2, dim, 16, dtype, seed=window + rows), window, sinks)


def test_sequences_without_rows_or_tokens():
    b = Batch([0, 2, 1, 0, 3], [0, 50, 0, 20, 2], 4, 2, 64, 16)     # row 2: no token at all; the last: 3 rows, 2 tokens
    out = check(b)
    assert (out[2] == 0).all() and (out[3] == 0).all() and (out[4] != 0).any()


def test_long_cache_in_many_chunks():
    b = Batch([1, 2], [9001, 5000], 8, 2, 128, 64, seed=5, width=400)   # a table far wider than the sequences
    check(b)
    check(b, window=3000, sinks=70)


def test_a_row_alone_equals_the_row_in_a_round():
    """Bit for bit: T rows of a verify round and T calls of one row, on tables of one width."""
    for dim, heads, kv_heads, window, sinks in ((64, 8, 2, 0, 0), (128, 8, 1, 0, 0), (256, 8, 2, 0, 0), (128, 6, 2, 300, 5)):
        b = Batch([4, 4], [1030, 77], heads, kv_heads, dim, 16, seed=dim)
        q, k, v, cu, kv_len, table, _ = b.args()
        lse = torch.empty(8, heads, device="cuda")
        whole = paged_attention(q, k, v, cu, kv_len, table, 4, window, sinks, lse=lse)
        one = torch.arange(3, dtype=torch.int32, device="cuda")
        for i in range(4):
            l1 = torch.empty(2, heads, device="cuda")
            got = paged_attention(q[i::4].contiguous(), k, v, one, kv_len - 3 + i, table, 1, window, sinks, lse=l1)
            assert torch.equal(got.view(torch.int16), whole[i::4].contiguous().view(torch.int16))
            assert torch.equal(l1, lse[i::4])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_unseen_places_do_not_matter(dim, bad, dtype):
    """The cache past a sequence's tokens, before its window and in pages it does not hold."""
    b = Batch([3, 1], [90, 205], 4, 2, dim, 16, dtype, tail=bad, seed=3)
    b.table[1, 1:9] = -1                                  # tokens 16 .. 143 are not held: the window begins at 145
    check(b, window=60, sinks=16)
    # a later row's own token is not seen by the rows before it
    b = Batch([3], [90], 4, 2, dim, 16, dtype, seed=4)
    want = check(b)
    last = int(b.table[0, 89 // 16]), 89 % 16
    b.k[last[0], :, last[1]] = bad
    b.v[last[0], :, :, last[1]] = bad
    got = paged_attention(*b.args())
    assert torch.equal(got[:2].view(torch.int16), want[:2].view(torch.int16))
    assert torch.isnan(got[2]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_value_in_sight(dtype):
    """An infinity in a tile that one row sees and another does not: the rows that see it hold it, the others their value."""
    b = Batch([2], [70], 2, 1, 64, 16, dtype, seed=6)
    page, off = int(b.table[0, 69 // 16]), 69 % 16
    want = paged_attention(*b.args())
    b.v[page, 0, 5, off] = math.inf
    b.v[page, 0, 6, off] = -math.inf
    got = paged_attention(*b.args())
    assert torch.equal(got[0].view(torch.int16), want[0].view(torch.int16))
    assert (got[1, :, 5] == math.inf).all() and (got[1, :, 6] == -math.inf).all()
    keep = [d for d in range(64) if d not in (5, 6)]
    assert torch.equal(got[1][:, keep], want[1][:, keep])


def test_strided_queries_outputs_and_padding_rows():
    b = Batch([1, 2, 1], [30, 31, 200], 8, 2, 128, 32, seed=8)
    q, k, v, cu, kv_len, table, n = b.args()
    fused = torch.zeros(6, 13, 128, dtype=q.dtype, device="cuda")   # q inside a wider projection, with two padding rows
    fused[:4, 2:10] = q
    out = torch.full((6, 8, 128), 5.0, dtype=q.dtype, device="cuda")
    lse = torch.full((6, 8), 5.0, device="cuda")
    got = paged_attention(fused[:, 2:10], k, v, cu, kv_len, table, n, out=out, lse=lse)
    assert got.data_ptr() == out.data_ptr()
    assert (out[4:] == 5).all() and (lse[4:] == 5).all()
    assert torch.equal(out[:4].view(torch.int16), paged_attention(q, k, v, cu, kv_len, table, n).view(torch.int16))


def test_scale():
    b = Batch([2], [100], 4, 4, 64, 16, seed=9)
    got = paged_attention(*b.args(), scale=0.3).double().cpu()
    assert ((got - attention64(b, scale=0.3)[0]).abs() <= attention_bound(b, scale=0.3)).all()


def test_large_scores():
    """Scores of some hundreds: the running maximum moves by large steps and nothing overflows."""
    b = Batch([2], [600], 4, 2, 64, 16, torch.float16, seed=10)
    b.q *= 20
    got = paged_attention(*b.args()).double().cpu()
    want = attention64(b)[0]
    # a score of size S is off by S 2^-22 in fp32 sums of 64 products, its probability by that much relative
    s = (b.q.double().abs().amax() * 5 * 8).item()
    assert ((got - want).abs() <= attention_bound(b) + 2 * s * 2.0 ** -22 * attention64(b, absolute=True)[0]).all()


def test_offsets_past_32_bits():
    """Pages whose byte offset in the cache passes 2^32 and whose element offset passes 2^31."""
    kv_heads, page, dim, n = 8, 256, 256, 4200                         # 4.4 GB of keys
    k = torch.zeros(n, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(n, kv_heads, dim, page, dtype=torch.bfloat16, device="cuda")
    b = Batch([1], [300], 8, 8, dim, page, seed=11, spare=0)
    far = torch.tensor([n - 1, n - 3], dtype=torch.int32)
    for j in range(2):
        k[int(far[j])] = b.k[int(b.table[0, j])].cuda()
        v[int(far[j])] = b.v[int(b.table[0, j])].cuda()
    want = paged_attention(*b.args())
    q, _, _, cu, kv_len, _, _ = b.args()
    got = paged_attention(q, k, v, cu, kv_len, far.cuda()[None].contiguous(), 1)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_bad_pages_and_batches_are_raised():
    """Page ids outside the cache where a token is needed, row counts and lengths that contradict the call: cut, raised,
    the other sequences as ever."""
    b = Batch([1, 1], [100, 100], 4, 2, 64, 16, seed=12)
    want, _ = attention64(b)
    b.table[0, 2] = b.k.shape[0]
    got = paged_attention(*b.args())
    assert _lib.device_error() == ERR_PAGE and _lib.device_error() == 0
    assert ((got.double().cpu() - attention64(b)[0]).abs() <= attention_bound(b)).all()    # as if not held
    b = Batch([1, 1], [100, 100], 4, 2, 64, 16, seed=12)
    q, k, v, cu, kv_len, table, _ = b.args()
    for bad_cu, bad_len in (([0, 1, 3], [100, 100]), ([0, 1, 2], [100, 1000]), ([-1, 1, 2], [100, 100]),
                            ([0, 1, 2], [100, -5])):
        out = paged_attention(q, k, v, torch.tensor(bad_cu, dtype=torch.int32, device="cuda"),
                              torch.tensor(bad_len, dtype=torch.int32, device="cuda"), table, 1)
        assert _lib.device_error() == ERR_BATCH
        if bad_cu[0] == 0 and bad_len[0] == 100:
            assert ((out[0].double().cpu() - want[0]).abs() <= attention_bound(b)[0]).all()
    assert _lib.device_error() == 0


def test_other_stream_and_captured_graph():
    """Work on a side stream, and a captured call that follows the lengths, tables and queries written between replays."""
    b = Batch([1, 1, 1], [900, 35, 600], 8, 2, 128, 16, seed=13, width=64)
    q, k, v, cu, kv_len, table, n = b.args()
    want = paged_attention(q, k, v, cu, kv_len, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(q, k, v, cu, kv_len, table, n)
    side.synchronize()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(want)
    with torch.cuda.graph(graph):
        paged_attention(q, k, v, cu, kv_len, table, n, out=out)
    for step in range(4):
        q.copy_(torch.randn_like(q))
        kv_len.copy_(torch.tensor([900 - 100 * step, 35 - step, 16 * step], dtype=torch.int32))
        graph.replay()
        want = paged_attention(q, k, v, cu, kv_len, table, n)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)), step
    assert _lib.device_error() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [
    (1, 1, 64, 16, torch.bfloat16), (4, 1, 64, 64, torch.float16), (5, 1, 128, 32, torch.bfloat16), (8, 4, 128, 64, torch.float16),
    (3, 1, 256, 16, torch.bfloat16), (2, 2, 256, 128, torch.float16), (16, 1, 64, 256, torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (64, 64), (130, 17)])
def test_prompt_chunks(heads, kv_heads, dim, page, dtype, window, sinks):
    """Chunks of many rows, from an empty cache and behind one, of mixed sizes, with lengths at the edges of tiles."""
    check(Batch([130, 9, 1, 0, 64, 65], [130, 200, 77, 50, 64, 129], heads, kv_heads, dim, page, dtype, seed=heads + dim),
          window, sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_split_over_its_length(dim):
    """Few row tiles behind a long context: the tokens are shared out and joined."""
    b = Batch([20, 33], [2100, 3333], 4, 2, dim, 64, seed=dim)
    check(b)
    check(b, window=1500, sinks=40)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("long", [False, True])
def test_prompt_unseen_places_do_not_matter(dim, bad, long):
    """As for few rows: past the tokens, before the window, in pages not held, at later rows' tokens; with and without the
    split over the length."""
    n = 2500 if long else 150
    b = Batch([40, 12], [n, 205], 4, 2, dim, 16, tail=bad, seed=3)
    b.table[1, 1:6] = -1                                  # tokens 16 .. 95 are not held: the windows begin at 134 and later
    check(b, window=60, sinks=16)
    b = Batch([40], [n], 4, 2, dim, 16, seed=4)
    want = check(b)
    at = n - 10                                           # the token of row 30: seen by it and the rows behind it
    page, off = int(b.table[0, at // 16]), at % 16
    b.k[page, :, off] = bad
    got = paged_attention(*b.args())
    assert torch.equal(got[:30].view(torch.int16), want[:30].view(torch.int16)) and torch.isnan(got[30:]).all()
    b = Batch([40], [n], 4, 2, dim, 16, seed=4)
    b.v[page, 1, 7, off] = bad
    got = paged_attention(*b.args())
    keep = torch.ones(4, dim, dtype=torch.bool, device="cuda")
    keep[2:, 7] = False
    assert torch.equal(got[:30].view(torch.int16), want[:30].view(torch.int16))
    assert torch.equal(got[30:][:, keep].view(torch.int16), want[30:][:, keep].view(torch.int16))
    seen = got[30:, 2:, 7].float()
    assert torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all()


def test_prompt_bad_pages_are_raised():
    b = Batch([100], [400], 4, 2, 64, 16, seed=12)
    b.table[0, 2] = -1
    b.table[0, 22] = b.k.shape[0]
    got = paged_attention(*b.args())
    assert _lib.device_error() == ERR_PAGE
    assert ((got.double().cpu() - attention64(b)[0]).abs() <= attention_bound(b)).all()


def test_prompt_strides_padding_rows_and_graph():
    b = Batch([70, 20], [70, 300], 8, 2, 128, 32, seed=8)
    q, k, v, cu, kv_len, table, n = b.args()
    fused = torch.zeros(95, 13, 128, dtype=q.dtype, device="cuda")
    fused[:90, 2:10] = q
    out = torch.full((95, 8, 128), 5.0, dtype=q.dtype, device="cuda")
    lse = torch.full((95, 8), 5.0, device="cuda")
    graph = torch.cuda.CUDAGraph()
    paged_attention(fused[:, 2:10], k, v, cu, kv_len, table, n, out=out, lse=lse)
    assert (out[90:] == 5).all() and (lse[90:] == 5).all()
    want = paged_attention(q, k, v, cu, kv_len, table, n)
    assert torch.equal(out[:90].view(torch.int16), want.view(torch.int16))
    with torch.cuda.graph(graph):
        paged_attention(fused[:, 2:10], k, v, cu, kv_len, table, n, out=out)
    for step in range(3):
        fused.normal_()
        kv_len[1] -= step
        graph.replay()
        want = paged_attention(fused[:90, 2:10], k, v, cu, kv_len, table, n)
        assert torch.equal(out[:90].view(torch.int16), want.view(torch.int16)), step


def test_output_behind_its_queries():
    b = Batch([2, 12], [300, 400], 8, 2, 64, 16, seed=5)
    q, *rest = b.args()
    want = paged_attention(q, *rest)
    both = torch.empty((2, *q.shape), dtype=q.dtype, device="cuda")
    both[0] = q
    assert paged_attention(both[0], *rest, out=both[1]).data_ptr() == both[1].data_ptr()
    assert torch.equal(both[1], want) and torch.equal(both[0], q)
    with pytest.raises(_lib.SsmoeError, match="overlap"):
        paged_attention(both[0], *rest, out=both[0])


@pytest.mark.parametrize("window", [16370, 16376, 16379, 16380])
def test_rows_under_a_window_have_the_bits_they_have_alone(window):
    """The rows of a call and each row alone, where a chunk's size is about to change: 2 x (window + rows + first tokens) tokens over
    256 workgroups pass 128."""
    b = Batch([4], [20000], 4, 2, 64, 64, seed=window)
    q, k, v, cu, kv_len, table, n = b.args()
    got = paged_attention(q, k, v, cu, kv_len, table, n, window=window, sinks=4)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for i in range(4):
        alone = paged_attention(q[i:i + 1], k, v, one, kv_len - 3 + i, table, 1, window=window, sinks=4)
        assert torch.equal(got[i], alone[0]), i


@pytest.mark.parametrize("rows,heads", [(1, 4), (1, 24), (3, 24), (8, 16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_short_sequences_on_a_wide_table(dim, rows, heads):
    """A table of 8,192 tokens is split into chunks: sequences that end at, before and behind a chunk's and a tile's end."""
    lens = [rows, 31, 32, 33, 127, 128, 129, 255, 257, 511, 512, 513, 1025, 2049]
    for page, window, sinks in ((64, 0, 0), (16, 100, 7)):
        check(Batch([rows] * len(lens), [max(n, rows) for n in lens], heads, 2, dim, page, seed=dim + rows, width=8192 // page),
              window, sinks)


def test_a_row_is_the_same_on_tables_of_one_chunk_and_of_several():
    """A table of 512 tokens of 128 dimensions is one chunk, one of 4,096 is several: both against the definition, and one against the other within twice
    its bound."""
    outs = []
    for width in (32, 256):
        b = Batch([2, 1], [500, 77], 8, 2, 128, 16, seed=3, width=width)
        outs.append(check(b).double().cpu())
    assert ((outs[0] - outs[1]).abs() <= 2 * attention_bound(b)).all()


@pytest.mark.parametrize("rows", [2, 9])
def test_infinite_value_past_32_bits(rows):
    """An infinity that the last row alone sees, in a page whose byte offset passes 2^32."""
    kv_heads, page, dim, n = 8, 256, 256, 4200
    v = torch.zeros(n, kv_heads, dim, page, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(n, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda")
    b = Batch([rows], [300], 8, 8, dim, page, seed=12, spare=0)
    b.v[int(b.table[0, 1]), :, 7, 299 - 256] = math.inf
    far = torch.tensor([n - 1, n - 3], dtype=torch.int32)
    for j in range(2):
        k[int(far[j])] = b.k[int(b.table[0, j])].cuda()
        v[int(far[j])] = b.v[int(b.table[0, j])].cuda()
    want = paged_attention(*b.args())
    assert (want[-1, :, 7] == math.inf).all() and torch.isfinite(want[:-1]).all()
    q, _, _, cu, kv_len, _, m = b.args()
    got = paged_attention(q, k, v, cu, kv_len, far.cuda()[None].contiguous(), m)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))

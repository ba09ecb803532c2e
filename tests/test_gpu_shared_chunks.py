"""Calls whose row tiles share their chunks (many rows over e4m3 pages and of trees on wide tables), from one sequence to more than a wave
has lanes, against the definitions in 64 bits. Every test asks whether its call is of that form, by the workspace that it needs."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels import paged_attention as pa
from tests import test_gpu_e4m3_cache as causal, test_gpu_tree as tree
from tests.test_gpu_tree import as_int64, make, trees

pytestmark = pytest.mark.gpu

WIDTH = 4160   # tokens of a table: beyond what the few-row form takes


def shares(b, words, kind):
    """Whether the call's workspace is that of shared chunks: their sums for 128 columns of each key head, then a word a sequence and one."""
    cap, group = b.table.shape[1] * b.page, b.heads // b.kv_heads
    tiles, parts = -(-b.max_rows * group // 128), 2 if b.dim == 256 else 1
    want = 512 // (b.kv_heads * parts)
    slots = min(want, len(b.rows) * tiles * -(-cap // 128)) * b.kv_heads * 128
    e8 = kind == "e4m3"
    nb = pa._plan(b.q, b.k8 if e8 else b.k, b.v8 if e8 else b.v, b.cu, b.kv_len, b.table, b.max_rows, 0, 0, None, b.scales if e8 else None,
                  as_int64(words) if words else None)[3]
    return want >= 2 * len(b.rows) * tiles and nb == -(-slots * b.dim * 4 // 256) * 256 + slots * 8 + 4 * (1 + len(b.rows))


def batch(kind, seqs, heads, kv_heads, dim, page, most, longest=900, seed=0):
    """Rows and lengths of every size, none among them; one of the longest behind the first 64."""
    g = torch.Generator().manual_seed(seed + seqs)
    rows = [int(torch.randint(0, most + 1, (1,), generator=g)) for _ in range(seqs)]
    lens = [int(torch.randint(0, longest, (1,), generator=g)) if i % 5 else i % 40 for i in range(seqs)]
    rows[-1], lens[-1], rows[0] = most, 4000, most
    if seqs > 2:
        rows[1] = 0
    if seqs > 66:
        rows[64], lens[64], rows[63], lens[63] = most, 2500, most, 1700
    return make(kind, rows, lens, heads, kv_heads, dim, page, seed=seed + seqs, width=WIDTH // page)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("seqs", [1, 2, 3, 63, 64, 65, 128, 130, 250])
def test_trees_of_many_sequences(kind, seqs):
    b = batch(kind, seqs, 8, 1, 64, 16, 12)
    words = trees(b)
    assert shares(b, words, kind)
    tree.check(b, words)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("seqs,heads,kv_heads,dim,page,most", [(65, 16, 1, 64, 64, 16), (70, 14, 2, 128, 32, 12), (66, 8, 1, 256, 32, 10),
                                                             (100, 8, 1, 128, 64, 20), (33, 16, 2, 128, 16, 17)])
def test_trees_of_many_sequences_by_layouts(kind, seqs, heads, kv_heads, dim, page, most):
    """Two row tiles a sequence, two key heads, halves of the output."""
    b = batch(kind, seqs, heads, kv_heads, dim, page, most, longest=300)
    words = trees(b)
    assert shares(b, words, kind)
    tree.check(b, words)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 130])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_causal_rows_of_many_sequences(seqs, dim, page):
    b = batch("e4m3", seqs, 8, 1, dim, page, 12, longest=500)
    assert shares(b, None, "e4m3")
    causal.check(b)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_captured_call_of_many_sequences_follows_their_lengths(kind):
    b = batch(kind, 90, 8, 1, 64, 16, 12)
    words = trees(b)
    assert shares(b, words, kind)
    q, k, v, cu, kv_len, table, most = b.args()
    sc, mask, out = b.scales.cuda() if kind == "e4m3" else None, as_int64(words).cuda(), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pa.paged_attention(q, k, v, cu, kv_len, table, most, scales=sc, tree=mask, out=out)
    full = kv_len.clone()
    for i in range(4):
        kv_len.copy_(torch.where(torch.arange(90, device="cuda") % 4 == i, full // 3, full) if i else full)
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pa.paged_attention(q, k, v, cu, kv_len, table, most, scales=sc, tree=mask))
    kv_len.zero_()                                            # no sequence has tokens: every row sees nothing
    out.fill_(9)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 0).all()
    assert _lib.device_error() == 0

"""Trees of drafts and a cache in 8 bits without a GPU: what the entry points refuse before a device is touched (addresses are
dummies), the Python checks, and the pages of a cache in 8 bits."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.accept import TreeResult
from slotstream_spark_amd.kernels import kv_pages, paged_attention as pa, rope, tree
from slotstream_spark_amd.memory.kv_pages import KVPages
from tests.test_paged_host import EINVAL, L, attn, rope_args  # noqa: F401  (L is a fixture)
from tests.test_kv_pages import HostPages, check
from tests.tree_util import E4M3, Batch8, accept64, masks_of, random_parents

M = 1 << 24
ATTN = {n: (i + 1) * M for i, n in enumerate(["q", "k_pages", "v_pages", "cu_rows", "kv_len", "table", "out", "lse", "ws"])}
SC, TR = 20 * M, 21 * M


def test_attention_refuses(L):  # noqa: F811
    call = lambda sc=SC, tr=TR, **kw: L.ssmoe_paged_attention_ext(attn(**{**ATTN, **kw}), sc, tr, None)  # noqa: E731
    for kw, msg in ((dict(type=1), b"SSMOE_BF16"), (dict(max_rows=65), b"at most 64 rows"), (dict(max_rows=20, window=19), b"window must hold"),
                    (dict(sc=SC + 8), b"16-byte"), (dict(tr=TR + 4), b"8-byte"), (dict(tr=ATTN["out"]), b"overlap"),
                    (dict(sc=ATTN["out"]), b"overlap"), (dict(tr=ATTN["lse"] - 8), b"overlap"), (dict(dim=96), b"dim must")):
        assert call(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())
    # a 16-bit call may have more rows and narrower windows, and e4m3 pages are half as long: nothing behind them overlaps
    assert L.ssmoe_paged_attention_ext_workspace_bytes(attn(max_rows=65), 0, 0) >= 0
    assert L.ssmoe_paged_attention_ext_workspace_bytes(attn(max_rows=65), 0, 1) == -1
    assert L.ssmoe_paged_attention_ext_workspace_bytes(attn(type=1), 1, 0) == -1
    assert L.ssmoe_paged_attention_ext_workspace_bytes(attn(type=1), 0, 1) >= 0
    assert L.ssmoe_paged_attention_ext(attn(rows=0, q=None), None, TR, None) == 0


def test_rope_refuses(L):  # noqa: F811
    at = {n: (i + 1) * M for i, n in enumerate(["q", "k", "v", "positions", "inv_freq", "k_pages", "v_pages", "cu_rows", "kv_len",
                                                "table", "q_out"])}
    call = lambda sc=SC, **kw: L.ssmoe_rope_append_e4m3(rope_args(**{**at, **kw}), sc, None)  # noqa: E731
    for kw, msg in ((dict(type=1), b"SSMOE_BF16"), (dict(sc=None), b"scales"), (dict(sc=at["k_pages"]), b"overlap"),
                    (dict(sc=at["v"]), b"overlap"), (dict(sc=at["q_out"] + 16), b"overlap"), (dict(rot=24), b"rot must be")):
        assert call(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())


def test_move_refuses(L):  # noqa: F811
    def move(k=M, v=2 * M, sc=SC, layers=2, n_pages=10, page_bytes=1024, scale_bytes=32, src=3 * M, dst=4 * M, n=3, table=None, entries=0):
        return L.ssmoe_move_pages_e4m3(k, v, sc, layers, n_pages, page_bytes, scale_bytes, src, dst, n, table, entries, None)
    for kw, msg in ((dict(page_bytes=1000), b"multiple of 1024"), (dict(scale_bytes=0), b"scale_bytes"), (dict(scale_bytes=40), b"scale_bytes"),
                    (dict(scale_bytes=2048), b"scale_bytes"), (dict(sc=None), b"scales"), (dict(sc=SC + 4), b"16-byte"),
                    (dict(sc=M), b"overlap"), (dict(src=SC + 32), b"overlap")):
        assert move(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())
    assert move(n=0, k=None) == 0


def test_tree_calls_refuse(L):  # noqa: F811
    masks = lambda p=M, cu=2 * M, kv=3 * M, m=4 * M, pos=5 * M, rows=9, seqs=2, most=8: L.ssmoe_tree_masks(  # noqa: E731
        p, cu, kv, m, pos, rows, seqs, most, None)
    for kw, msg in ((dict(most=65), b"max_rows in 1"), (dict(most=0), b"max_rows in 1"), (dict(rows=-1), b"rows"), (dict(p=None), b"non-null"),
                    (dict(kv=None), b"non-null"), (dict(m=4 * M + 4), b"8-byte"), (dict(m=M - 8), b"overlap"), (dict(pos=2 * M), b"overlap"),
                    (dict(pos=4 * M + 64), b"overlap")):
        assert masks(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())
    assert masks(rows=0, p=None) == 0 and masks(seqs=0, p=None) == 0
    size = lambda rows=9, vocab=1000: L.ssmoe_accept_tree_workspace_bytes(rows, 2, 8, vocab)  # noqa: E731
    assert size() == 9 * 8 and size(vocab=0) == -1 and size(rows=-1) == -1 and size(vocab=(1 << 24) + 1) == -1
    assert size(rows=64, vocab=248320) % 8 == 0
    accept = lambda t=M, k=2 * M, p=3 * M, cu=4 * M, rows=9, most=8, vocab=1000, ws=5 * M, nb=72, out=6 * M: L.ssmoe_accept_tree(  # noqa: E731
        t, k, p, cu, rows, 2, most, vocab, ws, nb, out, None)
    for kw, msg in ((dict(most=65), b"max_rows in 1"), (dict(t=None), b"non-null"), (dict(out=None), b"non-null"), (dict(ws=None), b"workspace holds 0"),
                    (dict(nb=71), b"workspace holds 71"), (dict(ws=5 * M + 4), b"8-byte"), (dict(out=M + 16), b"overlap"),
                    (dict(ws=M + 9 * 4000 - 8), b"overlap"), (dict(out=5 * M + 64), b"overlap"), (dict(t=M + 2), b"4-byte")):
        assert accept(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())
    keep = lambda k=M, v=2 * M, sc=None, layers=2, pages=10, h=2, page=16, dim=64, size=2, cu=3 * M, kv=4 * M, t=5 * M, w=8, took=6 * M, rows=16, most=8: (  # noqa: E731,E501
        L.ssmoe_keep_rows(k, v, sc, layers, pages, h, page, dim, size, cu, kv, t, w, took, rows, 2, most, None))
    for kw, msg in ((dict(most=65), b"at most 64"), (dict(size=4), b"must be 1"), (dict(size=1), b"scales"), (dict(layers=0), b"layers"),
                    (dict(page=24), b"page must"), (dict(took=None), b"non-null"), (dict(k=M + 8), b"16-byte"), (dict(v=M + 4096), b"overlap"),
                    (dict(took=2 * M + 64), b"overlap"), (dict(size=1, sc=M + 64), b"overlap"), (dict(pages=1 << 31), b"n_pages")):
        assert keep(**kw) == EINVAL, kw
        assert msg in L.ssmoe_last_error(), (kw, L.ssmoe_last_error())
    assert keep(rows=0, k=None) == 0


def test_python_refusals():
    b = Batch8([1, 2], [10, 20], 4, 2, 64, 16)
    good = dict(zip(("q", "k_pages", "v_pages", "cu_rows", "kv_len", "table", "max_rows"), b.args("cpu")), scales=b.scales)
    words = torch.ones(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="same GPU"):
        pa.paged_attention(**good, tree=words)
    for kw, msg in ((dict(scales=None), "with scales"), (dict(scales=b.scales[:1]), "scales must be"), (dict(scales=b.scales.float()), "scales must be"),
                    (dict(scales=b.scales.transpose(0, 1)), "scales must be"), (dict(q=b.q.half()), "bfloat16"), (dict(tree=words.int()), "tree must be"),
                    (dict(tree=words[:2]), "tree must be"), (dict(tree=torch.ones(6, dtype=torch.int64)[::2]), "tree must be"),
                    (dict(tree=words, max_rows=65), "at most 64"), (dict(tree=words, window=1), "window must hold"),
                    (dict(k_pages=b.k8.float(), v_pages=b.v8.float()), "belong to")):
        with pytest.raises(ValueError, match=msg):
            pa.paged_attention(**{**good, **kw})
    inv, pos, kv = torch.ones(8, dtype=torch.float64), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    args = (b.q, kv, kv, pos, inv, b.k8, b.v8, b.cu, b.kv_len, b.table, 2)
    with pytest.raises(ValueError, match="same GPU"):
        rope.rope_append(*args, scales=b.scales)
    for sc, msg in ((None, "with scales"), (b.scales[..., :8], "scales must be")):
        with pytest.raises(ValueError, match=msg):
            rope.rope_append(*args, scales=sc)
    k, v = torch.zeros(2, 5, 2, 16, 64).to(E4M3), torch.zeros(2, 5, 2, 64, 16).to(E4M3)
    sc, took = torch.zeros(2, 5, 2, 2, 16, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.int32)
    good = dict(k=k, v=v, cu_rows=b.cu, kv_len=b.kv_len, table=b.table, accepted=took, scales=sc)
    with pytest.raises(ValueError, match="same GPU"):
        tree.keep_rows(**good)
    for kw, msg in ((dict(scales=None), "with scales"), (dict(k=k.float(), v=v.float()), "with scales"), (dict(v=v.transpose(3, 4)), "v must be"),
                    (dict(scales=sc[:1]), "scales must be"), (dict(accepted=took[:, :7]), "accepted must be"), (dict(accepted=took[:1]), "accepted must be"),
                    (dict(accepted=torch.zeros(2, 134, dtype=torch.int32)), "accepted must be"), (dict(k=k[0], v=v[0]), "k must be"),
                    (dict(k=k[:, :, :, :8], v=v[..., :8]), "pages hold"), (dict(kv_len=b.kv_len.long()), "int32")):
        with pytest.raises(ValueError, match=msg):
            tree.keep_rows(**{**good, **kw})
    with pytest.raises(ValueError, match="same GPU"):
        tree.tree_masks(pos, b.cu, b.kv_len, 2)
    for args, msg in (((pos.long(), b.cu, b.kv_len, 2), "parents"), ((pos, b.cu, b.kv_len, 65), "1 to 64"), ((pos, b.cu, b.kv_len[:1], 2), "kv_len"),
                      ((pos, b.cu[None], b.kv_len, 2), "cu_rows"), ((pos[None], b.cu, b.kv_len, 2), "parents")):
        with pytest.raises(ValueError, match=msg):
            tree.tree_masks(*args)
    with pytest.raises(ValueError, match="masks must be"):
        tree.tree_masks(pos, b.cu, b.kv_len, 2, masks=pos)
    x = torch.zeros(3, 10)
    with pytest.raises(ValueError, match="same GPU"):
        tree.accept_tree(x, pos, pos, b.cu, 2)
    for args, msg in (((x.half(), pos, pos, b.cu, 2), "target"), ((x, pos[:2], pos, b.cu, 2), "tokens"), ((x, pos, pos.long(), b.cu, 2), "parents"),
                      ((x, pos, pos, b.cu, 0), "1 to 64"), ((x[:, :0], pos, pos, b.cu, 2), "target"), ((x.t(), pos, pos, b.cu, 2), "target")):
        with pytest.raises(ValueError, match=msg):
            tree.accept_tree(*args)
    with pytest.raises(ValueError, match="out must be"):
        tree.accept_tree(x, pos, pos, b.cu, 2, out=took[:, :6].contiguous())
    ids = torch.zeros(1, dtype=torch.int32)
    for kw, msg in ((dict(scales=sc.float()), "scales must be"), (dict(scales=sc[:, :3]), "scales must be"),
                    (dict(k=k.bfloat16(), v=v.bfloat16(), scales=sc), "of a byte")):
        with pytest.raises(ValueError, match=msg):
            kv_pages.move_pages(**{**dict(k=k, v=v, src=ids, dst=ids), **kw})


def test_the_words_and_the_round_of_the_oracle():
    """The tests' own masks and walk on a tree worked out by hand."""
    assert masks_of([-1, 0, 0, 1, 2, 3]) == [1, 0b11, 0b101, 0b1011, 0b10101, 0b101011]
    target = torch.full((6, 4), -1.0)
    for i, t in enumerate([2, 1, 3, 0, 0, 1]):
        target[i, t] = 1.0
    tokens = torch.tensor([9, 2, 2, 1, 3, 0], dtype=torch.int32)   # rows 1 and 2 both hold the root's choice: the first is taken
    got = accept64(target, tokens, torch.tensor([-1, 0, 0, 1, 2, 3]), [0, 6], 6)[0].tolist()
    assert got == [3, 4, 0, 0, 2, 1, 0, 1, -1, -1, 0, 1, 3, 5, -1, -1]
    res = TreeResult.from_out(got)
    assert (res.n_accept, res.n_emit, res.flags, res.tokens, res.path) == (3, 4, 0, [2, 1, 0, 1], [0, 1, 3, 5])
    p = random_parents(64, 1)
    assert all(0 <= q < i for i, q in enumerate(p) if i)


class HostPages8(HostPages):
    def _move(self, src, dst, table=None):
        super()._move(src, dst, table)
        self.scales[:, dst] = self.scales[:, src].clone()


def test_pages_in_8_bits():
    kv = HostPages8(2, 6, 1, 64, 16, max_seqs=3, max_tokens=96, dtype=E4M3, device="cpu")
    assert kv.k.dtype == E4M3 and tuple(kv.scales.shape) == (2, 6, 1, 2, 16) and kv.of_layer(1)["scales"].data_ptr() == kv.scales[1].data_ptr()
    kv.k, kv.v = kv.k.view(torch.uint8), kv.v.view(torch.uint8)      # the stand-in moves by indexing
    s = kv.new()
    kv.extend(s, 20)
    for w, p in enumerate(kv.pages_of(s)):
        kv.scales[:, p] = 100 + w
    child = kv.fork(s)
    assert [int(kv.scales[1, p, 0, 1, 3]) for p in kv.pages_of(child)] == [100, 101] and kv.pages_of(child)[1] != kv.pages_of(s)[1]
    kv.free(s)
    check(kv)
    kv.compact()
    kv.resize(3)
    assert tuple(kv.scales.shape) == (2, 3, 1, 2, 16)
    assert [int(kv.scales[0, p, 0, 0, 0]) for p in kv.pages_of(child)] == [100, 101]
    assert KVPages(1, 2, 1, 64, 16, device="cpu").scales is None and KVPages(1, 2, 1, 64, 16, device="cpu").of_layer(0) == {}
    with pytest.raises(ValueError, match="e4m3"):
        KVPages(1, 2, 1, 64, 16, dtype=torch.float8_e5m2, device="cpu")


def test_keep_rows_bounds_its_parts(L):  # noqa: F811
    """A thread's part is counted in 31 bits: more layers and key heads than that are refused."""
    for layers, heads, page, seqs in ((1 << 22, 2, 16, 2), (1 << 21, 4, 16, 1), (1 << 20, 4, 16, 1 << 10)):
        assert L.ssmoe_keep_rows(M, 1 << 50, None, layers, 1, heads, page, 64, 2, 3, 4, 5, 8, 6, 16, seqs, 8, None) == EINVAL
        assert b"too many" in L.ssmoe_last_error(), L.ssmoe_last_error()

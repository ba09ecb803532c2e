"""The paged cache's entry points without a GPU: argument refusals of the C ABI before a device is touched, workspace
sizes, the Python mirrors' ValueErrors, and the definition the GPU tests compare with against torch's own softmax."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels import kv_pages, paged_attention as pa, rope
from tests.paged_util import Batch, attention64, rope64

EINVAL = 1
P = 4096  # aligned dummy address; never dereferenced where a call is refused


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libssmoe.so not built (python -m slotstream_spark_amd.build)")
    return _lib.lib()


def attn(**kw):
    a = dict(q=P, q_row=512, q_head=64, k_pages=P, v_pages=P, cu_rows=P, kv_len=P, table=P, out=P, lse=None, ws=P,
             ws_bytes=1 << 40, n_pages=10, rows=4, seqs=2, max_rows=2, heads=8, kv_heads=2, dim=64, page=16, width=8, window=0,
             sinks=0, type=0, scale=0.125)
    a.update(kw)
    return pa.pack_args(**{k: 0 if v is None else v for k, v in a.items()})


@pytest.mark.parametrize("kw,msg", [
    (dict(dim=96), b"dim must be"), (dict(page=48), b"page must be"), (dict(page=8), b"page must be"),
    (dict(heads=7), b"multiple of kv_heads"), (dict(kv_heads=0), b"multiple of kv_heads"), (dict(heads=0), b"multiple of"),
    (dict(max_rows=0), b"max_rows >= 1"), (dict(rows=-1), b"rows >= 0"), (dict(seqs=-1), b"seqs >= 0"),
    (dict(width=0), b"table row"), (dict(width=1 << 27), b"table row"), (dict(n_pages=0), b"n_pages"),
    (dict(n_pages=1 << 31), b"n_pages"), (dict(type=2), b"type must be"), (dict(window=-1), b"window and sinks"),
    (dict(heads=65536, kv_heads=32768, dim=256, page=128, width=1), b"below 2 GiB"),
    (dict(sinks=-1), b"window and sinks"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"),
    (dict(scale=math.nan), b"scale"), (dict(scale=math.inf), b"scale"), (dict(q=None), b"non-null"),
    (dict(k_pages=None), b"non-null"), (dict(out=None), b"non-null"), (dict(table=None), b"non-null"),
    (dict(q=P + 8), b"16-byte"), (dict(out=P + 2), b"16-byte"), (dict(q_row=514), b"strides"), (dict(q_head=-8), b"strides"),
    (dict(width=4096, ws_bytes=8), b"workspace holds"), (dict(width=4096, ws=None), b"workspace holds"),
    (dict(width=4096, ws=P + 16), b"workspace holds"),
])
def test_attention_refuses(L, kw, msg):
    assert L.ssmoe_paged_attention(attn(**kw), None) == EINVAL
    assert msg in L.ssmoe_last_error(), L.ssmoe_last_error()


def test_chunks_do_not_go_by_the_rows_of_a_call(L):
    """The workspace is slots x rows x heads: with `rows` fixed its size says how a sequence is cut into chunks, which must be the
    same for every max_rows that decoding and verification use (a row's bits go by it)."""
    for window in range(0, 4096, 37):
        for kv_heads, seqs in ((1, 3), (2, 32), (4, 11)):
            sizes = {L.ssmoe_paged_attention_workspace_bytes(attn(
                rows=64, max_rows=m, kv_heads=kv_heads, seqs=seqs, page=64, width=700, window=window, sinks=5))
                for m in range(1, 9)}
            assert len(sizes) == 1, (window, kv_heads, seqs, sizes)


def test_attention_workspace(L):
    size = lambda **kw: L.ssmoe_paged_attention_workspace_bytes(attn(**kw))
    assert size(width=8) == 0                      # a table of one chunk: nothing to join
    assert size(width=4096) > 0 and size(dim=100) == -1 and L.ssmoe_paged_attention_workspace_bytes(None) == -1
    assert size(width=4096, window=64) < size(width=4096)
    assert L.ssmoe_paged_attention(None, None) == EINVAL
    assert L.ssmoe_paged_attention(attn(rows=0, q=None), None) == 0      # nothing to do, no launch
    assert L.ssmoe_paged_attention(attn(seqs=0, q=None), None) == 0


def rope_args(**kw):
    a = dict(q=P, k=P, v=P, q_row=512, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, q_out=P, positions=P,
             pos_stride=4, inv_freq=P, axis=None, k_pages=P, v_pages=P, cu_rows=P, kv_len=P, table=P, n_pages=10, rows=4,
             seqs=2, max_rows=2, heads=8, kv_heads=2, dim=64, page=16, width=8, rot=64, axes=1, adjacent=0, type=0, factor=1.0)
    a.update(kw)
    return rope.pack_args(**{k: 0 if v is None else v for k, v in a.items()})


@pytest.mark.parametrize("kw,msg", [
    (dict(rot=24), b"rot must be"), (dict(rot=80), b"rot must be"), (dict(rot=0), b"rot must be"), (dict(axes=0), b"axes"),
    (dict(factor=math.inf), b"factor"), (dict(dim=32), b"dim must be"), (dict(page=17), b"page must be"),
    (dict(q=None), b"non-null"), (dict(inv_freq=None), b"non-null"), (dict(v_pages=None), b"non-null"),
    (dict(k=P + 8), b"16-byte"), (dict(v_row=129), b"strides"), (dict(inv_freq=P + 4), b"8-byte"), (dict(heads=3), b"multiple"),
])
def test_rope_refuses(L, kw, msg):
    assert L.ssmoe_rope_append(rope_args(**kw), None) == EINVAL
    assert msg in L.ssmoe_last_error(), L.ssmoe_last_error()


def test_outputs_over_inputs_are_refused(L):
    """4 rows of 8 heads of 64, packed rows of 512 elements from P on (what is accepted is run on the GPU)."""
    q, far = dict(q=P, q_row=512, q_head=64, rows=4), 1 << 24
    for out in (P, P + 16, P + 4 * 1024 - 16, P - 4 * 1024 + 16):
        assert L.ssmoe_paged_attention(attn(**q, out=out), None) == EINVAL
        assert b"out must not overlap q" in L.ssmoe_last_error(), out
    for kw in (dict(q_out=P + 16), dict(q_out=P, q_row=1024), dict(q_out=far), dict(q_out=2 * far + 16),
               dict(q_out=far - 4 * 1024 + 16), dict(q_out=P, k=P + 1024)):
        assert L.ssmoe_rope_append(rope_args(**{**q, "k": far, "v": 2 * far, **kw}), None) == EINVAL
        assert b"q_out must be q itself" in L.ssmoe_last_error(), kw


def test_rope_nothing_to_do(L):
    assert L.ssmoe_rope_append(None, None) == EINVAL
    assert L.ssmoe_rope_append(rope_args(rows=0, q=None), None) == 0


def test_move_refuses(L):
    def move(k=P, v=P, layers=2, n_pages=10, page_bytes=2048, src=P, dst=P, n=3, table=None, entries=0):
        return L.ssmoe_move_pages(k, v, layers, n_pages, page_bytes, src, dst, n, table, entries, None)
    assert move(page_bytes=2047) == EINVAL and b"page_bytes" in L.ssmoe_last_error()
    assert move(page_bytes=0) == EINVAL and move(layers=0) == EINVAL and move(n_pages=0) == EINVAL
    assert move(n=-1) == EINVAL and move(entries=-1) == EINVAL and move(entries=1 << 31) == EINVAL
    assert move(k=None) == EINVAL and b"non-null" in L.ssmoe_last_error()
    assert move(src=None) == EINVAL and move(k=P + 8) == EINVAL
    assert move(layers=1 << 20, n=1 << 20) == EINVAL and b"too many" in L.ssmoe_last_error()
    assert move(n=0, k=None) == 0


def test_python_refusals():
    b = Batch([1, 2], [10, 20], 4, 2, 64, 16)
    good = dict(zip(("q", "k_pages", "v_pages", "cu_rows", "kv_len", "table", "max_rows"), b.args("cpu")))
    with pytest.raises(ValueError, match="same GPU"):
        pa.paged_attention(**good)
    for kw, msg in ((dict(q=b.q.float()), "like the cache"), (dict(q=b.q[:, :3]), "multiple"), (dict(q=b.q[0]), "q must be"),
                    (dict(q=b.q[..., :32]), "q must be"), (dict(v_pages=b.v.transpose(2, 3).contiguous()), "v_pages must be"),
                    (dict(k_pages=b.k.float(), v_pages=b.v.float()), "bf16 or fp16"), (dict(k_pages=b.k[:, :1]), "v_pages must"),
                    (dict(k_pages=b.k[:, :, :12], v_pages=b.v[..., :12]), "pages hold"),
                    (dict(k_pages=b.k[:, :1], v_pages=b.v[:, :1]), "contiguous"), (dict(cu_rows=b.cu.long()), "int32"),
                    (dict(cu_rows=b.cu[:2]), "cu_rows must be"), (dict(kv_len=b.kv_len[:1]), "kv_len"),
                    (dict(table=b.table[0]), "table must be"), (dict(max_rows=0), "max_rows"),
                    (dict(q=torch.zeros(3, 4, 65, dtype=b.dtype)[:, :, 1:]), "multiples of 8"),
                    (dict(q=torch.zeros(3, 4, 100, dtype=b.dtype)[:, :, :64]), "multiples of 8")):
        with pytest.raises(ValueError, match=msg):
            pa.paged_attention(**{**good, **kw})
    qkv = torch.zeros(3, 8, 64, dtype=b.dtype)
    args = dict(q=qkv[:, :4], k=qkv[:, 4:6], v=qkv[:, 6:], positions=torch.zeros(3, dtype=torch.int32),
                inv_freq=torch.ones(32, dtype=torch.float64), **{k: v for k, v in good.items() if k != "q"})
    with pytest.raises(ValueError, match="same GPU"):
        rope.rope_append(**args)
    for kw, msg in ((dict(inv_freq=torch.ones(32)), "fp64"), (dict(inv_freq=torch.ones(5, dtype=torch.float64)), "rot must be"),
                    (dict(inv_freq=torch.ones(40, dtype=torch.float64)), "rot must be"), (dict(k=qkv[:, :3]), "k must be"),
                    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must"), (dict(v=qkv[:2, 6:]), "same rows"),
                    (dict(positions=torch.zeros(3)), "positions must"), (dict(axis=torch.zeros(32)), "axis must"),
                    (dict(out=torch.zeros(3, 4, 64)), "same GPU|out must")):
        with pytest.raises(ValueError, match=msg):
            rope.rope_append(**{**args, **kw})
    k, v, one = b.k[None].contiguous(), b.v[None].contiguous(), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="same GPU"):
        kv_pages.move_pages(k, v, one, one)
    for a, msg in (((k, v[:, :1], one, one), "one type and size"), ((k, v, one.long(), one), "src must"),
                   ((k, v, one, one[:0]), "same length"), ((k[..., :8].contiguous(), v[..., :2, :].contiguous(), one, one), "one type|2048"),
                   ((k, v, one, one, one.float()), "table must"), ((b.k[:, :, 0].contiguous(), b.v[..., 0].contiguous(), one, one), "2048")):
        with pytest.raises(ValueError, match=msg):
            kv_pages.move_pages(*a)


def test_a_checked_shape_does_not_let_other_strides_pass():
    """What the checks found is kept by shapes, types and strides: a strided tensor of a known shape is still refused."""
    k, v = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(8, 2, 64, 16, dtype=torch.bfloat16)
    q, x = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(cu_rows=i32(4), kv_len=i32(3), table=i32(3, 2))
    f, pos, axis = torch.ones(16, dtype=torch.float64), i32(3), i32(16)
    for _ in range(2):
        with pytest.raises(ValueError, match="same GPU"):
            pa.paged_attention(q, k, v, **good, max_rows=1)
        with pytest.raises(ValueError, match="same GPU"):
            rope.rope_append(q, x, x, pos, f, k, v, **good, max_rows=1, axis=axis)
    for name, bad in (("cu_rows", i32(8)[::2]), ("kv_len", i32(6)[::2]), ("table", i32(3, 4)[:, ::2])):
        with pytest.raises(ValueError, match=f"{name} must be a contiguous"):
            pa.paged_attention(q, k, v, **{**good, name: bad}, max_rows=1)
        with pytest.raises(ValueError, match=f"{name} must be a contiguous"):
            rope.rope_append(q, x, x, pos, f, k, v, **{**good, name: bad}, max_rows=1, axis=axis)
    with pytest.raises(ValueError, match="axis must be"):
        rope.rope_append(q, x, x, pos, f, k, v, **good, max_rows=1, axis=i32(32)[::2])
    with pytest.raises(ValueError, match="positions must be"):
        rope.rope_append(q, x, x, i32(6)[::2], f, k, v, **good, max_rows=1, axis=axis)
    with pytest.raises(ValueError, match="inv_freq must be"):
        rope.rope_append(q, x, x, pos, torch.ones(32, dtype=torch.float64)[::2], k, v, **good, max_rows=1, axis=axis)


@pytest.mark.parametrize("kw", [dict(max_rows=1 << 31), dict(window=1 << 31), dict(sinks=1 << 40), dict(window=-1),
                                dict(scale=1e39), dict(scale=0.0), dict(scale=math.nan)])
def test_numbers_that_do_not_fit_are_refused(kw):
    k, v = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(8, 2, 64, 16, dtype=torch.bfloat16)
    q, i32 = torch.zeros(3, 4, 64, dtype=torch.bfloat16), lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError, match="max_rows|window|scale"):
        pa.paged_attention(q, k, v, i32(4), i32(3), i32(3, 2), **{"max_rows": 1, **kw})
    with pytest.raises(ValueError, match="factor"):
        rope.rope_append(q, q[:, :2], q[:, :2], i32(3), torch.ones(16, dtype=torch.float64), k, v, i32(4), i32(3), i32(3, 2), 1,
                         factor=1e39)


def test_definition_against_torch():
    """attention64 on whole causal sequences is torch's softmax attention, rope64 a rotation of complex numbers."""
    b = Batch([20, 7], [20, 7], 4, 2, 64, 16)
    out, lse = attention64(b, window=5, sinks=2)
    r = 0
    for s, n in enumerate(b.rows):
        ids = b.table[s].long()
        k = b.k[ids.clamp(min=0)].transpose(1, 2).reshape(-1, 2, 64)[:n].double().repeat_interleave(2, 1)
        v = b.v[ids.clamp(min=0)].permute(0, 3, 1, 2).reshape(-1, 2, 64)[:n].double().repeat_interleave(2, 1)
        x = torch.einsum("ihd,jhd->hij", b.q[r:r + n].double(), k) / 8
        i, j = torch.arange(n)[:, None], torch.arange(n)
        x = x.masked_fill(~((j <= i) & ((i - j < 5) | (j < 2))), -math.inf)
        assert torch.allclose(out[r:r + n], torch.einsum("hij,jhd->ihd", x.softmax(-1), v), atol=1e-12)
        assert torch.allclose(lse[r:r + n], x.logsumexp(-1).t(), atol=1e-12)
        r += n
    x = torch.randn(5, 3, 64, dtype=torch.float64)
    pos, f = torch.arange(5)[None], torch.rand(32, dtype=torch.float64)
    z = torch.complex(x[..., :32], x[..., 32:]) * torch.polar(torch.ones(5, 32, dtype=torch.float64), pos.t() * f)[:, None]
    assert torch.allclose(rope64(x, pos, f), torch.cat([z.real, z.imag], -1), atol=1e-12)
    z = torch.complex(x[..., ::2], x[..., 1::2]) * torch.polar(torch.ones(5, 32, dtype=torch.float64), pos.t() * f)[:, None]
    assert torch.allclose(rope64(x, pos, f, adjacent=True), torch.view_as_real(z).flatten(-2), atol=1e-12)

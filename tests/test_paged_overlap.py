"""Outputs that share memory with each other or with an input are refused by the entry points of the paged cache before a device is
touched (addresses are dummies; what lies apart is run on the GPU by every other test)."""
import pytest

from slotstream_spark_amd import _lib
from tests.test_paged_host import EINVAL, L, attn, rope_args  # noqa: F401  (L is a fixture)

M = 1 << 24   # apart: nothing here is larger


def layout(names):
    return {n: (i + 1) * M for i, n in enumerate(names)}


# 4 rows of 8 heads of 64 (packed), 2 key heads, 10 pages of 16 tokens (40,960 bytes of keys), 2 sequences, table of 8
ATTN = layout(["q", "k_pages", "v_pages", "cu_rows", "kv_len", "table", "out", "lse", "ws"])
SIZES = dict(q=4096, out=4096, lse=128, k_pages=40960, v_pages=40960, cu_rows=12, kv_len=8, table=64, k=1024, v=1024, q_out=4096,
             positions=16, inv_freq=256, axis=128)


@pytest.mark.parametrize("written,other", [
    ("lse", "q"), ("lse", "out"), ("lse", "k_pages"), ("lse", "v_pages"), ("out", "k_pages"), ("out", "v_pages"), ("out", "table"),
    ("out", "cu_rows"), ("out", "kv_len"), ("lse", "table"), ("out", "q")])
def test_attention(L, written, other):  # noqa: F811
    near = ATTN[other] + SIZES[other] - 16 if SIZES[other] > 16 else ATTN[other]
    for at in (ATTN[other], near, ATTN[other] - SIZES[written] + 16):
        assert L.ssmoe_paged_attention(attn(**{**ATTN, written: at}), None) == EINVAL, at
        assert b"overlap" in L.ssmoe_last_error(), L.ssmoe_last_error()


def test_attention_workspace(L):  # noqa: F811
    """A call in several chunks: 4096 pages wide, so its table has 32,768 bytes."""
    big = dict(ATTN, width=4096, ws_bytes=M)
    for other in ("q", "k_pages", "v_pages", "out", "lse", "table"):
        assert L.ssmoe_paged_attention(attn(**{**big, "ws": ATTN[other]}), None) == EINVAL
        assert b"overlap" in L.ssmoe_last_error(), other


ROPE = layout(["q", "k", "v", "positions", "inv_freq", "axis", "k_pages", "v_pages", "cu_rows", "kv_len", "table", "q_out"])


@pytest.mark.parametrize("written,other", [
    ("q_out", "k_pages"), ("q_out", "v_pages"), ("k_pages", "v_pages"), ("k_pages", "q"), ("k_pages", "k"), ("v_pages", "v"),
    ("v_pages", "table"), ("q_out", "positions"), ("q_out", "inv_freq"), ("q_out", "axis"), ("q_out", "cu_rows"),
    ("k_pages", "kv_len")])
def test_rope(L, written, other):  # noqa: F811
    rows = dict(q_row=512, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64)
    near = ROPE[other] + SIZES[other] - 16 if SIZES[other] > 16 else ROPE[other]
    for at in (ROPE[other], near, ROPE[other] - SIZES[written] + 16):
        assert L.ssmoe_rope_append(rope_args(**{**ROPE, **rows, written: at}), None) == EINVAL, at
        assert b"overlap" in L.ssmoe_last_error(), L.ssmoe_last_error()


def test_move(L):  # noqa: F811
    """2 layers of 10 pages of 2,048 bytes, 3 moves, a table of 100 entries."""
    at = layout(["k", "v", "src", "dst", "table"])

    def move(**kw):
        a = {**at, **kw}
        return L.ssmoe_move_pages(a["k"], a["v"], 2, 10, 2048, a["src"], a["dst"], 3, a["table"], 100, None)
    for kw in (dict(v=at["k"]), dict(v=at["k"] + 40960 - 16), dict(v=at["k"] - 40960 + 16), dict(table=at["k"] + 4096),
               dict(src=at["v"] + 64), dict(dst=at["k"]), dict(table=at["src"]), dict(table=at["dst"] - 396)):
        assert move(**kw) == EINVAL and b"overlap" in L.ssmoe_last_error(), kw

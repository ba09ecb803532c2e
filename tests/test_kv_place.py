"""A sequence that goes back and writes again (engine/attention.SeqCache over memory/kv_pages.KVPages), on the CPU: what a refused
call leaves, which pages serve it, and how often the table goes to the device."""
import numpy as np
import pytest

from slotstream_spark_amd import _lib
from tests.test_kv_pages import check, pages, read, write


@pytest.mark.parametrize("n_pages", [4, 5, 8])
def test_a_refused_place_changes_nothing(n_pages):
    """A sequence of 40 tokens goes back to token 20 and asks for more than there is: it keeps what it had."""
    from slotstream_spark_amd.engine.attention import SeqCache
    kv = pages(n=n_pages, page=16)
    cache, other = SeqCache(kv), kv.new()
    kv.extend(other, 16)
    cache.place(0, 40)
    write(kv, cache.seq, 0, range(1, 41))
    before = kv._table.copy(), kv._refs.copy(), sorted(kv._free), list(kv.length)
    for pos, n in ((20, 110), (0, 150), (40, 200)):
        with pytest.raises(_lib.Exhausted if pos + n <= 200 else ValueError):
            cache.place(pos, n)
        check(kv)
        assert np.array_equal(before[0], kv._table) and np.array_equal(before[1], kv._refs)
        assert before[2:] == (sorted(kv._free), list(kv.length)) and read(kv, cache.seq) == list(range(1, 41))


def test_pages_given_up_serve_the_same_call():
    """No page is free: a copy of a shared page takes the place of one that the call gives up."""
    from slotstream_spark_amd.engine.attention import SeqCache
    kv = pages(n=3, page=16)
    cache = SeqCache(kv)
    cache.place(0, 16)
    write(kv, cache.seq, 0, range(1, 17))
    child = kv.fork(cache.seq)
    cache.place(16, 32)
    assert kv.free_pages == 0
    cache.place(10, 3)
    write(kv, cache.seq, 10, [50, 51, 52])
    check(kv)
    assert read(kv, child) == list(range(1, 17)) and read(kv, cache.seq) == list(range(1, 11)) + [50, 51, 52]
    assert kv.free_pages == 1


def test_rounds_over_a_page_border_keep_their_pages():
    """Verify rounds of three rows whose first row moves on by one: the table is published once a page."""
    from slotstream_spark_amd.engine.attention import SeqCache
    kv, published = pages(n=12, page=16), []
    publish = kv._publish
    kv._publish = lambda seq: (published.append(seq), publish(seq))
    cache = SeqCache(kv)
    for pos in range(0, 100):
        cache.place(pos, 3)
        check(kv)
        assert kv.length[cache.seq] == pos + 3
    assert len(published) == -(-102 // 16)


def test_the_batch_tensors_of_all_row_counts_share_one_memory():
    """A long-lived sequence meets every prompt length: what it holds on the device does not grow, the tensors of one row count stay
    in place, and each says its own count."""
    from slotstream_spark_amd.engine.attention import SeqCache
    kv = pages(n=13, page=16, tokens=200)
    cache, places, held = SeqCache(kv), {}, set()
    for _ in range(2):
        for n in range(1, 201):
            cache.place(0, n)
            cu, kv_len, table, positions = cache.rows(n)
            assert cu.tolist() == [0, n] and kv_len.tolist() == [n] and positions.tolist() == list(range(n))
            at = [t.data_ptr() for t in (cu, kv_len, table, positions)]
            assert places.setdefault(n, at) == at and all(t.is_contiguous() for t in (cu, positions))
            held |= {t.untyped_storage().data_ptr() for t in (cu, positions)}
            cache.reset()
    assert len(held) <= 2
    cache.place(0, 7)
    cache.place(7, 3)
    assert cache.rows(3)[3].tolist() == [7, 8, 9] and cache.rows(5)[0].tolist() == [0, 5] and cache.rows(0)[0].tolist() == [0, 0]
    with pytest.raises(ValueError, match="exceed"):
        cache.rows(kv.width * kv.page + 1)

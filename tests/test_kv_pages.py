"""Who holds which page (memory/kv_pages.KVPages), on the CPU: random sequences of calls against a plain model that keeps every
token's content, copy on write, eviction, compaction, shrinking, and that a refused call changes nothing. Page moves are done
by indexing here; the launch is tested on the GPU."""
import random

import numpy as np
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.memory.kv_pages import KVPages


class HostPages(KVPages):
    def _move(self, src, dst, table=None):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.k[:, dst], self.v[:, dst] = self.k[:, src].clone(), self.v[:, src].clone()
        if table is not None:
            to = {s: d for s, d in zip(src, dst)}
            table.copy_(torch.tensor([[to.get(p, p) for p in row] for row in table.tolist()], dtype=torch.int32))


def pages(n=12, page=16, seqs=5, tokens=200, layers=2):
    return HostPages(layers, n, 1, 64, page, max_seqs=seqs, max_tokens=tokens, device="cpu")


def write(kv, seq, at, values):
    """Token at + i of the sequence := values[i] in every layer, through the table, as rope_append writes."""
    for i, x in enumerate(values):
        p = int(kv.table[seq, (at + i) // kv.page])
        assert p >= 0
        kv.k[:, p, :, (at + i) % kv.page] = x
        kv.v[:, p, :, :, (at + i) % kv.page] = x


def read(kv, seq):
    out = []
    for t in range(kv.length[seq]):
        p = int(kv.table[seq, t // kv.page])
        out.append(None if p < 0 else int(kv.k[1, p, 0, t % kv.page, 3]))
        if p >= 0:
            assert int(kv.v[0, p, 0, 5, t % kv.page]) == out[-1]
    return out


def check(kv):
    held = kv._table[kv._table >= 0]
    assert np.array_equal(np.bincount(held, minlength=kv.n_pages), kv._refs)
    assert sorted(kv._free) == np.flatnonzero(kv._refs == 0).tolist()
    assert np.array_equal(kv.table.numpy(), kv._table)


@pytest.mark.parametrize("seed", range(12))
def test_against_a_plain_model(seed):
    rng, model, count = random.Random(seed), {}, 0
    kv = pages(n=rng.choice([6, 12, 30]), page=rng.choice([16, 32]))
    for _ in range(150):
        do = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact", "resize", "rewrite"])
        before = (kv._table.copy(), kv._refs.copy(), sorted(kv._free), list(kv.length), kv.n_pages)
        try:
            if do == "new":
                model[kv.new()] = []
            elif do == "compact":
                n = kv.compact()
                assert n == int((kv._refs > 0).sum()) and (kv._refs[:n] > 0).all()
            elif do == "resize":
                kv.resize(rng.choice([6, 12, 30]))
            elif model:
                s = rng.choice(sorted(model))
                if do == "extend":
                    n, at = rng.choice([0, 1, 1, 3, 17, 40]), kv.length[s]
                    kv.extend(s, n)
                    values = [(count + i) % 120 for i in range(n)]
                    count += n
                    write(kv, s, at, values)
                    model[s] = model[s] + values
                elif do == "fork":
                    model[kv.fork(s)] = list(model[s])
                elif do == "truncate":
                    n = rng.randint(0, len(model[s]))
                    kv.truncate(s, n)
                    model[s] = model[s][:n]
                elif do == "free":
                    kv.free(s)
                    del model[s]
                elif do == "rewrite" and model[s]:   # a round that is taken back and written anew, over shared pages too
                    n = rng.randint(0, min(5, len(model[s]) - 1))
                    kv.truncate(s, len(model[s]) - n)
                    kv.extend(s, n)
                    write(kv, s, len(model[s]) - n, [7] * n)
                    model[s] = model[s][:len(model[s]) - n] + [7] * n
        except (_lib.Exhausted, ValueError):
            if do != "rewrite":
                assert np.array_equal(before[0], kv._table) and np.array_equal(before[1], kv._refs)
                assert before[2:] == (sorted(kv._free), list(kv.length), kv.n_pages)
            else:
                model[s] = model[s][:kv.length[s]]
        check(kv)
        for s, want in model.items():
            assert kv.length[s] == len(want) and read(kv, s) == want


def test_fork_shares_full_pages_and_copies_the_open_one():
    kv = pages()
    a = kv.new()
    kv.extend(a, 40)
    write(kv, a, 0, list(range(40)))
    b = kv.fork(a)
    assert kv.pages_of(a)[:2] == kv.pages_of(b)[:2] and kv.pages_of(a)[2] != kv.pages_of(b)[2]
    kv.extend(b, 1)
    write(kv, b, 40, [99])
    assert read(kv, a) == list(range(40)) and read(kv, b) == list(range(40)) + [99]
    kv.truncate(b, 20)                       # into a shared page: the next write copies it
    kv.extend(b, 1)
    write(kv, b, 20, [77])
    assert read(kv, a) == list(range(40)) and read(kv, b) == list(range(20)) + [77]
    c = kv.fork(a)
    kv.free(a)
    assert read(kv, c) == list(range(40))


def test_evict_keeps_the_window_and_the_first_tokens():
    kv = pages()
    s = kv.new()
    kv.extend(s, 100)
    write(kv, s, 0, list(range(100)))
    assert kv.evict(s, 30, 4, back=8) == 2   # rows from 92 on see 63 ..: pages 1 and 2 go, page 0 holds the first tokens
    got = read(kv, s)
    assert got[:16] == list(range(16)) and got[16:48] == [None] * 32 and got[48:] == list(range(48, 100))
    assert kv.evict(s, 30, 4, back=8) == 0
    kv.extend(s, 30)
    assert kv.evict(s, 30, 0, back=0) == 4   # rows from 130 on see 101 ..: pages 0, 3, 4 and 5
    check(kv)
    b = kv.fork(s)
    assert kv.pages_of(b)[:6] == [-1] * 6
    kv.free(s)
    kv.compact()
    check(kv)
    kv.truncate(b, 90)
    with pytest.raises(ValueError, match="evicted"):
        kv.extend(b, 1)


@pytest.mark.parametrize("pos", [0, 5, 16, 20, 31, 32, 33, 39])
def test_rows_written_again_leave_a_fork_alone(pos):
    """A sequence of 40 tokens is forked, then goes back to `pos` (a rejected draft) and writes from there: the fork keeps every token."""
    from slotstream_spark_amd.engine.attention import SeqCache
    kv = pages()
    cache = SeqCache(kv)
    cache.place(0, 40)
    write(kv, cache.seq, 0, range(1, 41))
    child = kv.fork(cache.seq)
    cache.place(pos, 4)
    assert cache.rows(4)[1].tolist() == [pos + 4] and cache.rows(4)[3].tolist() == list(range(pos, pos + 4))
    write(kv, cache.seq, pos, range(101, 105))
    assert read(kv, child) == list(range(1, 41))
    assert read(kv, cache.seq) == list(range(1, pos + 1)) + list(range(101, 105))


def test_refusals():
    kv = pages(n=3)
    s = kv.new()
    with pytest.raises(_lib.Exhausted):
        kv.extend(s, 60)
    assert kv.length[s] == 0 and kv.free_pages == 3
    with pytest.raises(ValueError, match="exceed"):
        kv.extend(s, 1000)
    with pytest.raises(ValueError, match="truncate"):
        kv.extend(s, -1)
    with pytest.raises(ValueError, match="no sequence"):
        kv.extend(3, 1)
    with pytest.raises(ValueError, match="cannot keep"):
        kv.truncate(s, 1)
    kv.extend(s, 40)
    with pytest.raises(_lib.Exhausted):
        kv.fork(s)                           # the open page has no place
    check(kv)
    with pytest.raises(_lib.Exhausted):
        kv.resize(2)
    for bad in (dict(n=0), dict(page=8), dict(seqs=0), dict(tokens=0)):
        with pytest.raises(ValueError):
            pages(**bad)
    kv.free(s)
    with pytest.raises(ValueError, match="no sequence"):
        kv.free(s)
    assert kv.free_pages == 3

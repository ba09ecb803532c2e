"""Forks of the draft head's state over its one cache, on the CPU: the head's calls with its matrix products left out and an
attention that writes the rows' tokens into the pages and reads back all that a row would see. What a call does not refuse
it must run over exactly the tokens that its state was fed."""
import random

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine import mtp
from slotstream_spark_amd.engine.attention import SeqCache
from tests.test_kv_pages import pages

H = 64


class Layer:
    """Rows are tokens: x[i, 0]."""

    def append(self, x, positions, k, v, cu, kv_len, table, n):
        assert cu.tolist() == [0, n] and int(kv_len) == int(positions[0]) + n
        for i, p in enumerate(positions.tolist()):
            k[int(table[0, p // 16]), :, p % 16] = x[i, 0]
        self.seen = [int(k[int(table[0, p // 16]), 0, p % 16, 0]) for p in range(int(kv_len))]

    def __call__(self, x, *args):
        self.append(x, *args)
        return x


class Weights:
    down = up = torch.zeros(1, H)


class Attn:
    def __init__(self, kv):
        self.pages, self.layer, self.hc = kv, Layer(), Weights()


class Head(mtp.MTPHead):
    def __init__(self, kv, max_ctx=100):
        self.attn, self.cache = Attn(kv), SeqCache(kv)
        self.H, self.hc, self.max_rows, self.topk = H, 1, 4, 1
        self.w = type("W", (), {"mlp_hc": Weights, "mixer_hc": Weights, "embed": torch.zeros(1, H)})
        self.state, self.consumed, self.prev_multi, self._draft_rows = mtp.MTPState(max_ctx), 0, None, {}
        if hasattr(mtp, "CacheRows"):
            self.held = mtp.CacheRows()
        self.seen = []

    def fuse(self, embedded, multi, r=None, i=0, idx=None):
        return embedded if idx is None else idx[:, None].expand(1, H).to(torch.bfloat16)

    def hc_mix(self, hcw, hyp, hn, low, mix_w, mixed, inj=None):
        return hyp, inj

    def _step_rows(self, embedded, multi, r, i, idx=None, pos=0, base=None):
        h = self.fuse(embedded, multi, r, i, idx)
        self._attend(h, pos, base)
        self.seen.append(self.attn.layer.seen)
        return h, h

    def argmax(self, o, ids):
        ids.copy_((o[0, 0].to(torch.int32) * 7 + 3) % 100)   # the next draft, a function of the last one

    def feed(self, tokens, state, state_only=False):
        self.seen = []
        x = torch.tensor(tokens, dtype=torch.bfloat16)[:, None].expand(-1, H).contiguous()
        self.step(x, x, state, state_only=state_only)
        return self.attn.layer.seen

    def drafts(self, token, k, state=None):
        self.seen = []
        out = torch.zeros(k, dtype=torch.int32)
        self.draft_async(torch.tensor([token], dtype=torch.int32), torch.zeros(1, H, dtype=torch.bfloat16), k, out, state=state)
        return [token] + out.tolist()[:-1]


@pytest.fixture
def head(monkeypatch):
    monkeypatch.setattr(mtp, "hc_inject", lambda h, y, inj, out=None: h)
    return Head(pages(n=20, seqs=2, tokens=200))


def test_one_fork_after_another(head):
    """A fork is stepped on and on behind the head's rows, then another; the head's own rows stay."""
    own = list(range(1, 21))
    assert head.feed(own, head.state, state_only=True) == own
    a, b = head.state.fork(), head.state.fork()
    assert head.feed([30, 31], a) == own + [30, 31] and head.feed([32], a) == own + [30, 31, 32]
    c = a.fork()
    assert head.feed([33], c) == own + [30, 31, 32, 33]
    assert head.feed([34], a) == own + [30, 31, 32, 34]          # c's row is gone
    with pytest.raises(ValueError, match="no longer holds"):
        head.feed([35], c)
    assert head.feed([40], b) == own + [40]
    with pytest.raises(ValueError, match="no longer holds"):
        head.feed([41], a)
    assert head.drafts(50, 3) == [50, 53, 74] and head.seen == [own + [50], own + [50, 53], own + [50, 53, 74]]
    with pytest.raises(ValueError, match="no longer holds"):
        head.feed([42], b)
    assert head.feed([60], head.state) == own + [60] and head.state.pos == 21


def test_an_older_fork_leaves_the_heads_rows_alone(head):
    """40 rows, a fork of row 5, and the head goes on: nothing that the head counts as its own is given back."""
    head.feed(list(range(5)), head.state, state_only=True)
    old = head.state.fork()
    head.feed(list(range(5, 40)), head.state, state_only=True)
    with pytest.raises(ValueError, match="head's own rows"):
        head.feed([90], old)
    with pytest.raises(ValueError, match="head's own rows"):
        head.drafts(90, 2, state=old)
    with pytest.raises(ValueError, match="head's own rows"):
        head.feed([90], mtp.MTPState(100))
    other = head.cache.pages.new()
    head.cache.pages.extend(other, 32)
    head.cache.pages.k[:, head.cache.pages.pages_of(other)] = 99.0
    assert head.feed([40], head.state) == list(range(41))


def test_forks_from_before_a_reset(head):
    head.feed([1, 2, 3], head.state, state_only=True)
    fork, start = head.state.fork(), mtp.MTPState(100)
    head.reset()
    with pytest.raises(ValueError, match="no longer holds"):
        head.feed([9], fork)
    assert head.feed([8], start) == [8]                           # nothing before it, nothing of the head's behind it
    assert head.feed([4, 5, 6], head.state) == [4, 5, 6]
    with pytest.raises(ValueError):
        head.feed([9], fork)
    with pytest.raises(ValueError):
        head.feed([9], start)


def test_positions_set_by_hand(head):
    head.feed(list(range(10)), head.state, state_only=True)
    head.state.pos = 6                                            # the head goes back
    assert head.feed([70, 71], head.state) == list(range(6)) + [70, 71]
    fork = head.state.fork()
    fork.pos = 9
    with pytest.raises(ValueError, match="no longer holds"):      # rows that nobody wrote
        head.feed([1], fork)


@pytest.mark.parametrize("seed", range(8))
def test_any_order_of_calls(seed, head):
    """Every call that goes through sees its state's own tokens; the head's own state and a fork of it made on the spot are
    never refused."""
    rng, model, count, refused = random.Random(seed), {id(head.state): []}, 0, 0
    states = [head.state]
    for _ in range(120):
        s = rng.choice(states)
        do = rng.choice(["step", "step", "step", "draft", "fork", "reset"] if rng.random() < 0.2 else ["step", "draft", "fork"])
        past = model[id(s)]
        try:
            if do == "fork":
                states.append(s.fork())
                model[id(states[-1])] = list(past)
            elif do == "reset":
                head.reset()
                model[id(head.state)] = []
            elif len(past) > 80:
                continue
            elif do == "draft":
                got = head.drafts(count % 100, 3, state=s)
                assert head.seen == [past + got[:i + 1] for i in range(3)]
                model[id(s)] = past + got
            else:
                new = [(count + i) % 100 for i in range(rng.randint(1, 4))]
                assert head.feed(new, s, state_only=rng.random() < 0.5) == past + new
                model[id(s)] = past + new
            count += 5
        except ValueError:
            refused += 1
            assert s is not head.state
            assert s.pos == len(past)
            fresh = head.state.fork()
            own = model[id(head.state)]
            if len(own) < 90:
                assert head.feed([1], fresh) == own + [1]
        for t in states:
            assert t.pos == len(model[id(t)])
    assert refused


def test_a_step_that_fails_does_not_advance(head):
    """Too few pages, or an attention that refuses its arguments: the state stays where it was, and goes on afterwards."""
    head, own = Head(pages(n=6, seqs=2, tokens=200)), list(range(14))
    head.feed(own, head.state, state_only=True)
    other = head.cache.pages.new()
    head.cache.pages.extend(other, head.cache.pages.free_pages * 16)
    for state_only in (False, True):
        with pytest.raises(_lib.Exhausted):
            head.feed([1] * 3, head.state, state_only)
        assert head.state.pos == 14
    head.cache.pages.free(other)

    def refuse(*args):
        raise ValueError("refused")

    layer, head.attn.layer = head.attn.layer, Layer()
    head.attn.layer.append = refuse
    for state_only in (False, True):
        with pytest.raises(ValueError, match="refused"):
            head.feed([1, 2], head.state, state_only)
        assert head.state.pos == 14
    head.attn.layer = layer
    assert head.feed([1, 2], head.state) == own + [1, 2]


def test_drafts_over_a_page_border_publish_the_table_once(head):
    """15 rows and three drafts, pages of 16 tokens: one page is taken, once, and stays for the next drafts."""
    head.feed(list(range(15)), head.state, state_only=True)
    kv, published = head.cache.pages, []
    publish = kv._publish
    kv._publish = lambda seq: (published.append(seq), publish(seq))
    for _ in range(3):
        head.drafts(50, 3)
    assert len(published) == 1
    assert head.feed([60, 61], head.state) == list(range(15)) + [60, 61] and len(published) == 1

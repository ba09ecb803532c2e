"""MoEStack without a GPU: what it holds after a refusal and how its positions move, with the step graph, the prompt layers and the
lm_head replaced by stand-ins."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine import generate, rollback as rb
from slotstream_spark_amd.engine.step import MoEWeights
from tests.test_kv_pages import pages

H, V = 64, 32


class Graph:
    """Stands for MTPStepGraph: rows pass through."""

    def __init__(self, pool, layers, lm_head, depth, norm_weights=None, eps=1e-6, top_k=10, device="cpu", attn=None,
                 attn_norms=None, cache=None):
        self.nl, self.rows, self.eps = len(layers), depth + 1, eps
        self.norm_weights, self.attn, self.attn_norms = [None] * (self.nl + 1), attn, [None] * self.nl
        self.x_in = torch.zeros(self.rows, H, dtype=torch.bfloat16)
        self.streams, self.mixed = [self.x_in] * (self.nl + 1), [self.x_in] * (self.nl + 1)
        self.drafts = torch.zeros(depth, dtype=torch.int32)

    def step(self):
        return None

    def result(self):
        return None


class Argmax:
    def __init__(self, lm_head, max_rows, round_bf16, device):
        pass

    def __call__(self, x, ids, logits):
        ids.fill_(3)
        logits.zero_()


class Prompt:
    def __init__(self, *args, **kw):
        pass

    def __call__(self, x):
        return (x,)


class Pool:
    hidden = H


class Head:
    n = V


@pytest.fixture
def build(monkeypatch):
    monkeypatch.setattr(generate, "MTPStepGraph", Graph)
    monkeypatch.setattr(generate, "LMHeadArgmax", Argmax)
    monkeypatch.setattr(generate, "MoEPrefillLayer", Prompt)
    monkeypatch.setattr(generate, "gather_rows", lambda src, idx, out=None: src[idx.long()] if out is None else out.copy_(src[idx.long()]))

    def make(kv, **kw):
        w = MoEWeights(*[torch.zeros(4, H, dtype=torch.bfloat16)] * 5)
        return generate.MoEStack(Pool, [w, w], Head, torch.zeros(V, H, dtype=torch.bfloat16), depth=2, device="cpu",
                                 attn=None if kv is None else [None, None], pages=kv, **kw)
    return make


@pytest.mark.parametrize("part", ["MTPStepGraph", "MoEPrefillLayer", "LMHeadArgmax"])
def test_a_refused_stack_keeps_no_sequence(build, monkeypatch, part):
    """Whatever part refuses, the only sequence of the pages is free again."""
    def refuse(*a, **kw):
        raise ValueError("refused")

    kv = pages(seqs=1)
    with monkeypatch.context() as m:
        m.setattr(generate, part, refuse)
        for _ in range(2):
            with pytest.raises(ValueError, match="refused"):
                build(kv, prompt_chunk=16)
    assert build(kv).cache.seq == 0


def test_prompt_layers_refuse_affine_shared_weights():
    """The verify layer takes 4-bit shared weights (AffineWeight), the prompt layer does not: a ValueError says so."""
    from slotstream_spark_amd.engine.prefill import MoEPrefillLayer
    from slotstream_spark_amd.kernels.gemv_affine import AffineWeight

    pool = type("P", (), {"hidden": H, "inter": H, "experts": 4, "device": "cpu"})
    bf = torch.zeros(4, H, dtype=torch.bfloat16)
    q4 = AffineWeight(torch.zeros(4, H // 8, dtype=torch.int32), bf[:, :1], bf[:, :1], 4, 64, 4, H)
    for name in ("router_w", "sh_gate", "sh_up", "sh_down", "sh_g"):
        with pytest.raises(ValueError, match="contiguous bf16"):
            MoEPrefillLayer(pool, 0, **{**dict(router_w=bf, sh_gate=bf, sh_up=bf, sh_down=bf, sh_g=bf), name: q4})


@pytest.mark.parametrize("with_cache", [False, True])
def test_a_refused_round_leaves_no_record_behind(build, with_cache):
    """A verify round whose pass raises is no outstanding round; the next one is."""
    stack = build(pages(n=3, seqs=2) if with_cache else None)
    if with_cache:
        other = stack.cache.pages.new()
        stack.cache.pages.extend(other, 48)
        with pytest.raises(_lib.Exhausted):
            stack.step([1, 2, 3])
        stack.cache.pages.free(other)
    else:
        with pytest.raises(IndexError):
            stack.step([1, 2, V])
    assert stack.record.outstanding == 0 and stack.record.rounds == 0 and stack.st.pos == 0 and stack.st.tokens == []
    ck = rb.checkpoint(stack)
    stack.step([1, 2, 3])
    assert stack.record.outstanding == 1 and stack.record.rounds == 1
    rb.rollback(stack, stack.record, ck, 2, 3)
    assert stack.record.outstanding == 0 and stack.st.tokens == [1, 2]


@pytest.mark.parametrize("prompt_chunk", [0, 16])
def test_the_caches_position_follows_the_stacks(build, monkeypatch, prompt_chunk):
    """SeqCache.pos is the sequence's position after prompts, plain steps, rounds kept whole or in part, and a reset."""
    monkeypatch.setattr(generate, "residual_rmsnorm", lambda *a, **kw: None)
    stack = build(pages(n=12), prompt_chunk=prompt_chunk)
    stack.graph.attn = [lambda x, *args: x] * 2
    same = lambda n: stack.st.pos == stack.cache.pos == stack.st.attn["cache"].pos == len(stack.st.tokens) == n  # noqa: E731
    stack.prompt(list(range(1, 20)))
    assert same(19)
    stack.forward([5])
    assert same(20)
    stack.forward([5, 6, 7, 8])
    assert same(24)
    for keep in (1, 3, 2):
        at, ck = stack.st.pos, rb.checkpoint(stack)
        stack.step([1, 2, 3])
        assert same(at + 3)
        rb.rollback(stack, stack.record, ck, keep, 3)
        assert same(at + keep) and stack.cache.last is None
    stack.reset()
    assert same(0)


@pytest.mark.parametrize("attn", [False, True])
def test_a_prompt_norms_each_row_once(build, monkeypatch, attn):
    """Launches of the norm over a chunk: the first, and behind every residual the norm that the next segment takes."""
    calls = []
    monkeypatch.setattr(generate, "residual_rmsnorm", lambda x, y, mixed, stream_out=None, weight=None, eps=0: calls.append(
        (y is not None, stream_out is x, weight)))
    stack = build(pages(n=12) if attn else None, prompt_chunk=16)
    g = stack.graph
    g.norm_weights, g.attn_norms = ["mlp0", "mlp1", "final"], ["attn0", "attn1"]
    g.attn = [lambda x, *args: x] * 2
    stack.prompt(list(range(20)))
    want = [(False, False, "attn0"), (True, True, "mlp0"), (True, True, "attn1"), (True, True, "mlp1"), (True, True, "final")]
    assert calls == 2 * (want if attn else [(False, False, "mlp0"), (True, True, "mlp1"), (True, True, "final")])


def test_the_prompt_layers_of_a_stack_share_their_buffers(build, monkeypatch):
    """48 layers for chunks of 2,048 tokens would hold 10 GB of buffers that only one of them uses at a time."""
    from slotstream_spark_amd.engine.prefill import MoEPrefillLayer

    if not _lib.LIB_PATH.exists():
        pytest.skip("libssmoe.so not built (python -m slotstream_spark_amd.build)")
    monkeypatch.setattr(generate, "MoEPrefillLayer", MoEPrefillLayer)
    for name, value in (("inter", 128), ("experts", 4), ("device", "cpu")):
        monkeypatch.setattr(Pool, name, value, raising=False)
    layers = build(pages(seqs=2), prompt_chunk=16, top_k=2).prompt_layers
    buffers = [[t.data_ptr() for t in (l.workspace, l.h_buf, l.out_rows, l.ids, l.weights, l.routed)] for l in layers]
    assert len(buffers) == 2 and buffers[0] == buffers[1] and layers[0].sh_cat is not layers[1].sh_cat
    bf = torch.zeros(4, H, dtype=torch.bfloat16)
    alone = MoEPrefillLayer(Pool, 0, bf, bf, bf, bf, bf, top_k=2, max_tokens=16)
    assert alone.h_buf.data_ptr() not in buffers[0]
    for kw in (dict(max_tokens=17), dict(top_k=3)):
        with pytest.raises(ValueError, match="do not fit"):
            MoEPrefillLayer(Pool, 0, bf, bf, bf, bf, bf, **{"top_k": 2, "max_tokens": 16, **kw}, buffers=alone)

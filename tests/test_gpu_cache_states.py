"""States, sequences and refusals around the paged cache as the engine's parts use it: forks of the draft head's state, calls that
fail half way, what a stack holds."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.generate import mtp_decode
from slotstream_spark_amd.engine.mtp import MTPState
from slotstream_spark_amd.engine.prefill import MoEPrefillLayer
from slotstream_spark_amd.memory.synth import normal_bf16
from tests.test_gpu_attention_layer import H, K, NL, V, bits, make_head, make_stack, parts  # noqa: F401  (parts is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hc", [1, 4])
def test_forks_of_the_heads_state(parts, hc):  # noqa: F811
    """A fork stepped token by token computes what a draft computes, and leaves no trace; one that lost its rows is refused."""
    ids = [5, 77, 300, 1024, 9, 2000, 31]
    multi = normal_bf16((len(ids), hc * H), 1.0, 930)
    a, b = make_head(parts, hc), make_head(parts, hc)
    for head in (a, b):
        head.consume(ids, multi)
    drafts = a.draft(42, 3)
    want = [t.clone() for t in a.draft_rows(3).out]
    fork, first, h = a.state.fork(), a.state.fork(), a.prev_multi
    for i, token in enumerate([42] + drafts[:2]):
        out, h = a.step(a.embed([token]), h, fork)
        assert torch.equal(bits(out), bits(want[i]))
    assert fork.pos == a.state.pos + 3
    a.step(a.embed([7]), a.prev_multi, first)
    with pytest.raises(ValueError, match="no longer holds"):
        a.step(a.embed([42]), h, fork)
    for head in (a, b):
        head.consume([42], multi[:1])
    with pytest.raises(ValueError, match="head's own rows"):
        a.step(a.embed([7]), a.prev_multi, MTPState(64), state_only=True)
    assert a.draft(9, 3) == b.draft(9, 3) and torch.equal(bits(a.draft_rows(3).out), bits(b.draft_rows(3).out))
    assert _lib.device_error() == 0


def test_prompt_layers_with_shared_buffers(parts):  # noqa: F811
    """A prompt through layers that share their buffers has the bits of one through layers with buffers of their own."""
    pool, lws, lm = parts
    a, b = make_stack(parts, 16), make_stack(parts, 16)
    b.prompt_layers = [MoEPrefillLayer(pool, l, w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g, top_k=K, max_tokens=16)
                       for l, w in enumerate(lws[:NL])]
    tokens = [(37 * i + 5) % V for i in range(40)]
    (na, ma), (nb, mb) = a.prompt(tokens), b.prompt(tokens)
    assert na == nb and torch.equal(bits(ma), bits(mb)) and _lib.device_error() == 0


@pytest.mark.parametrize("prompt_chunk", [0, 16])
def test_positions_of_a_loop(parts, prompt_chunk):  # noqa: F811
    """With the head's own drafts and without: stack, cache and head stand at the end of what was emitted."""
    stack, head, prompt = make_stack(parts, prompt_chunk), make_head(parts, 1), [5, 17, 300, 8, 1234, 77, 9, 9, 2, 64, 1000, 41, 3, 50, 11]
    for draft_fn in (None, lambda pending, depth, n_out: [1] * depth):
        stack.reset()
        head.reset()
        out, nan, _, st = mtp_decode(stack, head, prompt, 20, draft_fn=draft_fn)
        assert len(out) == 20 and not nan and st["rounds"] > 0
        assert stack.st.pos == stack.cache.pos == head.consumed == len(prompt) + 19 and head.state.aligned(head.consumed)
        assert stack.st.tokens == prompt + out[:19]                # the last token is emitted and not run
    assert _lib.device_error() == 0


def test_pages_behind_the_window_given_back_between_rounds(parts):  # noqa: F811
    """A loop under windows that evicts before each round emits the same tokens and holds fewer pages."""
    prompt, outs, free = [5, 17, 300, 8, 1234, 77, 9, 9, 2, 64, 1000, 41, 3, 50, 11, 600, 23, 90, 4], [], []
    for evict in (False, True):
        stack, head = make_stack(parts, 16, max_tokens=96, window=20), make_head(parts, 1)

        def drafts(pending, depth, n_out):
            if evict:
                stack.cache.pages.evict(stack.cache.seq, 20, 2, back=stack.rows)
            return [pending, 1] if n_out % 3 else [1, pending]

        out, nan, _, st = mtp_decode(stack, head, prompt, 40, draft_fn=drafts)
        assert not nan and st["rounds"] > 10
        outs.append(out)
        free.append(stack.cache.pages.free_pages)
    assert outs[0] == outs[1] and free[1] > free[0] and _lib.device_error() == 0

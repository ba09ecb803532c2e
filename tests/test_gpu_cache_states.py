"""States, sequences and refusals around the paged cache as the engine's parts use it: forks of the draft head's state, calls that
fail half way, what a stack holds."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.mtp import MTPState
from slotstream_spark_amd.memory.synth import normal_bf16
from tests.test_gpu_attention_layer import H, bits, make_head, parts  # noqa: F401  (parts is a fixture)

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

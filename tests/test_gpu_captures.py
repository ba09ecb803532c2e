"""Captures of rounds and draft chains beside garbage: what Python's cyclic collector frees is never freed inside one."""
import gc

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.mtp import DraftGraph
from slotstream_spark_amd.memory.synth import normal_bf16
from tests.test_gpu_attention_layer import H, make_head, make_stack, parts  # noqa: F401  (parts is a fixture)

pytestmark = pytest.mark.gpu


class Litter:
    """A callable that leaves a cycle behind at each call; the cycle's end notes whether a capture was on."""

    def __init__(self, inner, ends):
        self.inner, self.ends = inner, ends

    def __call__(self, *a, **kw):
        class End:
            def __init__(self, ends):
                self.ends, self.me = ends, self

            def __del__(self):
                self.ends.append(torch.cuda.is_current_stream_capturing())

        End(self.ends)
        return self.inner(*a, **kw)

    def __getattr__(self, name):
        return getattr(self.inner, name)


@pytest.fixture
def eager():
    """The collector at every few objects, as in a program that makes many."""
    was = gc.get_threshold()
    gc.set_threshold(5, 2, 2)
    yield
    gc.set_threshold(*was)


def test_a_round_is_captured_without_collections(parts, eager):  # noqa: F811
    ends, stack = [], make_stack(parts)
    stack.graph.layers = [Litter(x, ends) for x in stack.graph.layers]
    stack.prompt([5, 17, 300, 8])
    gc.collect()
    assert len(ends) >= 4 and not any(ends) and gc.isenabled() and _lib.device_error() == 0


def test_a_draft_chain_is_captured_without_collections(parts, eager):  # noqa: F811
    ends, head = [], make_head(parts, 1)
    head.consume([5, 77, 300], normal_bf16((3, H), 1.0, 930))
    head.moe = Litter(head.moe, ends)
    graph = DraftGraph(head, 2)
    graph.token.fill_(42)
    graph.multi.copy_(head.prev_multi)
    graph.replay()
    torch.cuda.synchronize()
    gc.collect()
    assert len(ends) >= 4 and not any(ends) and gc.isenabled() and _lib.device_error() == 0


def test_the_collector_stays_off_where_it_was_off(parts):  # noqa: F811
    gc.disable()
    try:
        make_stack(parts).prompt([5, 17])
        assert not gc.isenabled()
    finally:
        gc.enable()

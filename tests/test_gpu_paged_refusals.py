"""What the operators on a paged cache are given that they cannot follow: raised in the device status or refused, the rest as ever."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.kernels.rope import rope_append
from tests.paged_util import Batch, half_step, rope64
from tests.test_gpu_rope import freqs, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [3, -1, 2 ** 31 - 1])
def test_an_axis_that_does_not_exist_is_raised(bad):
    """Its frequency is turned by position 0; the others as ever."""
    b = Batch([9, 3], [20, 40], 4, 2, 64, 16)
    qkv, pos = inputs(b, 7, axes=3)
    axis = (torch.arange(32) % 3).to(torch.int32)
    rest = [freqs(64).cuda()] + b.args()[1:]
    d = qkv.cuda()
    call = lambda ax: rope_append(d[:, :4], d[:, 4:6], d[:, 6:], pos.cuda(), *rest, axis=ax.cuda())  # noqa: E731
    call(axis)
    assert _lib.device_error() == 0
    axis[5] = bad
    got = call(axis)
    assert _lib.device_error() == 64 and _lib.device_error() == 0
    zero = torch.cat([pos, torch.zeros_like(pos[:1])])
    axis[5] = 3
    want = rope64(qkv[:, :4], zero, freqs(64), axis)
    # one rounding of the result, and fp32 steps before it of values of a few units (as in test_gpu_rope)
    assert ((got.double().cpu() - want).abs() <= half_step(b.dtype) * want.abs() + 1e-5).all()


def test_a_batch_on_the_default_table_keeps_the_whole_card():
    """64 sequences of 2,000 tokens on their own table and on one of 131,072 (KVPages' default): the same result within its bound, and
    a call that costs idle workgroups more. On one of the 8 XCDs it took 14 times as long; 1.4 times is measured."""
    g = torch.Generator(device="cuda").manual_seed(3)
    seqs, kv_heads, page, held = 64, 8, 64, 32
    k = torch.randn(seqs * held, kv_heads, page, 128, generator=g, device="cuda").to(torch.bfloat16)
    v = torch.randn(seqs * held, kv_heads, 128, page, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(seqs, 32, 128, generator=g, device="cuda").to(torch.bfloat16)
    narrow = torch.arange(seqs * held, dtype=torch.int32, device="cuda").view(seqs, held)
    wide = torch.full((seqs, 2048), -1, dtype=torch.int32, device="cuda")
    wide[:, :held] = narrow
    cu = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    kv_len = torch.full((seqs,), 2000, dtype=torch.int32, device="cuda")

    def call(table):
        out = paged_attention(q, k, v, cu, kv_len, table, 1)
        torch.cuda.synchronize()
        times = []
        for _ in range(9):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                paged_attention(q, k, v, cu, kv_len, table, 1)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return out.double(), sorted(times)[4]

    (a, t_narrow), (b, t_wide) = call(narrow), call(wide)
    # each is off by its rounding and by those of the probabilities (paged_util.attention_bound), the values' mass at most 5
    assert ((a - b).abs() <= half_step(q.dtype) * (a.abs() + b.abs()) + 2 * (half_step(q.dtype) + 2.0 ** -16) * 5).all()
    assert t_wide < 5 * t_narrow, (t_wide, t_narrow)
    assert _lib.device_error() == 0

"""What the operators on a paged cache are given that they cannot follow: raised in the device status or refused, the rest as ever."""
import pytest
import torch

from slotstream_spark_amd import _lib
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

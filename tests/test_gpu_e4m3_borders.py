"""Keys whose largest turned element lies beside 448 2^n, where the cache's power of two changes: the bytes are those of the rows turned in
64 bits, to the last one."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.rope import rope_append
from tests.paged_util import Batch, rope64
from tests.tree_util import E4M3, quantise64, values64

pytestmark = pytest.mark.gpu


def keys_beside(rows, kv_heads, dim, rot, adjacent, top, g):
    """Key rows in which one turned element is +-top 2^n, the other of its pair up to as large, and the rest small."""
    half = rot // 2
    k = (torch.rand(rows, kv_heads, dim, generator=g, dtype=torch.float64) - 0.5) * top
    f = torch.randint(0, half, (rows, kv_heads), generator=g)
    i0, i1 = (2 * f, 2 * f + 1) if adjacent else (f, f + half)
    swap = torch.rand(rows, kv_heads, generator=g) < 0.5
    i0, i1 = torch.where(swap, i1, i0), torch.where(swap, i0, i1)
    sign = (torch.randint(0, 2, (rows, kv_heads), generator=g) * 2 - 1).double()
    other = (torch.rand(rows, kv_heads, generator=g, dtype=torch.float64) * 2 - 1) * 0.9 * top
    other[torch.rand(rows, kv_heads, generator=g) < 0.1] = 0.0
    k.scatter_(2, i0[..., None], (sign * top)[..., None])
    k.scatter_(2, i1[..., None], other[..., None])
    return (k * torch.exp2(torch.randint(-60, 60, (rows, kv_heads, 1), generator=g).double())).to(torch.bfloat16)


@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 16), (128, 128), (128, 48), (256, 256), (256, 64)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("axes,factor", [(1, 1.0), (3, 1.0), (1, 1.75)])
def test_bytes_of_keys_beside_a_border(dim, rot, adjacent, axes, factor):
    rows, kv_heads, page = 260, 3, 64
    print(f"[border] dim={dim} rot={rot} adjacent={adjacent} axes={axes} factor={factor}", flush=True)
    b = Batch([rows, 1], [rows + 70, 5], 6, kv_heads, dim, page, seed=dim + rot)
    g = torch.Generator().manual_seed(dim * rot + axes)
    total = rows + 1
    k = keys_beside(total, kv_heads, dim, rot, adjacent, 2.0 if factor == 1.75 else 3.5, g)
    q, v = (torch.randn(total, h, dim, generator=g).to(torch.bfloat16) for h in (6, kv_heads))
    # angles from a few units down to 10^-13, both ways: the border is passed by as little as the other element's share
    inv = 10.0 ** (-13 * torch.rand(rot // 2, generator=g, dtype=torch.float64))
    inv *= torch.randint(0, 2, (rot // 2,), generator=g) * 2 - 1
    pos = torch.randint(0, 40, (axes, total), generator=g).to(torch.int32)
    axis = torch.arange(rot // 2, dtype=torch.int32) % axes if axes > 1 else None
    n = b.k.shape[0]
    k8 = torch.zeros(n, kv_heads, page, dim, dtype=torch.uint8, device="cuda").view(E4M3)
    v8 = torch.zeros(n, kv_heads, dim, page, dtype=torch.uint8, device="cuda").view(E4M3)
    sc = torch.zeros(n, kv_heads, 2, page, dtype=torch.uint8, device="cuda")
    rope_append(q.cuda(), k.cuda(), v.cuda(), pos.cuda(), inv.cuda(), k8, v8, b.cu.cuda(), b.kv_len.cuda(), b.table.cuda(), b.max_rows,
                axis=None if axis is None else axis.cuda(), adjacent=adjacent, factor=factor, scales=sc)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    turned = rope64(k, pos, inv, axis, adjacent, factor)
    _, want = quantise64(turned)
    at = torch.cat([torch.arange(70, 70 + rows), torch.tensor([4])])
    ids = torch.cat([b.table[0].long()[at[:-1] // page], b.table[1].long()[at[-1:] // page]])
    got = sc.cpu()[ids, :, 0, at % page]
    top = turned.abs().amax(2)
    close = (top / torch.exp2(want.double() - 127) / 448 - 1).abs() < 1e-6
    assert close.any() and ((top / torch.exp2(want.double() - 127) / 224 - 1).abs() < 1e-6).any()  # both sides are there
    assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()} bytes"
    # one rounding of the numbers, 2^-4 of the value or half of the least step, of rows turned in fp32 (2^-20 of the largest, at most)
    codes = k8.cpu()[ids, :, at % page].double()
    by = torch.exp2(want.double() - 127)[..., None]
    assert ((codes * by - turned).abs() <= (2.0 ** -4 * turned.abs()).maximum(2.0 ** -10 * by) + 2.0 ** -20 * top[..., None]).all()

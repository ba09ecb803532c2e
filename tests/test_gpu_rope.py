"""Rotary positions and the cache write against their definition in 64 bits, and page moves against indexing. A turned
element x cos a - y sin a is computed in fp32 (a few 2^-24 of |x| + |y|) and rounded once to 16 bits."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.kv_pages import move_pages
from slotstream_spark_amd.kernels.rope import rope_append
from tests.paged_util import Batch, half_step, rope64

pytestmark = pytest.mark.gpu


def inputs(b, seed, axes=1, top=4000):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b.total, b.heads + 2 * b.kv_heads, b.dim, generator=g).to(b.dtype)
    pos = torch.randint(0, top, (axes, b.total), generator=g).to(torch.int32)
    return qkv, pos


def freqs(rot, base=1e6):
    return base ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))


def check(b, rot, axes=1, adjacent=False, factor=1.0, top=4000, seed=0):
    qkv, pos = inputs(b, seed, axes, top)
    f = freqs(rot)
    axis = (torch.arange(rot // 2) % axes).to(torch.int32) if axes > 1 else None
    _, kp, vp, cu, kv_len, table, n = b.args()
    d = qkv.cuda()
    q, k, v = d[:, :b.heads], d[:, b.heads:b.heads + b.kv_heads], d[:, b.heads + b.kv_heads:]
    out = rope_append(q, k, v, pos.cuda(), f.cuda(), kp, vp, cu, kv_len, table, n,
                      axis=None if axis is None else axis.cuda(), adjacent=adjacent, factor=factor)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    turned = rope64(qkv[:, :b.heads + b.kv_heads], pos, f, axis, adjacent, factor)
    # |x cos| + |y sin| <= factor * (|x| + |y|): one rounding to 16 bits, 8 fp32 half steps before it, and the angle's own
    # rounding in 64 bits (here and there: three steps of 2^-53 relative)
    mag = qkv[:, :b.heads + b.kv_heads].double().abs()
    pair = mag.clone()
    half = rot // 2
    if adjacent:
        pair[..., 0:rot:2] += mag[..., 1:rot:2]
        pair[..., 1:rot:2] += mag[..., 0:rot:2]
    else:
        pair[..., :half] += mag[..., half:rot]
        pair[..., half:rot] += mag[..., :half]
    bound = half_step(b.dtype) * turned.abs() + (8 * 2.0 ** -24 + top * 2.0 ** -51) * abs(factor) * pair + 2.0 ** -25
    assert ((out.double().cpu() - turned[:, :b.heads]).abs() <= bound[:, :b.heads]).all()
    if rot < b.dim:
        assert torch.equal(out[..., rot:].cpu(), qkv[:, :b.heads, rot:])
    wk, wv = b.k.double().clone(), b.v.clone()
    ek, r = torch.zeros_like(wk), 0
    for s, rows in enumerate(b.rows):
        for i in range(rows):
            p = b.lens[s] - rows + i
            if p >= 0:
                page, off = int(b.table[s, p // b.page]), p % b.page
                wk[page, :, off], ek[page, :, off] = turned[r, b.heads:], bound[r, b.heads:]
                wv[page, :, :, off] = qkv[r, b.heads + b.kv_heads:]
            r += 1
    assert ((kp.double().cpu() - wk).abs() <= ek).all()             # every other place as it was
    assert torch.equal(vp.cpu().view(torch.int16), wv.view(torch.int16))


@pytest.mark.parametrize("rot,axes,adjacent", [(64, 1, False), (64, 1, True), (32, 3, False), (16, 3, True), (48, 4, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_kinds(rot, axes, adjacent, dtype):
    check(Batch([1, 5, 9, 0, 64], [1, 20, 33, 7, 200], 6, 2, 64, 16, dtype), rot, axes, adjacent)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 32), (256, 64), (256, 256)])
def test_pages_and_dims(page, dim, rot):
    check(Batch([1, 3, 70, 8], [300, 258, 77, 8], 4, 1, dim, page, seed=page), rot, seed=dim)


def test_first_places_of_a_chunk():
    """Every start inside a group of 8 tokens, with few and many rows."""
    check(Batch([n for n in (1, 2, 7, 8, 9, 17) for _ in range(8)], [n + o for n in (1, 2, 7, 8, 9, 17) for o in range(8)],
                2, 1, 64, 16), 64)


def test_far_positions_keep_their_angles():
    check(Batch([9], [9], 2, 1, 64, 16), 64, top=2 ** 31 - 1)


def test_factor_and_negative_positions():
    check(Batch([9], [9], 2, 1, 64, 16), 64, factor=1.3)
    b = Batch([4], [40], 2, 2, 64, 16)
    qkv, pos = inputs(b, 3)
    a = [qkv.cuda()[:, :2], qkv.cuda()[:, 2:4], qkv.cuda()[:, 4:]]
    rest = b.args()[1:]
    got = rope_append(*a, (-pos).cuda(), freqs(64).cuda(), *rest)
    want = rope64(qkv[:, :2], -pos, freqs(64))
    assert ((got.double().cpu() - want).abs() <= half_step(b.dtype) * want.abs() + 1e-5).all()


def test_rows_without_a_place():
    """More rows than tokens: the first are turned and not written; rows past the batch are left alone."""
    check(Batch([5, 3], [2, 0], 2, 1, 64, 16), 64)
    b = Batch([2], [20], 2, 1, 64, 16)
    d = torch.randn(4, 4, 64, dtype=b.dtype, device="cuda")
    _, kp, vp, cu, kv_len, table, n = b.args()
    out = torch.full((4, 2, 64), 3.0, dtype=b.dtype, device="cuda")
    rope_append(d[:, :2], d[:, 2:3], d[:, 3:], torch.arange(4, dtype=torch.int32, device="cuda"), freqs(64).cuda(), kp, vp,
                cu, kv_len, table, n, out=out)
    assert (out[2:] == 3).all() and (out[:2] != 3).any()


def test_in_place_and_graph():
    b = Batch([1, 1], [50, 70], 4, 2, 64, 16)
    qkv, pos = inputs(b, 4)
    d = qkv.cuda()
    q = d[:, :4].contiguous()
    rest = [pos.cuda(), freqs(64).cuda()] + b.args()[1:]
    want = rope_append(q, d[:, 4:6], d[:, 6:], *rest)
    same = q.clone()
    assert rope_append(same, d[:, 4:6], d[:, 6:], *rest, out=same).data_ptr() == same.data_ptr()
    assert torch.equal(same, want)
    out, graph = torch.zeros_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope_append(q, d[:, 4:6], d[:, 6:], *rest, out=out)
    for step in range(3):
        rest[0].add_(step)
        rest[5].sub_(step)
        graph.replay()
        assert torch.equal(out, rope_append(q, d[:, 4:6], d[:, 6:], *rest))
    assert _lib.device_error() == 0


def test_bad_pages_are_not_written():
    b = Batch([3], [40], 2, 1, 64, 16)
    b.table[0, 2] = 99
    qkv, pos = inputs(b, 5)
    d = qkv.cuda()
    _, kp, vp, cu, kv_len, table, n = b.args()
    rope_append(d[:, :2], d[:, 2:3], d[:, 3:], pos.cuda(), freqs(64).cuda(), kp, vp, cu, kv_len, table, n)
    assert _lib.device_error() == 32
    assert torch.equal(kp.cpu(), b.k) and torch.equal(vp.cpu(), b.v)


# ---------------------------------------------------------------- page moves
@pytest.mark.parametrize("layers,pages,n,kv_heads,page,dim,dtype", [
    (1, 5, 1, 1, 16, 64, torch.bfloat16), (3, 40, 13, 3, 16, 64, torch.float16), (2, 3000, 1400, 1, 32, 128, torch.bfloat16),
    (12, 9, 4, 2, 256, 256, torch.bfloat16), (1, 9, 0, 1, 16, 64, torch.bfloat16)])
def test_move_pages(layers, pages, n, kv_heads, page, dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(pages)
    k = torch.randn(layers, pages, kv_heads, page, dim, generator=g, device="cuda").to(dtype)
    v = torch.randn(layers, pages, kv_heads, dim, page, generator=g, device="cuda").to(dtype)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    src, dst = perm[:n].contiguous(), perm[n:2 * n].contiguous()
    table = torch.randint(-1, pages, (7, 333), generator=g, device="cuda").to(torch.int32)
    wk, wv = k.clone(), v.clone()
    wk[:, dst.long()], wv[:, dst.long()] = k[:, src.long()], v[:, src.long()]
    to = {int(a): int(b) for a, b in zip(src.tolist(), dst.tolist())}
    want = torch.tensor([[to.get(p, p) for p in row] for row in table.tolist()], dtype=torch.int32)
    move_pages(k, v, src, dst, table)
    assert torch.equal(k.view(torch.int16), wk.view(torch.int16)) and torch.equal(v.view(torch.int16), wv.view(torch.int16))
    assert torch.equal(table.cpu(), want)
    assert _lib.device_error() == 0


def test_move_skips_pages_outside_the_cache():
    k = torch.randn(2, 6, 1, 16, 64, device="cuda").to(torch.bfloat16)
    v = torch.randn(2, 6, 1, 64, 16, device="cuda").to(torch.bfloat16)
    wk, wv = k.clone(), v.clone()
    wk[:, 3], wv[:, 3] = k[:, 0], v[:, 0]
    table = torch.tensor([0, 1, 2, -1, 9], dtype=torch.int32, device="cuda")
    move_pages(k, v, torch.tensor([0, 9, 1, -1], dtype=torch.int32, device="cuda"),
               torch.tensor([3, 4, 6, 5], dtype=torch.int32, device="cuda"), table)
    assert _lib.device_error() == 32
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert table.tolist() == [3, 1, 2, -1, 9]

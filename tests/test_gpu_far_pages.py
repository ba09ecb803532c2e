"""A cache in 8 bits whose pages lie past 4 GiB: every operator over it gives the bits that it gives over the same pages at the front of a small
one, in few and many rows, trees and causal rows."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.kv_pages import move_pages
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.kernels.rope import rope_append
from slotstream_spark_amd.kernels.tree import keep_rows
from tests.tree_util import E4M3, as_int64, masks_of, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 24])
def test_pages_past_4_gib(rows):
    heads, kv, dim, page, held, n = 16, 8, 256, 256, 6, 8210          # 512 KB a page: 4.3 GB of keys, as many of values
    g = torch.Generator(device="cuda").manual_seed(rows)
    near, far = torch.arange(held), torch.tensor([8209, 8195, 8200, 8193, 8208, 8199])
    caches = []
    for many, ids in ((held, near), (n, far)):
        k = torch.zeros((1, many, kv, page, dim), dtype=torch.uint8, device="cuda")
        v = torch.zeros((1, many, kv, dim, page), dtype=torch.uint8, device="cuda")
        sc = torch.zeros((1, many, kv, 2, page), dtype=torch.uint8, device="cuda")
        g.manual_seed(5)
        for p in ids.tolist():
            k[0, p] = (torch.randn((kv, page, dim), generator=g, device="cuda") * 80).to(E4M3).view(torch.uint8)
            v[0, p] = (torch.randn((kv, dim, page), generator=g, device="cuda") * 80).to(E4M3).view(torch.uint8)
            sc[0, p] = torch.randint(119, 122, (kv, 2, page), generator=g, device="cuda", dtype=torch.uint8)
        caches.append((k.view(E4M3), v.view(E4M3), sc, ids, ids.to(torch.int32).view(2, 3).cuda()))
    cu = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([600, 700], dtype=torch.int32, device="cuda")
    qkv = torch.randn((2 * rows, heads + 2 * kv, dim), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 5000, (1, 2 * rows), generator=g, device="cuda").to(torch.int32)
    inv = 1e4 ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    tree = as_int64(sum((masks_of(random_parents(rows, s)) for s in (1, 2)), [])).cuda()
    took = torch.full((2, 4 + 2 * rows), -1, dtype=torch.int32)
    path = list(range(0, rows, 2))
    took[:, 0], took[:, 4 + rows:4 + rows + len(path)] = len(path) - 1, torch.tensor(path, dtype=torch.int32)
    took, got = took.cuda(), []
    for k, v, sc, ids, table in caches:
        q = rope_append(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], pos, inv, k[0], v[0], cu, kv_len, table, rows, scales=sc[0])
        out = [q] + [paged_attention(q, k[0], v[0], cu, kv_len, table, rows, scales=sc[0], tree=t, window=w) for t in (None, tree) for w in (0, 300)]
        bad = int(ids[0])                                            # a NaN value of a token before the window reaches no row there
        v.view(torch.uint8)[0, bad, :, 3, 1] = 0x7F
        out += [paged_attention(q, k[0], v[0], cu, kv_len, table, rows, scales=sc[0], tree=t, window=w) for t in (None, tree) for w in (0, 300)]
        assert torch.isnan(out[5]).any() and not torch.isnan(out[6]).any()
        keep_rows(k, v, cu, kv_len, table, took, scales=sc)
        move_pages(k, v, ids[1:2].to(torch.int32).cuda(), ids[3:4].to(torch.int32).cuda(), scales=sc)
        held_now = [t.view(torch.uint8)[0, p].clone() for p in ids.tolist() for t in (k, v, sc)]
        assert all(torch.equal(x, y) for x, y in zip(held_now[3:6], held_now[9:12]))
        got.append([t.view(torch.int16) for t in out] + held_now)
    assert all(torch.equal(x, y) for x, y in zip(*got)) and len(got[0]) == len(got[1])
    assert _lib.device_error() == 0

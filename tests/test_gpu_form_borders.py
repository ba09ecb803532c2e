"""Calls on both sides of the borders between the few-row and the many-row form over e4m3 pages and for trees: packed rows (32, 64, 128),
tables (512, 768, 1,408, 4,096 tokens) and what a chunk holds (512, 768 or 1,024 tokens more)."""
import pytest
import torch

from tests import test_gpu_e4m3_cache as causal, test_gpu_tree as tree
from tests.test_gpu_tree import make, trees

pytestmark = pytest.mark.gpu

# heads on one key head and rows of a sequence: 32, 33 / 34, 64, 65 / 66, 128 and 129 / 132 packed rows
PACKED = [(2, 16), (3, 11), (2, 17), (4, 16), (5, 13), (6, 11), (8, 16), (4, 32), (3, 43), (4, 33)]
TABLES = [496, 512, 528, 752, 768, 784, 896, 912, 1136, 1152, 1392, 1408, 1424, 4096, 4112]


@pytest.mark.parametrize("table", TABLES)
@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("e4m3", 64), ("e4m3", 128), ("e4m3", 256), ("fp16", 256), ("bf16", 64)])
def test_trees(kind, dim, table):
    for i, (heads, rows) in enumerate(PACKED):
        b = make(kind, [rows, 1 + rows // 2], [min(table, rows + 37 * i + 300), rows], heads, 1, dim, 16, seed=table + i, width=table // 16)
        tree.check(b, trees(b))


@pytest.mark.parametrize("table", TABLES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_causal_rows(dim, table):
    for i, (heads, rows) in enumerate(PACKED):
        causal.check(make("e4m3", [rows, 1 + rows // 2], [min(table, rows + 37 * i + 300), rows], heads, 1, dim, 16, seed=table + i, width=table // 16))


@pytest.mark.parametrize("seqs,kv_heads", [(1, 1), (8, 4), (16, 4), (64, 1)])
@pytest.mark.parametrize("dim", [64, 256])
def test_tables_of_one_chunk(seqs, kv_heads, dim):
    """Few and many workgroups over tables that are one chunk or little more."""
    for table in (624, 1040, 1168):
        lens = [min(table, 13 + 29 * s % 400) for s in range(seqs)]
        lens[-1] = table
        rows = [min(12, n) for n in lens]
        for kind in ("bf16", "e4m3"):
            b = make(kind, rows, lens, 2 * kv_heads, kv_heads, dim, 16, seed=table + seqs, width=table // 16)
            tree.check(b, trees(b))
            if kind == "e4m3":
                causal.check(b)

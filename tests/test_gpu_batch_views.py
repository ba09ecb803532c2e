"""Trees whose batch tensors are views of a larger batch's (cu_rows[m:], kv_len[m:], table[m:]: prompts beside them go in another call): the
rows are absolute, so nothing may go by how many the view has."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.kernels.tree import accept_tree, keep_rows, tree_masks
from tests.test_gpu_tree import KINDS, make, round_of
from tests.tree_util import accept64, as_int64, masks_of, random_parents, tree64, tree_bound

pytestmark = pytest.mark.gpu

PROMPT, TREES, LENS = 256, [12, 0, 30, 1], [300, 12, 77, 400, 9]   # rows of the first sequence; the trees' rows; tokens of all


@pytest.mark.parametrize("kind", KINDS)
def test_a_round_beside_a_prompt(kind):
    """Masks, attention, acceptance and the branch's move over the view are those of the trees' own batch, and the prompt's rows and tokens stay."""
    rows, vocab, dim, page = [PROMPT] + TREES, 601, 64, 16
    b = make(kind, rows, LENS, 4, 2, dim, page, seed=31)
    total = sum(rows)
    parents = [random_parents(n, 40 + n) if n else [] for n in TREES]
    flat = torch.tensor([-1] * PROMPT + sum(parents, []), dtype=torch.int32)
    cu, kv_len, table = b.cu.cuda(), b.kv_len.cuda(), b.table.cuda()
    view = (cu[1:], kv_len[1:], table[1:])
    masks, pos = tree_masks(flat.cuda(), cu[1:], kv_len[1:], 30)
    words = sum((masks_of(p) for p in parents), [])
    assert masks[:PROMPT].abs().sum() == 0 and torch.equal(masks[PROMPT:].cpu(), as_int64(words))
    base = sum(([LENS[1 + s] - n] * n for s, n in enumerate(TREES)), [])
    assert pos[PROMPT:].cpu().tolist() == [t + bin(w).count("1") - 1 for t, w in zip(base, words)]
    pages = [b.k8.cuda(), b.v8.cuda()] if kind == "e4m3" else [b.k.cuda(), b.v.cuda()]
    sc = b.scales.cuda() if kind == "e4m3" else None
    out = torch.full((total, 4, dim), 3.0, dtype=b.dtype, device="cuda")
    paged_attention(b.q.cuda(), *pages, *view, 30, scales=sc, tree=masks, out=out)
    assert (out[:PROMPT] == 3).all()
    want, _ = tree64(b, [1] * PROMPT + words)
    bound = tree_bound(b, [1] * PROMPT + words)
    assert ((out.double().cpu() - want).abs() <= bound)[PROMPT:].all()
    target, tokens, _, _ = round_of(rows, vocab, 33, follow=0.0)
    for s, p in enumerate(parents):                       # the branch of a tree's last row is the target's choice
        at, i = int(b.cu[1 + s]), len(p) - 1
        while i > 0:
            tokens[at + i] = target[at + p[i]].argmax()
            i = p[i]
    took = accept_tree(target.cuda(), tokens.cuda(), flat.cuda(), cu[1:], 30)
    assert torch.equal(took.cpu(), accept64(target, tokens, flat, b.cu.tolist()[1:], 30))
    path = [r for r in took[2, 34:].tolist() if r >= 0]
    assert len(path) > 2 and path != list(range(len(path)))
    bits = torch.uint8 if kind == "e4m3" else torch.int16
    stack = [t.view(bits)[None].repeat(2, *[1] * t.dim()).contiguous() for t in pages] + ([sc[None].repeat(2, 1, 1, 1, 1)] if sc is not None else [])
    own = [t.clone() for t in stack]
    move = lambda t, *batch: keep_rows(t[0].view(pages[0].dtype), t[1].view(pages[0].dtype), *batch, took,  # noqa: E731
                                       scales=t[2] if sc is not None else None)
    before = stack[0].clone()
    move(own, (cu[1:] - PROMPT).contiguous(), kv_len[1:].clone(), table[1:].clone())
    move(stack, *view)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert not torch.equal(own[0], before) and all(torch.equal(x, y) for x, y in zip(stack, own))
    held = [int(p) for p in b.table[0] if p >= 0]
    assert torch.equal(stack[0][:, held], before[:, held])

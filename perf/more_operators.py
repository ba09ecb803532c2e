"""Speculation with trees of drafts over a paged key-value cache in 8 bits, as cases that can be timed and compared.

Five operators that one round calls in turn: `append` turns the query and key rows by their positions and writes key and value
rows into pages of e4m3 numbers, each token's and head's with a power of two of its own; `attend` is the attention of a batch's
new rows over such pages, from one decoded token to prompts; `tree` is the attention of a tree of drafted tokens, whose rows see
the cache and their own ancestors, over pages of 16 bits or of e4m3; `accept` walks each tree by the target's largest logits;
`keep` moves the accepted branch's keys and values to where the next round expects them, in every layer.

The cache of a layer: keys [pages, kv heads, page, dim], values [pages, kv heads, dim, page]; in 8 bits also `scales` uint8
[pages, kv heads, 2, page]: the token's keys are their e4m3 numbers times 2^(scales[.., 0, .] - 127), its values times
2^(scales[.., 1, .] - 127). A batch: `cu` int32 [seqs + 1], `kv_len` int32 [seqs], `table` int32 [seqs, width], as
perf/operators.py has them. A tree: `masks` int64 [rows], bit j of a row: it sees row j of its sequence (itself among them);
`parents` int32 [rows], a row's parent among its sequence's rows, -1 for the first.
With `own` false, `run` is the plain form in elementary torch operations; with `own` true the package's entry points.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
TOP = 448.0  # the largest e4m3 number


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # The new token's rows of 64 chats into 64 pages of 8 bits.
        dict(name="append_decode_64", op="append", seqs=64, rows=1, length=4096, heads=32, kv_heads=4, dim=128, rot=128,
             axes=1, page=64, ragged=True),
        # A prompt with images: three position axes over a quarter of a wide head, chunks that begin inside a page.
        dict(name="append_prompt_axes", op="append", seqs=2, rows=4095, length=6001, heads=16, kv_heads=2, dim=256, rot=64,
             axes=3, page=64, ragged=False),
        # The verify rows of depth-2 speculation of eight chats over a cache in 8 bits.
        dict(name="attend8_verify", op="attend", type="e4m3", seqs=8, rows=3, length=6145, heads=16, kv_heads=2, dim=256,
             window=0, sinks=0, page=64, ragged=True),
        # A full serving batch of single tokens, lengths mixed: the cache's bytes are what a token costs.
        dict(name="attend8_decode_batch", op="attend", type="e4m3", seqs=64, rows=1, length=16384, heads=32, kv_heads=8,
             dim=128, window=0, sinks=0, page=64, ragged=True),
        # A long prompt chunk behind a longer context.
        dict(name="attend8_prompt", op="attend", type="e4m3", seqs=1, rows=4095, length=9000, heads=32, kv_heads=8, dim=128,
             window=0, sinks=0, page=64, ragged=False),
        # A small tree of one short chat: nothing but latency.
        dict(name="tree_one", op="tree", type="bf16", seqs=1, rows=12, length=777, heads=32, kv_heads=4, dim=128, window=0,
             sinks=0, page=64, ragged=False),
        # Trees of up to 26 drafts for sixteen chats.
        dict(name="tree_batch", op="tree", type="bf16", seqs=16, rows=26, length=8000, heads=32, kv_heads=4, dim=128,
             window=0, sinks=0, page=64, ragged=True),
        # Trees of the largest size behind long contexts in 8 bits.
        dict(name="tree8_long", op="tree", type="e4m3", seqs=4, rows=64, length=50000, heads=32, kv_heads=8, dim=128,
             window=0, sinks=0, page=64, ragged=False),
        # One chat's tree against the logits of its rows.
        dict(name="accept_one", op="accept", seqs=1, rows=12, vocab=151936, ragged=False),
        # Sixteen chats' trees, the largest vocabulary.
        dict(name="accept_batch", op="accept", seqs=16, rows=26, vocab=248320, ragged=True),
        # The accepted branch of one chat, all layers.
        dict(name="keep_one", op="keep", type="bf16", layers=48, seqs=1, rows=12, length=777, kv_heads=4, dim=128, page=64,
             ragged=False),
        # Those of 32 chats in 8 bits.
        dict(name="keep_batch", op="keep", type="e4m3", layers=48, seqs=32, rows=64, length=300, kv_heads=8, dim=128, page=64,
             ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "tree", "tree", "accept", "keep"])
    ragged = rng.random() < 0.6
    if op == "accept":
        vocab = _log_int(rng, 1000, 248320)
        rows = _log_int(rng, 1, 64)
        return dict(op=op, seqs=max(1, min(_log_int(rng, 1, 64), int(1e8 / (vocab * rows)))), rows=rows, vocab=vocab, ragged=ragged)
    heads, kv_heads, dim = rng.choice([(32, 4, 128), (32, 8, 128), (16, 2, 256), (24, 8, 64), (20, 4, 128), (10, 2, 64),
                                       (16, 1, 128), (8, 8, 64), (9, 3, 128), (6, 2, 256)])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    shape = dict(kv_heads=kv_heads, dim=dim, page=page, ragged=ragged)
    if op == "keep":
        kind, rows = rng.choice(["bf16", "fp16", "e4m3"]), _log_int(rng, 2, 64)
        return dict(op=op, type=kind, layers=_log_int(rng, 1, 48), seqs=_log_int(rng, 1, 32), rows=rows,
                    length=rows + _log_int(rng, 1, 300) - 1, **shape)
    shape["heads"] = heads
    if op == "append":
        rows = rng.choice([1, rng.randint(2, 64), _log_int(rng, 9, 4000)])
        seqs = _log_int(rng, 1, max(1, min(200, 8000 // rows)))
        return dict(op=op, seqs=seqs, rows=rows, length=rows + _log_int(rng, 1, 4000) - 1, axes=rng.choice([1, 1, 3]),
                    rot=rng.choice([dim, dim, dim // 2, dim // 4]), **shape)
    shape.update(rng.choice([dict(window=0, sinks=0), dict(window=_log_int(rng, 64, 4096), sinks=rng.choice([0, 4, 17]))]))
    if op == "attend" and rng.random() < 0.4:  # a prompt
        length = _log_int(rng, 9, 9000)
        rows = min(length, _log_int(rng, 9, 4000), max(9, int(1.1e11 / (heads * dim * length))))
        return dict(op=op, type="e4m3", seqs=max(1, min(_log_int(rng, 1, 16), int(1.1e11 / (heads * dim * rows * length)))),
                    rows=rows, length=length, **shape)
    rows = rng.randint(1, 8) if op == "attend" else _log_int(rng, 2, 64)
    length = rows + _log_int(rng, 1, 60000)
    seqs = max(1, min(_log_int(rng, 1, 64), int(6e8 / (length * kv_heads * dim)), int(4e10 / (rows * heads * dim * length))))
    return dict(op=op, type="e4m3" if op == "attend" else rng.choice(["bf16", "fp16", "e4m3"]), seqs=seqs, rows=rows,
                length=length, **shape)


# ---------------------------------------------------------------- inputs
class State:
    """What a program keeps between calls: inputs, the cache and its tables, as attributes."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _sizes(case):
    """(new rows, cached tokens) of each sequence: up to the case's own, mixed where it is ragged."""
    rows, lens = [], []
    for s in range(case["seqs"]):
        f = (0.25 + 0.75 * math.modf((s + 1) * 0.6180339887498949)[0]) if case["ragged"] else 1.0
        n = max(1, round(case["rows"] * f)) if case["rows"] > 8 else case["rows"]
        rows.append(n)
        lens.append(max(n, round(case.get("length", n) * f)))
    return rows, lens


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, seed, dtype):
    return torch.randn(shape, generator=_gen(seed), device=DEV, dtype=dtype)


def _pages(shape, seed, kind):
    """Keys or values of a cache: normal ones, in 8 bits as e4m3 numbers of which the largest of a vector come near to TOP."""
    if kind != "e4m3":
        return _normal(shape, seed, TYPES[kind])
    return (_normal(shape, seed, torch.bfloat16) * 80).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)


def _exponents(shape, seed):
    """Scales of pages whose numbers stand for values of about one."""
    return torch.randint(119, 122, shape, generator=_gen(seed), device=DEV, dtype=torch.uint8)


def _parents(rows, seed):
    """A tree for each sequence, in the order that drafters level by level come to: a row's parent is up to three quarters back."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in rows:
        i = torch.arange(1, n)
        lo = (i - 1) // 4
        out += [torch.tensor([-1]), lo + (torch.rand(n - 1, generator=g) * (i - lo)).long()]
    return torch.cat(out).to(torch.int32)


def _masks(parents, cu):
    """Of every row, the rows of its sequence that it sees: itself and its ancestors. int64, bit j for row j."""
    p, seen = parents.tolist(), []
    for lo, hi in zip(cu, cu[1:]):
        for i in range(hi - lo):
            seen.append((1 << i) | (seen[lo + p[lo + i]] if p[lo + i] >= 0 else 0))
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in seen], dtype=torch.int64)


def prepare(case, seed):
    op, seed = case["op"], int(seed) * 1000 + 31
    rows, lens = _sizes(case)
    seqs, total, most = case["seqs"], sum(rows), max(rows)
    cu_list = [0] + torch.tensor(rows).cumsum(0).tolist()
    cu = torch.tensor(cu_list, dtype=torch.int32).to(DEV)
    if op == "accept":
        parents = _parents(rows, seed).to(DEV)
        target = _normal((total, case["vocab"]), seed + 1, torch.float32)
        # a drafter's tokens: two in three are what the target says after their parent
        first = torch.tensor(cu_list[:-1], device=DEV).repeat_interleave(torch.tensor(rows, device=DEV))
        best = target.argmax(1)[first + parents.clamp(min=0)]
        other = torch.randint(0, case["vocab"], (total,), generator=_gen(seed + 2), device=DEV)
        tokens = torch.where(torch.rand(total, generator=_gen(seed + 3), device=DEV) < 0.67, best, other)
        return State(target=target, tokens=tokens.to(torch.int32), parents=parents, cu=cu, max_rows=most)
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    kind = case.get("type", "e4m3")
    width = -(-max(lens) // page) + 1
    need = [-(-n // page) for n in lens]
    first = [0] * seqs
    if case.get("window"):  # pages wholly behind the window of the first new row are not held, but for the first tokens'
        first = [max(0, n - r - case["window"] + 1) // page for r, n in zip(rows, lens)]
    held = [[w for w in range(need[s]) if w >= first[s] or w * page < case["sinks"]] for s in range(seqs)]
    pages = sum(len(h) for h in held) + 3
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    table, at = torch.full((seqs, width), -1, dtype=torch.int32), 0
    for s, h in enumerate(held):
        table[s, torch.tensor(h, dtype=torch.long)] = ids[at:at + len(h)]
        at += len(h)
    lead = (case["layers"],) if op == "keep" else ()
    batch = dict(cu=cu, kv_len=torch.tensor(lens, dtype=torch.int32).to(DEV), table=table.to(DEV), max_rows=most, rows=total,
                 window=case.get("window", 0), sinks=case.get("sinks", 0),
                 k=_pages((*lead, pages, kv_heads, page, dim), seed + 2, kind),
                 v=_pages((*lead, pages, kv_heads, dim, page), seed + 3, kind),
                 scales=_exponents((*lead, pages, kv_heads, 2, page), seed + 6) if kind == "e4m3" else None)
    if op == "keep":  # what `accept` left: an accepted branch of each tree
        parents, took = _parents(rows, seed + 7).tolist(), torch.full((seqs, 4 + 2 * most), -1, dtype=torch.int32)
        pick = torch.rand(seqs, generator=torch.Generator().manual_seed(seed + 8)).tolist()
        for s, n in enumerate(rows):
            i, path = int((0.5 + 0.5 * pick[s]) * (n - 1) + 0.5), []
            while i >= 0:
                path.insert(0, i)
                i = parents[cu_list[s] + i]
            moved = [p for k, p in enumerate(path) if p != k]
            path = path[:moved[0]] if moved else path  # no row is both moved and written over: a pass can be repeated
            took[s, :4] = torch.tensor([len(path) - 1, len(path), 0, 0])
            took[s, 4:4 + len(path)] = 1
            took[s, 4 + most:4 + most + len(path)] = torch.tensor(path)
        return State(took=took.to(DEV), **batch)
    dtype = torch.bfloat16 if kind == "e4m3" else TYPES[kind]
    if op in ("attend", "tree"):
        s = State(q=_normal((total, case["heads"], dim), seed + 4, dtype) * 1.5, **batch)
        s.masks = _masks(_parents(rows, seed + 7), cu_list).to(DEV) if op == "tree" else None
        return s
    # the rows of a fused projection: query, key and value heads side by side
    qkv = _normal((total, case["heads"] + 2 * kv_heads, dim), seed + 4, torch.bfloat16)
    half = case["rot"] // 2
    inv_freq = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
    pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lens)])
    axis = None
    if case["axes"] > 1:  # frames of 24 x 16 patches: time, then rows and columns; the axes alternate over frequencies
        patch = pos % 384
        pos = torch.stack([pos // 384, patch // 16, patch % 16])
        axis = (torch.arange(half) % case["axes"]).to(torch.int32).to(DEV)
    return State(qkv=qkv, pos=pos.reshape(case["axes"], total).to(torch.int32).to(DEV), axis=axis,
                 inv_freq=inv_freq.to(DEV), **batch)


# ---------------------------------------------------------------- one pass
def run(s):
    if hasattr(s, "target"):
        if own:
            from slotstream_spark_amd.kernels.tree import accept_tree
            return accept_tree(s.target, s.tokens, s.parents, s.cu, s.max_rows)
        return _plain_accept(s)
    if hasattr(s, "took"):
        if own:
            from slotstream_spark_amd.kernels.tree import keep_rows
            keep_rows(s.k, s.v, s.cu, s.kv_len, s.table, s.took, scales=s.scales)
        else:
            _plain_keep(s)
        return [s.k, s.v] + ([s.scales] if s.scales is not None else [])
    if hasattr(s, "qkv"):
        h, n = s.k.shape[1], s.qkv.shape[1]
        q, k, v = s.qkv[:, :n - 2 * h], s.qkv[:, n - 2 * h:n - h], s.qkv[:, n - h:]
        if own:
            from slotstream_spark_amd.kernels.rope import rope_append
            out = rope_append(q, k, v, s.pos, s.inv_freq, s.k, s.v, s.cu, s.kv_len, s.table, s.max_rows, axis=s.axis,
                              scales=s.scales)
        else:
            out = _plain_append(s, q, k, v)
        return [out, s.k, s.v, s.scales]
    if own:
        from slotstream_spark_amd.kernels.paged_attention import paged_attention
        lse = torch.empty(s.q.shape[:2], dtype=torch.float32, device=s.q.device)
        out = paged_attention(s.q, s.k, s.v, s.cu, s.kv_len, s.table, s.max_rows, window=s.window, sinks=s.sinks, lse=lse,
                              scales=s.scales, tree=s.masks)
        return [out, lse]
    return _plain_attend(s)


def _rows_of(s):
    """Of every row: its sequence, its place among the sequence's rows and the place of the sequence's first row in the cache."""
    n = (s.cu[1:] - s.cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=n.device), n, output_size=s.rows)
    return seq, torch.arange(s.rows, device=n.device) - s.cu.long()[seq], s.kv_len.long()[seq] - n[seq]


def _eight(x):
    """(e4m3 numbers, exponents) of vectors in 64 bits: by the least power of two with which none is over TOP."""
    m, e = torch.frexp(x.abs().amax(-1) / TOP)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(-126, 127)
    return torch.ldexp(x, -e[..., None]).float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _plain_append(s, q, k, v):
    half = s.inv_freq.numel()
    pos = s.pos.double()[s.axis.long()].t() if s.axis is not None else s.pos.double()[0][:, None]
    ang = pos * s.inv_freq  # in 64 bits: positions far out leave no digits of the angle in 32
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def turn(x, c, n):
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * n, b * c + a * n, x[..., 2 * half:]], -1)

    seq, row, base = _rows_of(s)
    at, page = base + row, s.k.shape[2]
    ids, off = s.table.long()[seq, at // page], at % page
    kc, ke = _eight(turn(k.double(), cos, sin))  # in 64 bits: values next to a border between two of e4m3
    vc, ve = _eight(v.double())
    s.k.view(torch.uint8)[ids, :, off] = kc.view(torch.uint8)
    s.v.view(torch.uint8)[ids, :, :, off] = vc.view(torch.uint8)
    s.scales[ids, :, 0, off] = ke
    s.scales[ids, :, 1, off] = ve
    return turn(q.float(), cos.float(), sin.float()).to(q.dtype)


def _plain_attend(s):
    rows, heads, dim = s.q.shape
    kv_heads, page = s.k.shape[1], s.k.shape[2]
    seqs, width = s.table.shape
    group, length, t = heads // kv_heads, width * page, s.max_rows
    ids = s.table.clamp(min=0).long()
    if s.scales is None:
        k, v = s.k[ids].float(), s.v[ids].float()
    else:
        by = torch.exp2(s.scales[ids].float() - 127)  # [seqs, width, kv_heads, 2, page]
        k = s.k.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * by[:, :, :, 0, :, None]
        v = s.v.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * by[:, :, :, 1, None, :]
    k = k.transpose(1, 2).reshape(seqs * kv_heads, length, dim)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs * kv_heads, length, dim)
    seq, row, base = _rows_of(s)
    q = torch.zeros((seqs, t, heads, dim), device=s.q.device)
    q[seq, row] = s.q.float()
    q = q.reshape(seqs, t, kv_heads, group, dim).transpose(1, 2).reshape(seqs * kv_heads, t * group, dim)
    x = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(dim))
    x = x.view(seqs, kv_heads, t, group, length)
    i = torch.full((seqs, t), -1, device=seq.device)
    j = torch.arange(length, device=seq.device)
    if s.masks is None:
        i[seq, row] = base + row
        seen = j <= i[:, :, None]
    else:  # the rows before the tree, and of the tree's what the row's mask has
        bit = torch.arange(t, device=seq.device)
        sees = (s.masks[:, None] >> bit) & 1  # [rows, t]
        i[seq, row] = base + sees.sum(1) - 1
        mine = torch.zeros((seqs, t, t), dtype=torch.bool, device=seq.device)
        mine[seq, row] = sees.bool()
        start = s.kv_len.long() - (s.cu[1:] - s.cu[:-1]).long()
        node = j - start[:, None]
        seen = mine.gather(2, node.clamp(0, t - 1)[:, None].expand(seqs, t, length)) & (node < t)[:, None]
        seen = torch.where((node < 0)[:, None], (i >= 0)[:, :, None], seen)
    seen = seen & (s.table >= 0).repeat_interleave(page, 1)[:, None]
    if s.window:
        seen &= (i[:, :, None] - j < s.window) | (j < s.sinks)
    x.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs * kv_heads, t * group, length), v).view(seqs, kv_heads, t, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).squeeze(-1)
    out = out.transpose(1, 2).reshape(seqs, t, heads, dim)[seq, row]
    return [out.to(s.q.dtype), lse.transpose(1, 2).reshape(seqs, t, heads)[seq, row]]


def _plain_accept(s):
    """int32 [seqs, 4 + 2 max_rows]: accepted drafts, tokens, 0, flags (1: a row that is not finite), the tokens, the branch's rows."""
    rows, vocab = s.target.shape
    seqs, t, dev = s.cu.numel() - 1, s.max_rows, s.target.device
    top = s.target.amax(1, keepdim=True)
    at = torch.where(s.target == top, torch.arange(vocab, device=dev), vocab).amin(1)  # ties go to the lowest token
    fine = torch.isfinite(s.target).all(1)
    n = (s.cu[1:] - s.cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(seqs, device=dev), n, output_size=rows)
    first = s.cu.long()[seq]
    row = torch.arange(rows, device=dev) - first
    up = first + s.parents.long().clamp(min=0)
    # a row follows its parent where it is the first of the children with the parent's token
    good = (row > 0) & (s.parents >= 0) & (s.tokens == at[up]) & fine[up]
    same = (up[:, None] == up) & good & (torch.arange(rows, device=dev) < torch.arange(rows, device=dev)[:, None])
    good = (good & ~same.any(1)) | (row == 0)
    # and is reached where all its ancestors do: 2^d of them by d doublings of the step up
    reach, step = good, torch.where(row == 0, torch.arange(rows, device=dev), up)
    for _ in range(6):
        reach, step = reach & reach[step], step[step]
    depth = torch.zeros((seqs, t), dtype=torch.long, device=dev)
    depth[seq, row] = reach.long()
    place = depth.cumsum(1)[seq, row] - 1  # a branch's rows rise with their depth
    out = torch.full((seqs, 4 + 2 * t), -1, dtype=torch.int32, device=dev)
    out[:, 0] = (depth.sum(1) - 1).clamp(min=0)
    wide = torch.full((seqs, t + 1), -1, dtype=torch.int32, device=dev)
    path, toks = wide, wide.clone()
    path[seq, torch.where(reach, place, t)] = row.int()
    toks[seq, torch.where(reach & fine, place, t)] = at.int()
    out[:, 4:4 + t], out[:, 4 + t:] = toks[:, :t], path[:, :t]
    out[:, 1] = (out[:, 4:4 + t] >= 0).sum(1)
    out[:, 2] = 0
    out[:, 3] = torch.zeros(seqs, dtype=torch.int32, device=dev).index_add_(0, seq, (reach & ~fine).int())
    return out


def _plain_keep(s):
    seqs, t, page = s.took.shape[0], s.max_rows, s.k.shape[3]
    base = s.kv_len.long() - (s.cu[1:] - s.cu[:-1]).long()
    path = s.took[:, 4 + t:].long()
    seq, k = torch.nonzero((path >= 0) & (torch.arange(t, device=path.device) <= s.took[:, :1]), as_tuple=True)
    src, dst = base[seq] + path[seq, k], base[seq] + k
    table = s.table.long()
    a, ao, b, bo = table[seq, src // page], src % page, table[seq, dst // page], dst % page
    bits = torch.uint8 if s.scales is not None else torch.int16
    kk, vv = s.k.view(bits), s.v.view(bits)
    kk[:, b, :, bo] = kk[:, a, :, ao]
    vv[:, b, :, :, bo] = vv[:, a, :, :, ao]
    if s.scales is not None:
        s.scales[:, b, :, :, bo] = s.scales[:, a, :, :, ao]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, lens = _sizes(case)
    total = sum(rows)
    if case["op"] == "accept":
        return dict(bytes=total * case["vocab"] * 4 + 8 * total + 4 * case["seqs"] * (4 + 2 * max(rows)), flops=0)
    kv_heads, dim, size = case["kv_heads"], case["dim"], 1 if case.get("type", "e4m3") == "e4m3" else 2
    extra = 2 if size == 1 else 0  # scales of a token and head
    if case["op"] == "keep":  # a branch of some log2(rows) tokens
        moved = sum(max(1, round(math.log2(n + 1)) - 1) for n in rows)
        return dict(bytes=2 * moved * case["layers"] * kv_heads * (2 * dim * size + extra), flops=0)
    heads = case["heads"]
    if case["op"] == "append":
        return dict(bytes=total * (2 * heads + 2 * kv_heads) * dim * 2 + total * kv_heads * (2 * dim + 2)
                    + 4 * total * case["axes"], flops=3 * total * (heads + kv_heads) * case["rot"] + 4 * total * kv_heads * dim)
    tokens = pairs = 0
    for r, n in zip(rows, lens):
        w, k = case["window"] or n, case["sinks"]
        tokens += n - max(0, n - r - w + 1) + min(k, max(0, n - r - w + 1))
        if case["op"] == "tree":
            pairs += r * (min(n - r, w + k) + 1)
        else:  # the row at position i sees i + 1 tokens, of them at most w near ones and the k first
            free = max(0, min(n, w + k) - (n - r))
            pairs += free * (n - r) + free * (free + 1) // 2 + (r - free) * (w + k)
    return dict(bytes=tokens * kv_heads * (2 * dim * size + extra) + 2 * total * heads * dim * 2 + 4 * total * heads,
                flops=4 * pairs * dim * heads)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    op = case["op"]
    if op == "accept":
        return None  # whole numbers: no values in 64 bits
    s = prepare(case, seed)
    cu, lens, page = s.cu.tolist(), s.kv_len.tolist(), case["page"]
    if op == "keep":
        if s.k.numel() > 1.5e9:
            return None
        k, v = s.k.double(), s.v.double()
        took, table = s.took.tolist(), s.table.tolist()
        for b, n in enumerate(lens):
            base = n - (cu[b + 1] - cu[b])
            for i in range(took[b][0] + 1):
                x, y = base + took[b][4 + s.max_rows + i], base + i
                k[:, table[b][y // page], :, y % page] = s.k[:, table[b][x // page], :, x % page].double()
                v[:, table[b][y // page], :, :, y % page] = s.v[:, table[b][x // page], :, :, x % page].double()
        return [k, v] + ([None] if s.scales is not None else [])
    if op == "append":
        half, heads, kv_heads = case["rot"] // 2, case["heads"], case["kv_heads"]
        out = s.qkv.double()
        for i in range(half):
            p = s.pos[int(s.axis[i]) if s.axis is not None else 0].double() * float(s.inv_freq[i])
            z = torch.polar(torch.ones_like(p), p)[:, None] * torch.complex(out[:, :heads + kv_heads, i], out[:, :heads + kv_heads, half + i])
            out[:, :heads + kv_heads, i], out[:, :heads + kv_heads, half + i] = z.real, z.imag
        k, v = s.k.double(), s.v.double()
        by = torch.exp2(torch.ceil(torch.log2(out[:, heads:].abs().amax(2, keepdim=True) / TOP)))
        eight = out[:, heads:] / by
        for b, n in enumerate(lens):
            at = torch.arange(n - (cu[b + 1] - cu[b]), n, device=DEV)
            pages = s.table[b].long()[torch.div(at, page, rounding_mode="floor")]
            mine = eight[cu[b]:cu[b + 1]]
            k[pages, :, at % page] = mine[:, :kv_heads]
            v[pages, :, :, at % page] = mine[:, kv_heads:]
        return [out[:, :heads], k, v, None]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if 4 * dim * heads * sum(r * n for r, n in zip(*_sizes(case))) > 4e13:
        return None
    group = heads // kv_heads
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        base = n - (hi - lo)
        held = s.table[b].long()
        w = torch.nonzero(held >= 0)[:, 0]
        j = (w[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
        for h in range(kv_heads):
            kk = s.k[:, h].view(torch.uint8 if s.scales is not None else torch.int16)[held[w]].view(s.k.dtype).double()
            vv = s.v[:, h].view(torch.uint8 if s.scales is not None else torch.int16)[held[w]].view(s.v.dtype).double()
            if s.scales is not None:
                e = s.scales[held[w], h].double() - 127
                kk, vv = kk * 2.0 ** e[:, 0, :, None], vv * 2.0 ** e[:, 1, None, :]
            kk, vv = kk.reshape(-1, dim)[j < n], vv.transpose(1, 2).reshape(-1, dim)[j < n]
            t = j[j < n]
            for c in range(lo, hi, 1024):
                e = min(hi, c + 1024)
                q = s.q[c:e, h * group:(h + 1) * group].double().reshape(-1, dim)
                if s.masks is None:
                    i = torch.arange(base + c - lo, base + e - lo, device=DEV)[:, None]
                    seen = t <= i
                else:
                    sees = torch.tensor([[(m >> x) & 1 for x in range(hi - lo)] for m in s.masks[c:e].tolist()], device=DEV)
                    i = base + sees.sum(1, keepdim=True) - 1
                    seen = torch.cat([torch.ones(e - c, base, dtype=torch.bool, device=DEV), sees.bool()], 1)[:, t]
                if case["window"]:
                    seen = seen & ((i - t < case["window"]) | (t < case["sinks"]))
                x = (q @ kk.t() / math.sqrt(dim)).masked_fill_(~seen.repeat_interleave(group, 0), -math.inf)
                z = torch.logsumexp(x, 1)
                lse[c:e, h * group:(h + 1) * group] = z.view(-1, group)
                out[c:e, h * group:(h + 1) * group] = (torch.softmax(x, 1) @ vv).view(-1, group, dim)
    return [out, lse]

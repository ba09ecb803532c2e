"""Attention over a paged key-value cache, as cases that can be timed and compared.

Four operators that work on one cache: `rope` turns the query and key rows by their positions (one axis for text, three
for images and video) and writes key and value rows into the cache's pages; `attend` is the attention of a batch's new
rows over those pages, from one token of one sequence to whole prompt chunks, with a causal mask, an optional sliding
window and first tokens that stay visible; `move` copies pages (a fork's open pages, a compaction with its tables).

The cache of a layer: keys [pages, kv heads, page, dim], values [pages, kv heads, dim, page]. A batch: `cu` int32
[seqs + 1] (the rows of sequence s are cu[s] .. cu[s + 1]), `kv_len` int32 [seqs] (its tokens in the cache, the new rows
the last of them), `table` int32 [seqs, width] (the page of its tokens page * w ..; -1 where none is held).
With `own` false, `run` is the plain form in elementary torch operations; with `own` true the package's entry points.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # The new token's rows of 64 chats: angles, turned rows and 64 single rows into 64 pages.
        dict(name="rope_decode_64", op="rope", type="bf16", seqs=64, rows=1, length=4096, heads=32, kv_heads=4, dim=128,
             rot=128, axes=1, page=64, ragged=True),
        # A prompt with images: three position axes over a quarter of a wide head, chunks that begin inside a page.
        dict(name="rope_prompt_axes", op="rope", type="bf16", seqs=2, rows=4095, length=6001, heads=16, kv_heads=2, dim=256,
             rot=64, axes=3, page=64, ragged=False),
        # One token of one short chat: nothing but latency.
        dict(name="decode_one", op="attend", type="bf16", seqs=1, rows=1, length=777, heads=32, kv_heads=4, dim=128,
             window=0, sinks=0, page=64, ragged=False),
        # The verify rows of depth-2 speculation (one pending token, two drafts) of eight chats.
        dict(name="verify_t3", op="attend", type="bf16", seqs=8, rows=3, length=6145, heads=16, kv_heads=2, dim=256,
             window=0, sinks=0, page=64, ragged=True),
        # One token after a context of the longest supported size.
        dict(name="decode_long", op="attend", type="bf16", seqs=1, rows=1, length=131072, heads=32, kv_heads=4, dim=128,
             window=0, sinks=0, page=64, ragged=False),
        # A full serving batch of single tokens, lengths mixed.
        dict(name="decode_batch", op="attend", type="bf16", seqs=64, rows=1, length=16384, heads=32, kv_heads=8, dim=128,
             window=0, sinks=0, page=64, ragged=True),
        # Depth-3 verify rows of long chats that keep a window and the first tokens only; small pages, narrow heads.
        dict(name="verify_window", op="attend", type="fp16", seqs=32, rows=4, length=40000, heads=24, kv_heads=8, dim=64,
             window=1024, sinks=4, page=16, ragged=True),
        # The next turns of a few chats over what their caches hold.
        dict(name="prompt_turns", op="attend", type="bf16", seqs=3, rows=333, length=5000, heads=32, kv_heads=4, dim=128,
             window=0, sinks=0, page=64, ragged=True),
        # The default prompt chunk from an empty cache.
        dict(name="prompt_2048", op="attend", type="bf16", seqs=1, rows=2048, length=2048, heads=32, kv_heads=4, dim=128,
             window=0, sinks=0, page=64, ragged=False),
        # A long chunk behind a longer context under a sliding window with sinks.
        dict(name="prompt_window", op="attend", type="bf16", seqs=1, rows=8191, length=12000, heads=32, kv_heads=8, dim=128,
             window=4096, sinks=16, page=64, ragged=False),
        # The open pages of 48 forked sequences, every attention layer of them.
        dict(name="fork_48", op="move", type="bf16", layers=12, pages=2048, moved=48, kv_heads=4, dim=128, page=64,
             seqs=0, width=0),
        # A pool that shrinks: a third of its pages go to lower ids, the tables follow.
        dict(name="compact", op="move", type="bf16", layers=12, pages=1500, moved=500, kv_heads=4, dim=128, page=64,
             seqs=64, width=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "attend", "move"])
    heads, kv_heads, dim = rng.choice([(32, 4, 128), (32, 8, 128), (16, 2, 256), (24, 8, 64), (20, 4, 128), (10, 2, 64),
                                       (16, 1, 128), (8, 8, 64), (9, 3, 128), (6, 2, 256)])
    shape = dict(type=rng.choice(["bf16", "bf16", "fp16"]), kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 64, 128, 256]))
    if op == "move":
        pages = _log_int(rng, 40, 6000 * 8192 // (shape["page"] * kv_heads * dim))
        return dict(op=op, layers=_log_int(rng, 1, 12), pages=pages, moved=_log_int(rng, 1, pages // 3),
                    seqs=rng.choice([0, rng.randint(1, 64)]), width=_log_int(rng, 4, 600), **shape)
    shape.update(heads=heads, ragged=rng.random() < 0.6)
    kind = rng.choice(["single", "few", "prompt", "prompt"])
    if op == "rope":
        rows = {"single": 1, "few": rng.randint(2, 8)}.get(kind) or _log_int(rng, 9, 4000)
        seqs = _log_int(rng, 1, 200 if rows < 9 else max(1, 8000 // rows))
        return dict(op=op, seqs=seqs, rows=rows, length=rows + _log_int(rng, 1, 4000) - 1, axes=rng.choice([1, 1, 3]),
                    rot=rng.choice([dim, dim, dim // 2, dim // 4]), **shape)
    shape.update(rng.choice([dict(window=0, sinks=0), dict(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 4, 17]))]))
    if kind == "prompt":
        length = _log_int(rng, 9, 12000)
        rows = min(length, _log_int(rng, 9, 4000))
        rows = min(rows, max(9, int(1.3e11 / (heads * dim * length))))
        return dict(op=op, seqs=max(1, min(_log_int(rng, 1, 16), int(1.3e11 / (heads * dim * rows * length)))), rows=rows,
                    length=length, **shape)
    length = _log_int(rng, 9, 100000)
    seqs = max(1, min(_log_int(rng, 1, 128), int(6e8 / (length * kv_heads * dim))))
    return dict(op=op, seqs=seqs, rows=1 if kind == "single" else rng.randint(2, 8), length=length, **shape)


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
        n = case["rows"] if case["rows"] <= 8 else max(1, round(case["rows"] * f))
        rows.append(n)
        lens.append(max(n, round(case["length"] * f)))
    return rows, lens


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, seed, dtype):
    return torch.randn(shape, generator=_gen(seed), device=DEV, dtype=dtype)


def prepare(case, seed):
    seed, dtype, page = int(seed) * 1000 + 29, TYPES[case["type"]], case["page"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "move":
        n = case["pages"]
        perm = torch.randperm(n, generator=_gen(seed + 1), device=DEV).to(torch.int32)
        m = case["moved"]
        src, dst = perm[:m].contiguous(), perm[m:2 * m].contiguous()
        table = None
        if case["seqs"]:  # live pages, some of which move; a fifth of the places are empty
            live = torch.cat([perm[:m], perm[2 * m:]])
            at = torch.randint(0, live.numel(), (case["seqs"], case["width"]), generator=_gen(seed + 2), device=DEV)
            table = live[at].contiguous()
            table[torch.rand(table.shape, generator=_gen(seed + 3), device=DEV) < 0.2] = -1
        return State(k=_normal((case["layers"], n, kv_heads, page, dim), seed + 4, dtype),
                     v=_normal((case["layers"], n, kv_heads, dim, page), seed + 5, dtype), src=src, dst=dst, table=table)
    rows, lens = _sizes(case)
    seqs, total = case["seqs"], sum(rows)
    width = -(-max(lens) // page) + 1
    need = [-(-n // page) for n in lens]
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    first = [0] * seqs
    if case.get("window"):  # pages wholly behind the window of the first new row are not held, but for the first tokens'
        first = [max(0, n - r - case["window"] + 1) // page for r, n in zip(rows, lens)]
    held = [[w for w in range(need[s]) if w >= first[s] or w * page < case["sinks"]] for s in range(seqs)]
    pages = sum(len(h) for h in held) + 3
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    at = 0
    for s, h in enumerate(held):
        table[s, torch.tensor(h, dtype=torch.long)] = ids[at:at + len(h)]
        at += len(h)
    cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    batch = dict(cu=cu.to(DEV), kv_len=torch.tensor(lens, dtype=torch.int32).to(DEV), table=table.to(DEV),
                 max_rows=max(rows), rows=total, window=case.get("window", 0), sinks=case.get("sinks", 0))
    k = _normal((pages, kv_heads, page, dim), seed + 2, dtype)
    v = _normal((pages, kv_heads, dim, page), seed + 3, dtype)
    if case["op"] == "attend":
        return State(q=_normal((total, case["heads"], dim), seed + 4, dtype) * 1.5, k=k, v=v, **batch)
    # the rows of a fused projection: query, key and value heads side by side
    qkv = _normal((total, case["heads"] + 2 * kv_heads, dim), seed + 4, dtype)
    half = case["rot"] // 2
    inv_freq = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
    pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lens)])
    axis = None
    if case["axes"] > 1:  # frames of 24 x 16 patches: time, then rows and columns; the axes alternate over frequencies
        patch = pos % 384
        pos = torch.stack([pos // 384, patch // 16, patch % 16])
        axis = (torch.arange(half) % case["axes"]).to(torch.int32).to(DEV)
    return State(qkv=qkv, k=k, v=v, pos=pos.reshape(case["axes"], total).to(torch.int32).to(DEV), axis=axis,
                 inv_freq=inv_freq.to(DEV), **batch)


# ---------------------------------------------------------------- one pass
def run(s):
    if hasattr(s, "src"):
        if own:
            from slotstream_spark_amd.kernels.kv_pages import move_pages
            move_pages(s.k, s.v, s.src, s.dst, table=s.table)
        else:
            _plain_move(s)
        return [s.k, s.v] + ([s.table] if s.table is not None else [])
    if hasattr(s, "qkv"):
        h, n = s.k.shape[1], s.qkv.shape[1]
        q, k, v = s.qkv[:, :n - 2 * h], s.qkv[:, n - 2 * h:n - h], s.qkv[:, n - h:]
        if own:
            from slotstream_spark_amd.kernels.rope import rope_append
            out = rope_append(q, k, v, s.pos, s.inv_freq, s.k, s.v, s.cu, s.kv_len, s.table, s.max_rows, axis=s.axis)
        else:
            out = _plain_rope(s, q, k, v)
        return [out, s.k, s.v]
    if own:
        from slotstream_spark_amd.kernels.paged_attention import paged_attention
        lse = torch.empty(s.q.shape[:2], dtype=torch.float32, device=s.q.device)
        out = paged_attention(s.q, s.k, s.v, s.cu, s.kv_len, s.table, s.max_rows, window=s.window, sinks=s.sinks, lse=lse)
        return [out, lse]
    return _plain_attend(s)


def _plain_move(s):
    src, dst = s.src.long(), s.dst.long()
    s.k[:, dst] = s.k[:, src]
    s.v[:, dst] = s.v[:, src]
    if s.table is not None:
        new = torch.arange(s.k.shape[1], device=src.device, dtype=torch.int32)
        new[src] = s.dst
        s.table.copy_(torch.where(s.table >= 0, new[s.table.clamp(min=0).long()], s.table))


def _rows_of(s):
    """Of every row: its sequence and its token's position in the cache."""
    n = (s.cu[1:] - s.cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=n.device), n, output_size=s.rows)
    return seq, s.kv_len.long()[seq] - s.cu[1:].long()[seq] + torch.arange(s.rows, device=n.device)


def _plain_rope(s, q, k, v):
    half = s.inv_freq.numel()
    pos = s.pos.double()[s.axis.long()].t() if s.axis is not None else s.pos.double()[0][:, None]
    ang = pos * s.inv_freq  # in 64 bits: positions far out leave no digits of the angle in 32
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def turn(x):
        x = x.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    seq, at = _rows_of(s)
    page = s.k.shape[2]
    ids, off = s.table.long()[seq, at // page], at % page
    s.k[ids, :, off] = turn(k).to(s.k.dtype)
    s.v[ids, :, :, off] = v
    return turn(q).to(q.dtype)


def _plain_attend(s):
    rows, heads, dim = s.q.shape
    kv_heads, page = s.k.shape[1], s.k.shape[2]
    seqs, width = s.table.shape
    group, length, t = heads // kv_heads, width * page, s.max_rows
    ids = s.table.clamp(min=0).long()
    k = s.k[ids].transpose(1, 2).reshape(seqs * kv_heads, length, dim).float()
    v = s.v[ids].permute(0, 2, 1, 4, 3).reshape(seqs * kv_heads, length, dim).float()
    seq, at = _rows_of(s)
    row = torch.arange(rows, device=seq.device) - s.cu.long()[seq]
    q = torch.zeros((seqs, t, heads, dim), device=s.q.device)
    q[seq, row] = s.q.float()
    q = q.reshape(seqs, t, kv_heads, group, dim).transpose(1, 2).reshape(seqs * kv_heads, t * group, dim)
    x = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(dim))
    x = x.view(seqs, kv_heads, t, group, length)
    i = torch.full((seqs, t), -1, device=seq.device)
    i[seq, row] = at
    i, j = i[:, :, None], torch.arange(length, device=seq.device)
    seen = (j <= i) & (s.table >= 0).repeat_interleave(page, 1)[:, None]
    if s.window:
        seen &= (i - j < s.window) | (j < s.sinks)
    x.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs * kv_heads, t * group, length), v).view(seqs, kv_heads, t, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).squeeze(-1)
    out = out.transpose(1, 2).reshape(seqs, t, heads, dim)[seq, row]
    return [out.to(s.q.dtype), lse.transpose(1, 2).reshape(seqs, t, heads)[seq, row]]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kv_heads, dim, size = case["kv_heads"], case["dim"], 2
    if case["op"] == "move":
        one = case["layers"] * 2 * kv_heads * case["page"] * dim * size
        return dict(bytes=2 * case["moved"] * one + 2 * 4 * case["seqs"] * case["width"] + 8 * case["moved"], flops=0)
    rows, lens = _sizes(case)
    total, heads = sum(rows), case["heads"]
    if case["op"] == "rope":
        return dict(bytes=2 * total * (heads + 2 * kv_heads) * dim * size + 4 * total * case["axes"],
                    flops=3 * total * (heads + kv_heads) * case["rot"])
    tokens = pairs = 0
    for r, n in zip(rows, lens):
        w, k = case["window"] or n, case["sinks"]
        tokens += n - max(0, n - r - w + 1) + min(k, max(0, n - r - w + 1))
        # the row at position i sees i + 1 tokens, of them at most w near ones and the k first
        free = max(0, min(n, w + k) - (n - r))  # rows whose whole past is visible
        pairs += free * (n - r) + free * (free + 1) // 2 + (r - free) * (w + k)
    return dict(bytes=tokens * 2 * kv_heads * dim * size + 2 * total * heads * dim * size + 4 * total * heads,
                flops=4 * pairs * dim * heads)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "move":
        k, v = s.k.clone(), s.v.clone()
        for layer in range(case["layers"]):
            k[layer].index_copy_(0, s.dst.long(), s.k[layer].index_select(0, s.src.long()))
            v[layer].index_copy_(0, s.dst.long(), s.v[layer].index_select(0, s.src.long()))
        if s.table is None:
            return [k, v]
        to = dict(zip(s.src.tolist(), s.dst.tolist()))
        return [k, v, torch.tensor([[to.get(p, p) for p in row] for row in s.table.tolist()], dtype=torch.int32)]
    cu, lens, page = s.cu.tolist(), s.kv_len.tolist(), case["page"]
    if case["op"] == "rope":
        half, heads, kv_heads = case["rot"] // 2, case["heads"], case["kv_heads"]
        out = s.qkv.double()
        for i in range(half):
            p = s.pos[int(s.axis[i]) if s.axis is not None else 0].double() * float(s.inv_freq[i])
            z = torch.polar(torch.ones_like(p), p)[:, None] * torch.complex(out[:, :heads + kv_heads, i], out[:, :heads + kv_heads, half + i])
            out[:, :heads + kv_heads, i], out[:, :heads + kv_heads, half + i] = z.real, z.imag
        k, v = s.k.double(), s.v.double()
        for b, n in enumerate(lens):
            at = torch.arange(n - (cu[b + 1] - cu[b]), n, device=DEV)
            pages = s.table[b].long()[torch.div(at, page, rounding_mode="floor")]
            mine = out[cu[b]:cu[b + 1]]
            k[pages, :, at % page] = mine[:, heads:heads + kv_heads]
            v[pages, :, :, at % page] = mine[:, heads + kv_heads:]
        return [out[:, :heads], k, v]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        for h in range(kv_heads):
            held = s.table[b].long()
            w = torch.nonzero(held >= 0)[:, 0]
            j = (w[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
            kk = s.k[held[w], h].reshape(-1, dim)[j < n].double()
            vv = s.v[held[w], h].transpose(1, 2).reshape(-1, dim)[j < n].double()
            j = j[j < n]
            for c in range(lo, hi, 2048):
                e = min(hi, c + 2048)
                q = s.q[c:e, h * group:(h + 1) * group].double().reshape(-1, dim)
                i = torch.arange(n - hi + c, n - hi + e, device=DEV).repeat_interleave(group)[:, None]
                seen = j <= i
                if case["window"]:
                    seen &= (i - j < case["window"]) | (j < case["sinks"])
                x = (q @ kk.t() / math.sqrt(dim)).masked_fill_(~seen, -math.inf)
                z = torch.logsumexp(x, 1)
                lse[c:e, h * group:(h + 1) * group] = z.view(-1, group)
                out[c:e, h * group:(h + 1) * group] = (torch.softmax(x, 1) @ vv).view(-1, group, dim)
    return [out, lse]

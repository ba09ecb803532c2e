"""The attention operators as they are used together: a cache with its sequences, the attention layer over it, the draft head
with its attention, and the speculative loop over a stack with attention layers."""
import math

import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.attention import SeqCache
from slotstream_spark_amd.engine.generate import MoEStack, mtp_decode
from slotstream_spark_amd.engine.mtp import DraftGraph, HeadAttention, MTPHead
from slotstream_spark_amd.engine.step import MoEWeights
from slotstream_spark_amd.engine.verify import MoEVerifyLayer
from slotstream_spark_amd.kernels.gemv_affine import AffineWeight
from slotstream_spark_amd.kernels.paged_attention import paged_attention
from slotstream_spark_amd.memory.kv_pages import KVPages
from slotstream_spark_amd.memory.synth import LayerWeights, attention_layer, head_weights, normal_bf16
from tests.gpu_util import make_pool

pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.int16)


def layer64(layer, x, pos, window=0, sinks=0):
    """The layer over one whole sequence in 64 bits without roundings: (y, the largest score)."""
    h, kv, d = layer.heads, layer.kv_heads, layer.dim
    qkv = (x.double() @ layer.wqkv.double().t()).view(-1, h + 2 * kv, d)
    q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    if layer.qk_norm is not None:
        n = layer.qk_norm.double().view(h + kv, d)
        norm = lambda t, w: t / torch.sqrt(t.square().mean(-1, keepdim=True) + layer.eps) * w  # noqa: E731
        q, k = norm(q, n[:h]), norm(k, n[h:])
    half = layer.inv_freq.numel()
    a = pos.double()[:, None] * layer.inv_freq
    c, s = a.cos()[:, None], a.sin()[:, None]

    def turn(t):
        return torch.cat([t[..., :half] * c - t[..., half:2 * half] * s, t[..., half:2 * half] * c + t[..., :half] * s,
                          t[..., 2 * half:]], -1)

    q, k = turn(q), turn(k).repeat_interleave(h // kv, 1)
    v = v.repeat_interleave(h // kv, 1)
    x = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / math.sqrt(d)
    i, j = torch.arange(len(pos), device=pos.device)[:, None], torch.arange(len(pos), device=pos.device)
    see = j <= i
    if window:
        see &= (i - j < window) | (j < sinks)
    x = x.masked_fill(~see, -math.inf)
    o = torch.matmul(x.softmax(-1), v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(len(pos), h * d)
    return o @ layer.wo.double().t(), x[x.isfinite()].abs().max().item()


@pytest.mark.parametrize("heads,kv_heads,dim,norms,window,sinks", [(8, 2, 128, False, 0, 0), (16, 4, 64, True, 0, 0),
                                                                  (4, 1, 256, True, 40, 5)])
def test_prompt_then_tokens(heads, kv_heads, dim, norms, window, sinks):
    """A prompt in one chunk, then rounds of three rows and single tokens: every row against the definition in 64 bits."""
    H, n = 512, 150
    layer = attention_layer(H, heads, kv_heads, dim, 3, rot=dim // 2, norms=norms, window=window, sinks=sinks)
    x = normal_bf16((n, H), 1.0, 4)
    cache = SeqCache(KVPages(1, 20, kv_heads, dim, 32, max_tokens=400))
    ys, at = [], 0
    for rows in [100, 3, 3, 1, 1, 1, 30, 8, 1, 2]:
        cache.place(at, rows)
        cu, kv_len, table, positions = cache.rows(rows)
        ys.append(layer(x[at:at + rows].contiguous(), positions, cache.pages.k[0], cache.pages.v[0], cu, kv_len, table, rows))
        at += rows
    assert at == n
    got = torch.cat(ys).double()
    want, score = layer64(layer, x, torch.arange(n, device="cuda"), window, sinks)
    # Roundings to bf16 along the way (half steps 2^-8): the projection, the turned rows, the probabilities, the head outputs
    # and the result, and that of q and k moves a score by up to 2 half steps (twice, projection and turn; with norms once
    # more), its probability by as much relative.
    tol = (5 + 2 * (3 if norms else 2) * score) * 2.0 ** -8
    assert ((got - want).norm(dim=1) <= tol * want.norm(dim=1)).all()
    assert _lib.device_error() == 0


def test_rounds_equal_single_tokens_bit_for_bit():
    """Layer output and cache: three-row calls against one-row calls, and a round that is taken back and run again."""
    H = 512
    layer = attention_layer(H, 8, 2, 128, 5)
    x = normal_bf16((40, H), 1.0, 6)

    def run(steps):
        cache = SeqCache(KVPages(1, 10, 2, 128, 16, max_tokens=160))
        out = {}
        for at, rows in steps:
            cache.place(at, rows)
            cu, kv_len, table, positions = cache.rows(rows)
            y = layer(x[at:at + rows].contiguous(), positions, cache.pages.k[0], cache.pages.v[0], cu, kv_len, table, rows)
            out.update({at + i: y[i].clone() for i in range(rows)})
        return torch.stack([out[i] for i in range(36)])

    one = run([(i, 1) for i in range(36)])
    three = run([(i, 3) for i in range(0, 36, 3)])
    back = run([(0, 4)] + [s for i in range(1, 36, 2) for s in ((i, 3), (i, 2))])
    assert torch.equal(bits(one), bits(three)) and torch.equal(bits(one), bits(back))


def test_fork_compact_and_resize_between_steps():
    """Two continuations of one prompt in a fork, with compaction and shrinking between: the bits of undisturbed runs."""
    H, page = 512, 16
    layer = attention_layer(H, 8, 2, 64, 7)
    prompt, tails = normal_bf16((45, H), 1.0, 8), [normal_bf16((20, H), 1.0, 9 + i) for i in range(2)]

    def step(kv, seq, x):
        at = kv.length[seq]
        kv.extend(seq, x.shape[0])
        cu = torch.tensor([0, x.shape[0]], dtype=torch.int32, device="cuda")
        kv_len = torch.tensor([at + x.shape[0]], dtype=torch.int32, device="cuda")
        positions = torch.arange(at, at + x.shape[0], dtype=torch.int32, device="cuda")
        return layer(x, positions, kv.k[0], kv.v[0], cu, kv_len, kv.table[seq:seq + 1], x.shape[0])

    def pages(n):
        return KVPages(2, n, 2, 64, page, max_seqs=4, max_tokens=128)

    want = []
    for tail in tails:
        kv = pages(8)
        s = kv.new()
        step(kv, s, prompt)
        want.append([step(kv, s, tail[i:i + 1].contiguous()) for i in range(20)])
    kv = pages(40)
    junk = kv.new()
    kv.extend(junk, 100)                       # takes the low ids, so that freeing it leaves holes below
    a = kv.new()
    step(kv, a, prompt)
    b = kv.fork(a)
    kv.free(junk)
    got = [[], []]
    for i in range(20):
        for j, s in enumerate((a, b)):
            got[j].append(step(kv, s, tails[j][i:i + 1].contiguous()))
        if i == 6:
            assert kv.compact() == int((kv._refs > 0).sum())
            assert max(kv.pages_of(a) + kv.pages_of(b)) < 7
        if i == 12:
            kv.resize(12)
        assert torch.equal(kv.table.cpu(), torch.from_numpy(kv._table))
    for j in range(2):
        assert all(torch.equal(bits(p), bits(q)) for p, q in zip(got[j], want[j])), j
    assert _lib.device_error() == 0


def test_evicted_pages_do_not_change_a_window():
    H = 512
    layer = attention_layer(H, 8, 2, 64, 11, window=50, sinks=4)
    x = normal_bf16((140, H), 1.0, 12)

    def run(evict):
        cache, out = SeqCache(KVPages(1, 12, 2, 64, 16, max_tokens=192)), []
        for at in range(0, 140, 2):
            cache.place(at, 2)
            cu, kv_len, table, positions = cache.rows(2)
            out.append(layer(x[at:at + 2].contiguous(), positions, cache.pages.k[0], cache.pages.v[0], cu, kv_len, table, 2))
            if evict:
                cache.pages.evict(cache.seq, 50, 4, back=2)
        return torch.cat(out), cache.pages.free_pages

    (a, n_a), (b, n_b) = run(False), run(True)
    assert torch.equal(bits(a), bits(b)) and n_b > n_a and _lib.device_error() == 0


# ---------------------------------------------------------------- the draft head and the loop
H, I, E, K, NL, V, D = 2048, 512, 64, 4, 2, 4096, 2


def lm_head(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-2**31, 2**31 - 1, (V, H // 8), generator=g, device="cuda", dtype=torch.int32)
    sc = (torch.randn((V, H // 64), generator=g, device="cuda") * 0.02).abs().to(torch.bfloat16)
    return AffineWeight(q, sc, (-8 * sc.float()).to(torch.bfloat16), 4, 64, V, H)


@pytest.fixture(scope="module")
def parts():
    pool = make_pool(E, H, I, seed=900, layers=NL + 1)
    lws = [LayerWeights(H, E, 512, seed=901 + l) for l in range(NL + 1)]
    return pool, lws, lm_head(920)


def make_head(parts, hc, max_tokens=64):
    pool, lws, lm = parts
    w = lws[NL]
    hw = head_weights(H, hc, 32, V, seed=921)
    moe = MoEVerifyLayer(pool, NL, w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g, top_k=K, max_tokens=4)
    attn = HeadAttention(head_weights(H, hc, 32, 64, seed=923).mlp_hc, attention_layer(H, 16, 4, 64, 924),
                         KVPages(1, 8, 4, 64, 16, max_tokens=max_tokens))
    return MTPHead(hw, moe, lm, hc=hc, max_ctx=64, attn=attn)


@pytest.mark.parametrize("hc", [1, 4])
def test_head_with_attention(parts, hc):
    """Drafts depend on what was consumed, chunked consumption equals consumption token by token, drafting leaves no trace,
    and the captured drafts equal the eager ones as the head's state moves."""
    ids = [5, 77, 300, 1024, 9, 2000, 31]
    multi = normal_bf16((len(ids), hc * H), 1.0, 930)
    a, b, other = make_head(parts, hc), make_head(parts, hc), make_head(parts, hc)
    a.consume(ids, multi)
    for i in range(len(ids)):
        b.consume(ids[i:i + 1], multi[i:i + 1])
    other.consume([6] + ids[1:], multi.flip(0).contiguous())
    other.prev_multi = multi[-1:].clone()
    n = len(ids) - 1                         # the cache's rows so far
    for got, want in ((a.attn.pages.k, b.attn.pages.k), (a.attn.pages.v, b.attn.pages.v)):
        assert torch.equal(bits(got[0][0]), bits(want[0][0])) and n <= 16
    drafts = a.draft(42, 3)
    assert drafts == b.draft(42, 3) == a.draft(42, 3)
    assert torch.isfinite(a.draft_rows(3).out.float()).all()
    other.draft(42, 3)
    assert not torch.equal(a.draft_rows(3).out, other.draft_rows(3).out)    # the attended past differs
    graph = DraftGraph(a, 3)
    for step in range(4):
        graph.token.fill_(42 + step)
        graph.multi.copy_(a.prev_multi)
        got = graph.replay().cpu().tolist()
        assert got == a.draft(42 + step, 3), step
        a.consume([42 + step], normal_bf16((1, hc * H), 1.0, 940 + step))
    a.reset()
    a.consume(ids, multi)
    assert a.draft(42, 3) == drafts
    assert _lib.device_error() == 0


def make_stack(parts, prompt_chunk=0, max_tokens=96, window=0):
    pool, lws, lm = parts
    mw = [MoEWeights(w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g) for w in lws[:NL]]
    norms = [normal_bf16((H,), 0.1, 950 + l).float().add(1).to(torch.bfloat16) for l in range(NL + 1)]
    attn = [attention_layer(H, 16, 4, 64, 960 + l, window=window, sinks=2 if window else 0) for l in range(NL)]
    return MoEStack(pool, mw, lm, head_weights(H, 1, 32, V, seed=921).embed, depth=D, norm_weights=norms, top_k=K,
                    attn=attn, attn_norms=norms[:NL], pages=KVPages(NL, 8, 4, 64, 16, max_tokens=max_tokens),
                    prompt_chunk=prompt_chunk)


@pytest.mark.parametrize("prompt_chunk,window", [(0, 0), (16, 0), (16, 7)])
def test_loop_with_attention_emits_the_plain_sequence(parts, prompt_chunk, window):
    """With the head's drafts, with right, wrong and mixed ones, the loop emits what one-token steps emit, through rollbacks
    that leave rejected rows in the cache; and the sequence depends on the prompt's earlier tokens."""
    stack, head = make_stack(parts, prompt_chunk, window=window), make_head(parts, 1)
    prompt, n = [5, 17, 300, 8, 1234, 77, 9, 9, 2, 64, 1000, 41, 3, 50, 11, 600, 23, 90, 4], 24

    def plain(p):
        stack.reset()
        out = [stack.prompt(p)[0][-1]]
        while len(out) < n:
            out.append(stack.forward([out[-1]])[0][0])
        return out

    want, other = plain(prompt), plain([6] + prompt[1:])
    assert want != other
    assert len(set(want)) > 4

    def drafts_of(mode):
        def fn(pending, depth, n_out):
            right = (want + [0] * depth)[n_out:n_out + depth]
            wrong = [(t + 1) % V for t in right]
            return {"right": right, "wrong": wrong, "mixed": right if n_out % 2 else [right[0], wrong[1]]}[mode]
        return fn

    for mode in ("head", "right", "wrong", "mixed"):
        stack.reset()
        head.reset()
        out, nan, _, st = mtp_decode(stack, head, prompt, n, draft_fn=None if mode == "head" else drafts_of(mode))
        assert out == want and not nan, mode
        assert stack.st.pos == len(prompt) + n - 1 == stack.st.attn["cache"].pos or mode == "head"
        assert head.state.aligned(head.consumed) and head.consumed == stack.st.pos
    assert _lib.device_error() == 0


def test_loop_near_the_end_of_the_pages(parts):
    stack, head = make_stack(parts, max_tokens=16), make_head(parts, 1, max_tokens=16)
    assert stack.max_ctx == 16 - 3
    out, nan, _, st = mtp_decode(stack, head, [42, 7], 40)
    assert not nan and st["plain_steps"] > 0 and stack.st.pos <= 13
    stack.reset()
    tok = stack.forward([42, 7])[0][-1]
    plain = [tok]
    while len(plain) < len(out):
        plain.append(stack.forward([plain[-1]])[0][0])
    assert out == plain


def test_prompt_forms_agree(parts):
    """The stack's rows of a prompt through the prompt layers against those through the verify layers: the same model within
    the roundings: five of a layer to bf16 (half steps 2^-8; two layers) in another order of sums. A router's near tie may send
    a row to another expert, so the median row is held to it."""
    a, b = make_stack(parts, 0), make_stack(parts, 64)
    tokens = [(37 * i + 5) % V for i in range(40)]
    (na, ma), (nb, mb) = a.prompt(tokens), b.prompt(tokens)
    err = ((ma.double() - mb.double()).norm(dim=1) / ma.double().norm(dim=1)).sort().values
    assert err[len(err) // 2] <= 10 * 2.0 ** -8 and len(nb) == 1
    with pytest.raises(ValueError, match="attn and pages"):
        MoEStack(a.graph.layers[0].pool, [], None, a.embed, attn=[])


def test_refused_stacks_and_prompts(parts):
    pool, lws, lm = parts
    pages = KVPages(NL, 4, 4, 64, 16)
    mw = [MoEWeights(w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g) for w in lws[:NL]]
    embed = head_weights(H, 1, 32, V, seed=921).embed
    for _ in range(2):                       # one sequence only: the first refusal has given it back
        with pytest.raises(ValueError, match="one AttentionLayer"):
            MoEStack(pool, mw, lm, embed, depth=D, top_k=K, attn=[attention_layer(H, 16, 4, 64, 960)], pages=pages)
    for chunk in (0, 16):
        with pytest.raises(ValueError, match="at least one token"):
            make_stack(parts, chunk).prompt([])


def test_a_resized_cache_is_captured_anew(parts):
    """The captured round and the captured drafts follow k and v to their new places (the old ones are poisoned here)."""
    stack, head = make_stack(parts), make_head(parts, 1)
    prompt, rounds = [5, 17, 300, 8, 1234], [[77], [9], [2], [64], [1000]]

    def run(resize):
        stack.reset()
        head.reset()
        graph, out = DraftGraph(head, 2), []
        _, multi = stack.forward(prompt)
        head.consume(prompt, multi)
        for i, tokens in enumerate(rounds):
            if resize and i in (2, 4):
                for pages in (stack.cache.pages, head.cache.pages):
                    old = pages.k, pages.v
                    pages.resize(pages.n_pages + 3)
                    for t in old:
                        t.fill_(float("nan"))
            nxt, multi = stack.forward(tokens)
            head.consume(tokens, multi)
            graph.token.fill_(nxt[0])
            graph.multi.copy_(head.prev_multi)
            out += nxt + graph.replay().cpu().tolist()
        return out

    want = run(False)
    assert run(True) == want and stack.cache.pages.resizes == 2 and _lib.device_error() == 0


def test_two_streams_at_once():
    """Two sequences of one cache decoded on two streams at the same time."""
    layer = attention_layer(512, 8, 2, 128, 31)
    kv = KVPages(1, 80, 2, 128, 16, max_seqs=2, max_tokens=640)
    seqs = [kv.new(), kv.new()]
    x = [normal_bf16((600, 512), 1.0, 32 + i) for i in range(2)]
    args = []
    for s in seqs:
        kv.extend(s, 600)
        args.append((torch.arange(600, dtype=torch.int32, device="cuda"), kv.k[0], kv.v[0],
                     torch.tensor([0, 600], dtype=torch.int32, device="cuda"),
                     torch.tensor([600], dtype=torch.int32, device="cuda"), kv.table[s:s + 1], 600))
    for i in range(2):
        layer(x[i], *args[i])
    q = [normal_bf16((1, 8, 128), 1.0, 40 + i) for i in range(2)]
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    run = lambda i: paged_attention(q[i], *args[i][1:3], cu, *args[i][4:6], 1)  # noqa: E731
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    assert all(torch.equal(bits(g), bits(want[i])) for i in range(2) for g in got[i])

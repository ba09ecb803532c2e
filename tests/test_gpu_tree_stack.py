"""A cache in 8 bits and rounds over trees as they are used: the attention layer, the pages with their forks and moves, the draft head, and
the stack's loops, against the definitions and the plain sequence."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.attention import SeqCache
from slotstream_spark_amd.engine.generate import MoEStack, mtp_decode, tree_decode
from slotstream_spark_amd.engine.mtp import HeadAttention, MTPHead
from slotstream_spark_amd.engine.step import MoEWeights
from slotstream_spark_amd.engine.verify import MoEVerifyLayer
from slotstream_spark_amd.kernels.tree import tree_masks
from slotstream_spark_amd.memory.kv_pages import KVPages
from slotstream_spark_amd.memory.synth import attention_layer, head_weights, normal_bf16
from tests.test_gpu_attention_layer import D, E, H, K, NL, V, bits, layer64, parts  # noqa: F401  (parts is a fixture)
from tests.tree_util import E4M3, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (16, 4, 64), (4, 1, 256)])
def test_layer_over_8_bits(heads, kv_heads, dim):
    """A prompt in two chunks, rounds and single tokens over e4m3 pages. The layer's error is that of the keys' and values' rounding
    (2^-4 of each, at most) through scores of a few units, beside bf16's own: against the definition without roundings."""
    n = 150
    layer = attention_layer(512, heads, kv_heads, dim, 5)
    x = normal_bf16((n, 512), 1.0, 6)
    outs = []
    for dtype in (torch.bfloat16, E4M3):
        pages = KVPages(1, 12, kv_heads, dim, 16, max_tokens=192, dtype=dtype)
        cache, got, pos = SeqCache(pages), [], 0
        for m in (100, 20, 3, 3, 1, 8, 15):
            cache.place(pos, m)
            cu, kv_len, table, positions = cache.rows(m)
            got.append(layer(x[pos:pos + m].contiguous(), positions, pages.k[0], pages.v[0], cu, kv_len, table, m, **pages.of_layer(0)))
            pos += m
        assert pos == n
        outs.append(torch.cat(got).double())
    want, top = layer64(layer, x, torch.arange(n, device="cuda"))
    off16, off8 = ((o - want).norm() / want.norm() for o in outs)
    # a key's elements are off by at most 2^-4 of themselves, so a score by at most 2^-4 sum |q_i k_i| <= 2^-4 |q| |k|, in the mean (errors
    # that do not know of each other) by 2^-4 / sqrt(3 dim) of that; a value's by 2^-4, their weighted mean by no more
    assert off16 < 0.02 and off8 < 2.0 ** -4 + 0.02, (off16, off8, top)
    assert _lib.device_error() == 0


def test_forks_moves_and_resizes_in_8_bits():
    """What a fork, a compaction and a resize move are the pages with their scales: rows go on with the bits they would have had."""
    layer = attention_layer(512, 8, 2, 64, 7)
    x = normal_bf16((64, 512), 1.0, 8)
    pages = KVPages(1, 16, 2, 64, 16, max_seqs=4, max_tokens=96, dtype=E4M3)
    first, cache = SeqCache(pages), SeqCache(pages)
    first.place(0, 40)

    def run(c, pos, m, rows):
        c.place(pos, m)
        cu, kv_len, table, positions = c.rows(m)
        return layer(rows, positions, pages.k[0], pages.v[0], cu, kv_len, table, m, **pages.of_layer(0))

    run(cache, 0, 40, x[:40].contiguous())
    want = run(cache, 40, 4, x[40:44].contiguous()).clone()
    child = pages.fork(cache.seq)
    pages.free(first.seq)
    pages.compact()
    pages.resize(7)
    assert torch.equal(bits(run(cache, 40, 4, x[40:44].contiguous())), bits(want))     # copies the page that the child shares
    run(cache, 40, 4, x[50:54].contiguous())
    other = SeqCache(pages)
    pages.free(other.seq)
    other.seq, other.table = child, pages.table[child:child + 1]
    run(other, 44, 1, x[44:45].contiguous())
    assert torch.equal(bits(run(other, 40, 4, x[40:44].contiguous())), bits(want))
    assert _lib.device_error() == 0


def test_layer_over_a_tree_equals_its_branches():
    """Every row of a tree through the layer against the rows of its branch alone, to the roundings of both."""
    n, base = 24, 37
    layer = attention_layer(512, 8, 2, 128, 9)
    x = normal_bf16((base + n, 512), 1.0, 10)
    for dtype in (torch.bfloat16, E4M3):
        pages = KVPages(1, 24, 2, 128, 16, max_seqs=2, max_tokens=96, dtype=dtype)
        cache = SeqCache(pages)

        def run(pos, rows, **kw):
            m = rows.shape[0]
            cache.place(pos, m)
            cu, kv_len, table, positions = cache.rows(m)
            if "parents" in kw:
                masks, positions = tree_masks(kw["parents"], cu, kv_len, m)
                kw = dict(tree=masks)
            return layer(rows, positions, pages.k[0], pages.v[0], cu, kv_len, table, m, **pages.of_layer(0), **kw)

        run(0, x[:base].contiguous())
        parents = random_parents(n, 3)
        got = run(base, x[base:].contiguous(), parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))
        for i in range(n):
            path, p = [], i
            while p >= 0:
                path.insert(0, p)
                p = parents[p]
            alone = run(base, x[base + torch.tensor(path, device="cuda")].contiguous())[-1]
            # two results of one exact value: each is off by the rounding of its projections and probabilities, bf16's 2^-8 a few times
            assert (got[i].float() - alone.float()).norm() <= 2.0 ** -6 * alone.float().norm(), i
    assert _lib.device_error() == 0


def stack_of(parts, dtype, prompt_chunk=0, max_tokens=160, attention=True, pages=14, bias=None):  # noqa: F811
    pool, lws, lm = parts
    mw = [MoEWeights(w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g, bias) for w in lws[:NL]]
    norms = [normal_bf16((H,), 0.1, 950 + l).float().add(1).to(torch.bfloat16) for l in range(NL + 1)]
    kw = dict(attn=[attention_layer(H, 16, 4, 64, 960 + l) for l in range(NL)], attn_norms=norms[:NL],
              pages=KVPages(NL, pages, 4, 64, 16, max_tokens=max_tokens, dtype=dtype)) if attention else {}
    return MoEStack(pool, mw, lm, head_weights(H, 1, 32, V, seed=921).embed, depth=D, norm_weights=norms, top_k=K,
                    prompt_chunk=prompt_chunk, **kw)


PROMPT, N = [5, 17, 300, 8, 1234, 77, 9, 9, 2, 64, 1000, 41, 3, 50, 11, 600, 23, 90, 4], 24


def plain(stack, n=N):
    """(the sequence of one-token steps, each step's logits)."""
    stack.reset()
    out, logits = [stack.prompt(PROMPT)[0][-1]], []
    while len(out) < n:
        out.append(stack.forward([out[-1]])[0][0])
        logits.append(stack.plain_logits[0].clone())
    return out, logits


def branching(want):
    """A drafter that knows the sequence `want`: two wrong branches around the right one, whose rows are not neighbours."""
    def tree_fn(pending, room, n_out):
        right = (want + [0] * 4)[n_out:n_out + 4]
        drafts, par = [(right[0] + 1) % V, right[0], (right[0] + 2) % V], [0, 0, 0]
        drafts += [right[1], (right[1] + 3) % V, right[2], right[2], right[3]]
        par += [2, 2, 4, 1, 6]
        return drafts[:room], par[:room]
    return tree_fn


@pytest.mark.parametrize("routed", ["freely", "alike"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("prompt_chunk", [0, 32])
def test_rounds_over_trees_are_the_plain_steps(parts, dtype, prompt_chunk, routed):  # noqa: F811
    """Every kept row of a round against the same token as a one-token step of another stack that is fed what the rounds kept.

    The two work in another order of sums, so a row's stream is off by bf16's half step (2^-8) for each of a layer's two residual sums
    and what they carry on: 2^-6 of it after two layers. That moves a router's or the lm_head's logits by 2^-6 of their spread about
    (a row of weights sees the difference as it sees any vector). So where the routers choose other experts, the last chosen and the first
    left out were nearer than 2^-4 of the spread, and from that row on the sequences are not the same; where they choose the same and the
    next token is another one, the two tokens' logits were that near. Routed alike (a bias far above the logits) all rows take the same
    experts, so that only the latter can end the comparison."""
    bias = None
    if routed == "alike":
        bias = torch.zeros(E, device="cuda")
        bias[5:5 + K] = 1000.0
    ref, stack = stack_of(parts, dtype, prompt_chunk, bias=bias), stack_of(parts, dtype, prompt_chunk, bias=bias)
    want, _ = plain(ref)
    tree_fn = branching(want)
    seen = []

    class Watched:
        def __init__(self, layer):
            self.layer = layer

        def __call__(self, x, **kw):
            got = self.layer(x, **kw)
            seen.append(got[1].clone())
            return got

    plain_layers, prompt_layers = stack.graph.layers, stack.prompt_layers
    ref.reset()
    assert stack.prompt(PROMPT)[0] == ref.prompt(PROMPT)[0]
    out, compared, apart = [want[0]], 0, False
    while len(out) < N:
        drafts, par = tree_fn(out[-1], 63, len(out))
        seen.clear()
        watched = [Watched(x) for x in (plain_layers if prompt_layers is None else prompt_layers)]
        if prompt_layers is None:
            stack.graph.layers = watched
        else:
            stack.prompt_layers = watched
        res, rows = stack.tree_step([out[-1], *drafts], [-1, *par])
        stack.graph.layers, stack.prompt_layers = plain_layers, prompt_layers
        per = len(seen) // NL
        ids = [torch.cat(seen[l * per:(l + 1) * per]) for l in range(NL)]
        kept = [([out[-1]] + drafts)[r] for r in res.path]
        assert res.flags == 0 and kept[1:] == res.tokens[:-1] and res.n_emit == len(kept)
        for j, tok in enumerate([] if apart else kept):
            nxt, multi = ref.forward([tok])
            for l in range(NL):
                assert routed == "freely" or set(ref.graph.ids[l, 0].tolist()) == set(range(5, 5 + K))
                if set(ids[l][res.path[j]].tolist()) != set(ref.graph.ids[l, 0].tolist()):
                    x = (ref.graph.mixed[l][0].float() @ parts[1][l].router_w.float().t()).sort(descending=True)[0]
                    assert x[K - 1] - x[K] <= 2.0 ** -4 * x.std(), (len(out), j, l)
                    apart = True
                    break
            if apart:
                break
            assert (rows[j].float() - multi[0].float()).norm() <= 2.0 ** -6 * multi[0].float().norm(), (len(out), j)
            compared += 1
            if res.tokens[j] != nxt[0]:
                x = ref.plain_logits[0]
                assert x[nxt[0]] - x[res.tokens[j]] <= 2.0 ** -4 * x.std(), (len(out), j)
                apart = True
                break
        out += res.tokens
    assert compared >= (1 if routed == "alike" else 0)    # the first row is there to be compared, whatever it chooses
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("prompt_chunk", [0, 32])
def test_the_loop_over_trees_is_its_rounds(parts, dtype, prompt_chunk):  # noqa: F811
    """tree_decode emits what its rounds emit, call by call the same; its records and the stack's sequence agree with what it emitted."""
    stack = stack_of(parts, dtype, prompt_chunk)
    tree_fn = branching(plain(stack)[0])

    def rounds(n):
        stack.reset()
        out, counts = [stack.prompt(PROMPT)[0][-1]], []
        while len(out) < n:
            drafts, par = tree_fn(out[-1], 63, len(out))
            res, _ = stack.tree_step([out[-1], *drafts], [-1, *par])
            counts.append((len(drafts), res.n_accept, res.n_emit))
            out += res.tokens
        return out, counts

    want, counts = rounds(N)
    assert max(c[2] for c in counts) == 5       # a whole branch was followed
    calls = []
    stack.reset()
    out, nan, _, st = tree_decode(stack, PROMPT, N, tree_fn, on_token=calls.append)
    assert out == want[:N] == calls and not nan
    assert st["rounds"] == len(counts) and st["emitted_by_round"] == [c[2] for c in counts]
    assert st["drafted"] == sum(c[0] for c in counts) and st["accepted"] == sum(c[1] for c in counts)
    assert stack.st.pos == len(stack.st.tokens) == len(PROMPT) + N - 1 == stack.cache.pos
    assert stack.st.tokens[len(PROMPT):] == out[:-1]
    stack.reset()
    stop = want[7]
    short, _, _, _ = tree_decode(stack, PROMPT, N, tree_fn, eos=(stop,))
    assert short == want[:want.index(stop) + 1] and stack.st.pos == len(PROMPT) + len(short) - 1
    assert _lib.device_error() == 0


def test_trees_without_drafts_near_the_end_and_refusals(parts):  # noqa: F811
    stack = stack_of(parts, torch.bfloat16, 0, max_tokens=64, pages=4)
    out, _, _, st = tree_decode(stack, PROMPT, N, lambda p, room, n: ([], []))
    assert len(out) == N and st["accepted"] == 0 and st["emitted_by_round"] == [1] * (N - 1)
    stack.reset()
    rooms = []

    def greedy(p, room, n):
        rooms.append(room)
        return [7] * room, list(range(room))

    out, _, _, _ = tree_decode(stack, PROMPT, 10 ** 6, greedy)
    assert stack.st.pos == stack.max_ctx and min(rooms) >= 1 and len(out) == stack.max_ctx - len(PROMPT) + 1
    stack.reset()
    stack.prompt(PROMPT)
    before = (stack.st.pos, list(stack.st.tokens), stack.cache.pages.free_pages)
    for tokens, par in (([], []), ([1, 2], [-1]), ([1, 2], [-1, 1]), ([1, 2], [-1, -1]), (list(range(65)), [-1] + [0] * 64)):
        with pytest.raises(ValueError):
            stack.tree_step(tokens, par)
    assert before == (stack.st.pos, list(stack.st.tokens), stack.cache.pages.free_pages)
    with pytest.raises(ValueError):
        tree_decode(stack_of(parts, torch.bfloat16, 4), PROMPT, N, lambda p, room, n: ([1] * (room + 1), [0] * (room + 1)))


def test_trees_over_a_stack_without_attention(parts):  # noqa: F811
    stack = stack_of(parts, torch.bfloat16, attention=False)
    nxt = {}

    def f(t):
        if t not in nxt:
            stack.reset()
            nxt[t] = stack.forward([t])[0][0]
        return nxt[t]

    first = f(11)
    second = f(first)
    stack.reset()
    res, rows = stack.tree_step([11, (first + 1) % V, first, (second + 1) % V, second], [-1, 0, 0, 2, 2])
    assert res.path == [0, 2, 4] and res.tokens[:2] == [first, second] and res.n_accept == 2
    assert tuple(rows.shape) == (3, H) and stack.st.tokens == [11, first, second]
    # without attention a row has the bits of its token alone
    alone = stack.forward([second])[1]
    assert torch.equal(bits(rows[2:]), bits(alone))


def test_speculative_loop_over_8_bits(parts):  # noqa: F811
    """The chain's loop over e4m3 pages emits what one-token steps over e4m3 pages emit, bit for bit, with the head's cache in 8 bits too."""
    pool, lws, lm = parts
    stack = stack_of(parts, E4M3, 16)
    w = lws[NL]
    moe = MoEVerifyLayer(pool, NL, w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g, top_k=K, max_tokens=4)
    attn = HeadAttention(head_weights(H, 1, 32, 64, seed=923).mlp_hc, attention_layer(H, 16, 4, 64, 924),
                         KVPages(1, 8, 4, 64, 16, max_tokens=64, dtype=E4M3))
    head = MTPHead(head_weights(H, 1, 32, V, seed=921), moe, lm, hc=1, max_ctx=64, attn=attn)
    want, _ = plain(stack)
    for fn in (None, lambda p, depth, n: (want + [0] * depth)[n:n + depth], lambda p, depth, n: [3] * depth):
        stack.reset()
        head.reset()
        out, nan, _, st = mtp_decode(stack, head, PROMPT, N, draft_fn=fn)
        assert out == want and not nan
        assert stack.st.pos == len(PROMPT) + N - 1
    assert _lib.device_error() == 0

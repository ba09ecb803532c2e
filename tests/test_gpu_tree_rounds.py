"""Rounds over trees as a stack runs them: windows whose pages are given back between the rounds, rows that are not finite, the loop's ends,
and every kept row against one-token steps."""
import pytest
import torch

from slotstream_spark_amd import _lib
from slotstream_spark_amd.engine.generate import MoEStack, mtp_decode, tree_decode
from slotstream_spark_amd.engine.step import MoEWeights
from slotstream_spark_amd.memory.kv_pages import KVPages
from slotstream_spark_amd.memory.synth import attention_layer, head_weights, normal_bf16
from tests.test_gpu_attention_layer import D, E, H, K, NL, V, make_head, parts  # noqa: F401  (parts is a fixture)
from tests.test_gpu_tree_stack import PROMPT, branching, plain, stack_of
from tests.tree_util import E4M3

pytestmark = pytest.mark.gpu


def windowed(parts, window, dtype=torch.bfloat16, prompt_chunk=0, max_tokens=320, pages=22):  # noqa: F811
    pool, lws, lm = parts
    mw = [MoEWeights(w.router_w, w.sh_gate, w.sh_up, w.sh_down, w.sh_g) for w in lws[:NL]]
    norms = [normal_bf16((H,), 0.1, 950 + l).float().add(1).to(torch.bfloat16) for l in range(NL + 1)]
    return MoEStack(pool, mw, lm, head_weights(H, 1, 32, V, seed=921).embed, depth=D, norm_weights=norms, top_k=K,
                    attn=[attention_layer(H, 16, 4, 64, 960 + l, window=window, sinks=2) for l in range(NL)], attn_norms=norms[:NL],
                    pages=KVPages(NL, pages, 4, 64, 16, max_tokens=max_tokens, dtype=dtype), prompt_chunk=prompt_chunk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("size", [40, 48])
def test_pages_given_back_between_rounds(parts, dtype, size):  # noqa: F811
    """Trees much larger than the rows they leave, under a window that just holds them: a loop that gives pages back before each round by the
    stack's own recipe emits what one emits that keeps them, sees no missing page, and holds fewer."""
    window, n, outs, free = 48, 100, [], []
    for evict in (False, True):
        stack, held = windowed(parts, window, dtype), []

        def tree_fn(pending, room, n_out):
            if evict:
                stack.cache.pages.evict(stack.cache.seq, window, 2, back=stack.rows)
            held.append(stack.cache.pages.free_pages)
            m = min(room, size - 1)
            return [(pending + 3 * i) % V for i in range(m)], [(i - 1) // 4 if i else 0 for i in range(m)]

        out, nan, _, st = tree_decode(stack, PROMPT, n, tree_fn)
        assert _lib.device_error() == 0
        assert len(out) == n and not nan and st["rounds"] > n // 4 and st["drafted"] >= 20 * st["rounds"]
        assert stack.st.pos == len(PROMPT) + n - 1
        outs.append(out)
        free.append(held[-1])
    assert outs[0] == outs[1] and free[1] > free[0]


def test_a_sequence_has_the_tokens_that_rounds_left(parts):  # noqa: F811
    """After a round, and after tokens were taken back, the pages' own count is the stack's position."""
    stack = stack_of(parts, torch.bfloat16)
    pages, seq = stack.cache.pages, stack.cache.seq
    stack.prompt(PROMPT)
    res, _ = stack.tree_step([5] + [7] * 40, [-1] + [0] * 40)
    assert pages.length[seq] == stack.st.pos == len(PROMPT) + len(res.path)
    assert sum(p >= 0 for p in pages.table[seq].tolist()) == -(-stack.st.pos // pages.page)
    def fails(*a, **kw):
        raise RuntimeError("no pass")

    stack._through = fails                                  # a round that fails half way leaves none of its rows
    with pytest.raises(RuntimeError, match="no pass"):
        stack.tree_step([5] + [7] * 40, [-1] + [0] * 40)
    assert pages.length[seq] == stack.st.pos == len(stack.st.tokens) == len(PROMPT) + len(res.path)
    del stack._through                                      # the class's own again (put back by value it would hold the stack itself)
    stack.take_back(3)
    assert pages.length[seq] == stack.st.pos == len(stack.st.tokens) == len(PROMPT) + len(res.path) - 3
    assert _lib.device_error() == 0


def test_drafts_up_to_the_room_under_a_window(parts):  # noqa: F811
    """A tree's rows must fit every layer's window: the room that a drafter is told is one that a round takes."""
    stack, rooms = windowed(parts, 20), []

    def tree_fn(pending, room, n_out):
        rooms.append(room)
        return [pending] * room, [0] * room

    out, nan, _, _ = tree_decode(stack, PROMPT, 12, tree_fn)
    assert len(out) == 12 and not nan and set(rooms) == {19} and _lib.device_error() == 0
    with pytest.raises(ValueError, match="window"):
        stack.tree_step([1] * 21, [-1] + [0] * 20)
    one, drafted = windowed(parts, 1), []
    out, _, _, st = tree_decode(one, PROMPT, 5, lambda *a: drafted.append(a) or ([], []))
    assert len(out) == 5 and st["rounds"] == 4 and not drafted and _lib.device_error() == 0


@pytest.mark.parametrize("n", [0, -1, 1])
def test_no_token_asked_for(parts, n):  # noqa: F811
    """The prompt's own token comes first in either loop, and a loop that is asked for no more ends with it."""
    stack, head = stack_of(parts, torch.bfloat16), make_head(parts, 1)
    want, _, _, _ = mtp_decode(stack, head, PROMPT, n)
    stack.reset()
    out, nan, _, st = tree_decode(stack, PROMPT, n, lambda p, room, k: ([1], [0]))
    assert out == want and len(out) == 1 and not nan and st["rounds"] == 0
    assert stack.st.pos == stack.cache.pos == len(PROMPT)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("prompt_chunk", [0, 32])
def test_a_row_that_is_not_finite_ends_the_loop(parts, dtype, prompt_chunk):  # noqa: F811
    """A token whose embedding is NaN, drafted and accepted in the middle of a branch, or pending: its row's choice is not emitted, the loop
    ends, and the sequence is the prompt and all that was emitted (the last token's row has been run, as at mtp_decode's end)."""
    stack = stack_of(parts, dtype, prompt_chunk)
    tree_fn = branching(plain(stack)[0])
    stack.reset()
    want, _, _, st = tree_decode(stack, PROMPT, 24, tree_fn)
    ends, at = [], 1
    for n in st["emitted_by_round"]:
        ends.append(at)
        at += n
    ran = 0
    for i in (next(i for i in range(ends[1], 20) if want.index(want[i]) == i and i + 1 not in ends), ends[3] - 1):
        if want.index(want[i]) != i or want[i] in PROMPT:
            continue
        ran += 1
        bad = stack_of(parts, dtype, prompt_chunk)
        bad.embed = bad.embed.clone()
        bad.embed[want[i]] = float("nan")
        out, nan, _, st = tree_decode(bad, PROMPT, 24, tree_fn)
        assert nan and out == want[:i + 1], (i, out, want)
        assert bad.st.tokens == PROMPT + out and bad.st.pos == bad.cache.pos == bad.cache.pages.length[bad.cache.seq] == len(bad.st.tokens)
        assert _lib.device_error() == 0
        bad.reset()
        res, rows = (bad.prompt(PROMPT), bad.tree_step([want[i], 3, 4], [-1, 0, 0]))[1]
        assert (res.n_accept, res.n_emit, res.flags, res.path) == (0, 0, 1, [0]) and torch.isnan(rows[0]).any()
    assert ran


def test_an_end_before_a_row_that_is_not_finite(parts):  # noqa: F811
    """A round whose branch ends at a row that is not finite, behind a token that ends the sequence or is the last one asked for: the loop ends
    with that token, and nothing that it emits came after such a row."""
    stack = stack_of(parts, torch.bfloat16)
    tree_fn = branching(plain(stack)[0])
    stack.reset()
    want, _, _, st = tree_decode(stack, PROMPT, 24, tree_fn)
    at, found = 1, None
    for n in st["emitted_by_round"]:                         # a round of three tokens or more, the third of them a new one
        if found is None and n >= 3 and want.index(want[at + 1]) == at + 1 and want[at + 1] not in PROMPT:
            found = at
        at += n
    assert found is not None
    bad = stack_of(parts, torch.bfloat16)
    bad.embed = bad.embed.clone()
    bad.embed[want[found + 1]] = float("nan")
    out, nan, _, _ = tree_decode(bad, PROMPT, 24, tree_fn)
    assert nan and out == want[:found + 2]
    for kw in (dict(max_tokens=found + 2), dict(max_tokens=found + 1), dict(max_tokens=24, eos=(want[found + 1],))):
        bad.reset()
        out, nan, _, _ = tree_decode(bad, PROMPT, tree_fn=tree_fn, **kw)
        assert out == want[:min(kw["max_tokens"], found + 2)] and not nan
        assert bad.st.tokens == PROMPT + out[:-1] and bad.st.pos == bad.cache.pos == bad.cache.pages.length[bad.cache.seq] == len(PROMPT) + len(out) - 1
    assert _lib.device_error() == 0


@pytest.mark.parametrize("routed", ["freely", "alike"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("prompt_chunk", [0, 32])
def test_kept_rows_of_every_round(parts, dtype, prompt_chunk, routed):  # noqa: F811
    """Every kept row of every round, deep ones and those behind moved branches among them, against a one-token step of a stack that is fed
    what the rounds kept.

    A row's stream is off by bf16's half step (2^-8) for each of a layer's two residual sums and what they carry on: 2^-6 of it after two
    layers. Over e4m3 a key or value that is 2^-8 of itself off falls on the next code in one of 2^5 (a step is 2^-3 at most), 2^-5.5 in
    the mean square of what the attention adds: 2^-5 in all. A choice (of the lm_head, of a router) that differs was that near: four times
    that of the logits' spread. Routed alike nothing else may differ, so every kept row is compared, whatever was chosen. Routed freely, a
    row whose experts differ ends its round; the plain stack's cache is then made the rounds' own before the next."""
    bias = None
    if routed == "alike":
        bias = torch.zeros(E, device="cuda")
        bias[5:5 + K] = 1000.0
    far = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -5
    ref, stack = stack_of(parts, dtype, prompt_chunk, bias=bias), stack_of(parts, dtype, prompt_chunk, bias=bias)
    n = 40
    own, _, _, _ = tree_decode(stack, PROMPT, n + 5, lambda p, room, k: ([], []))
    tree_fn, seen = branching(own), []
    stack.reset()

    class Watched:
        def __init__(self, layer):
            self.layer = layer

        def __call__(self, x, **kw):
            got = self.layer(x, **kw)
            seen.append(got[1].clone())
            return got

    def same_cache():
        a, b = ref.cache, stack.cache
        for w in range(-(-stack.st.pos // a.pages.page)):
            x, y = int(a.table[0, w]), int(b.table[0, w])
            for s, t in ((a.pages.k, b.pages.k), (a.pages.v, b.pages.v)) + (((a.pages.scales, b.pages.scales),) if dtype == E4M3 else ()):
                s.view(torch.uint8)[:, x] = t.view(torch.uint8)[:, y]

    assert stack.prompt(PROMPT)[0][-1] == ref.prompt(PROMPT)[0][-1] == own[0]
    out, kept_rows, compared, deep, after, moved, apart = own[:1], 0, 0, 0, 0, False, False
    watched = "layers" if prompt_chunk == 0 else "prompt_layers"
    holder = stack.graph if prompt_chunk == 0 else stack
    layers = getattr(holder, watched)
    while len(out) < n:
        if apart:
            same_cache()
            apart = False
        drafts, par = tree_fn(out[-1], 63, len(out))
        seen.clear()
        setattr(holder, watched, [Watched(x) for x in layers])
        res, rows = stack.tree_step([out[-1], *drafts], [-1, *par])
        setattr(holder, watched, layers)
        per = len(seen) // NL
        ids = [torch.cat(seen[l * per:(l + 1) * per]) for l in range(NL)]
        kept = [([out[-1]] + drafts)[r] for r in res.path]
        assert res.flags == 0 and kept[1:] == res.tokens[:-1] and res.n_emit == len(kept)
        kept_rows += len(kept)
        for j, tok in enumerate(kept):
            nxt, multi = ref.forward([tok])
            for l in range(0 if apart else NL):
                if set(ids[l][res.path[j]].tolist()) != set(ref.graph.ids[l, 0].tolist()):
                    assert routed == "freely"
                    x = (ref.graph.mixed[l][0].float() @ parts[1][l].router_w.float().t()).sort(descending=True)[0]
                    assert x[K - 1] - x[K] <= 4 * far * x.std(), (len(out), j, l)
                    apart = True
                    break
            if apart:
                continue
            assert (rows[j].float() - multi[0].float()).norm() <= far * multi[0].float().norm(), (len(out), j)
            compared += 1
            deep += j >= 2
            after += moved
            if res.tokens[j] != nxt[0]:
                x = ref.plain_logits[0]
                assert x[nxt[0]] - x[res.tokens[j]] <= 4 * far * x.std(), (len(out), j)
        moved |= res.path != list(range(len(res.path)))
        out += res.tokens
    assert ref.st.tokens == stack.st.tokens and _lib.device_error() == 0
    print(f"[rounds] {routed} kept={kept_rows} compared={compared} deep={deep} after={after}", flush=True)
    if routed == "alike":
        assert compared == kept_rows and deep >= 8 and after >= 20
    else:
        assert compared >= 12 and deep >= 2 and after >= 8

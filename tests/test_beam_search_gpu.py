"""GPU: beam search over the paged 4-bit cache, its operators together as a server runs them: a prompt in two
parts (append and chunk attention), then steps of select, fork of the rows and of a recurrent state, growth by a
token, append and attention, eager and as one captured graph, against numpy in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import chunk_reference as CR
import kv4_reference as R
from conftest import load_mixer
from test_chunk_gpu import assert_near, begins_of
from test_kv4_gpu import assert_same, ints, result, upload

pytestmark = pytest.mark.gpu

M = load_mixer()
GROUPS, BEAMS, VOCAB, LAYERS = 2, 3, 1500, 2
ROWS = GROUPS * BEAMS
END = 7
STATE = 4096 + 16


@pytest.mark.parametrize("captured", [False, True])
def test_beam_search(captured):
    rng = np.random.default_rng(70)
    prompts = [100, 37]
    longest, most = 160, 128
    ctx = M.Context(0)
    ctx.reserve(ROWS, longest, most)
    ref = R.Cache(LAYERS, 40, ROWS, R.pages_of(longest), seed=71)
    c = upload(ctx, ref)
    cos, sin = M.rope_table(longest)
    gammas = [(0.1 * rng.standard_normal(256)).astype(np.float16) for _ in range(2)]
    rc, rs = ctx.upload(cos), ctx.upload(sin)
    q_norm, k_norm = (ctx.upload(g.view(np.uint16)) for g in gammas)
    bufs = {"q": ctx.alloc(most * 16384), "k": ctx.alloc(most * 2048), "v": ctx.alloc(most * 2048), "out": ctx.alloc(most * 8192)}
    res = [ints(ctx, [-77]) for _ in range(3)]

    def layer_inputs(n):
        q = CR.bf16(rng.standard_normal((n, 16, 512)))
        k, v = (CR.bf16(rng.standard_normal((n, 4, 256))) for _ in range(2))
        return q, k, v

    def layer(at, batch, slots, begins, tokens, max_new):
        ctx.kv4_append(c, at, batch, slots, begins, tokens, bufs["k"], bufs["v"], k_norm, rc, rs, longest, longest, res[0], dtype=M.QM_BF16)
        ctx.gqa_chunk_kv4(c, at, batch, slots, begins, tokens, max_new, bufs["q"], q_norm, rc, rs, longest, longest, res[0], bufs["out"])

    def check_layer(at, batch, slots, begins, tokens, max_new, q, k, v):
        CR.append(ref, at, batch, slots, begins, tokens, CR.bf16_value(k), CR.bf16_value(v), gammas[1], cos, sin, longest)
        want, bound, _ = CR.attend(ref, at, batch, slots, begins, tokens, max_new, CR.bf16_value(q), gammas[0], cos, sin, longest)
        assert_near(CR.bf16_value(ctx.download(bufs["out"], (tokens, 16, 256), np.uint16)), want, bound)

    # the prompts into the groups' first rows, in two parts
    slots = [g * BEAMS for g in range(GROUPS)]
    for part in range(2):
        news = [n // 2 if part == 0 else n - n // 2 for n in prompts]
        begins, tokens = begins_of(news), sum(news)
        ctx.kv4_resize(c, GROUPS, ints(ctx, slots), ints(ctx, news), res[0], M.QM_KV4_ADD)
        assert result(ctx, res[0]) == ref.resize(slots, news, add=True) == 0
        for at in range(LAYERS):
            q, k, v = layer_inputs(tokens)
            for key, x in (("q", q), ("k", k), ("v", v)):
                ctx.upload(x, bufs[key])
            layer(at, GROUPS, ints(ctx, slots), ints(ctx, begins), tokens, max(news))
            check_layer(at, GROUPS, slots, begins, tokens, max(news), q, k, v)
        assert_same(ctx, c, ref)

    # the other beams begin as copies without a score
    src = [r // BEAMS * BEAMS for r in range(ROWS)]
    ctx.kv4_fork(c, ROWS, ints(ctx, src), ints(ctx, list(range(ROWS))), res[0])
    assert result(ctx, res[0]) == ref.fork(src, list(range(ROWS))) == 0
    scores = np.where(np.arange(ROWS) % BEAMS == 0, 0, -np.inf).astype(np.float32)
    done = np.zeros(ROWS, np.int32)
    state = rng.integers(0, 2 ** 32, (ROWS, STATE // 4), dtype=np.uint32)
    x, s, d = ctx.alloc(ROWS * VOCAB * 4), ctx.upload(scores), ctx.upload(done)
    st, parents, tokens, identity = ctx.upload(state), ctx.alloc(4 * ROWS), ctx.alloc(4 * ROWS), ints(ctx, list(range(ROWS)))
    add, begins = ints(ctx, [1] * ROWS), ints(ctx, list(range(ROWS + 1)))

    def reorder():
        ctx.beam_select(GROUPS, BEAMS, BEAMS, VOCAB, x, s, d, END, parents, tokens, s, d)
        ctx.kv4_fork(c, ROWS, parents, identity, res[1])
        ctx.state_fork([(st, STATE, STATE)], ROWS, ROWS, parents, None, res[2])
        ctx.kv4_resize(c, ROWS, None, add, res[0], M.QM_KV4_ADD)
        layer(0, ROWS, None, begins, ROWS, 1)

    if captured:
        ctx.graph_begin()
        reorder()
        graph = ctx.graph_end()
    ended = False
    for step in range(12):
        print(f"case: beam search step {step}", flush=True)
        logits = (2 * rng.standard_normal((ROWS, VOCAB))).astype(np.float32)
        logits[rng.integers(0, ROWS), END] += 9
        q, k, v = layer_inputs(ROWS)
        for buf, arr in ((x, logits), (bufs["q"], q), (bufs["k"], k), (bufs["v"], v)):
            ctx.upload(arr, buf)
        if captured and step != 4:                                       # eager in between
            graph.launch()
        else:
            reorder()
        want = CR.select(GROUPS, BEAMS, BEAMS, VOCAB, logits, scores, done, END)
        got = [ctx.download(b, (ROWS,), t) for b, t in ((parents, np.int32), (tokens, np.int32), (s, np.float32), (d, np.int32))]
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
        assert (np.abs(got[2] - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 2.0 ** -19).all()
        scores, done = got[2], got[3]
        ended |= bool(done.any())
        assert [result(ctx, r) for r in res] == [0, 0, 0]
        assert ref.fork(got[0], list(range(ROWS))) == 0 and ref.resize(None, [1] * ROWS, add=True) == 0
        state = state[got[0]]
        assert np.array_equal(ctx.download(st, state.shape, np.uint32), state)
        check_layer(0, ROWS, None, list(range(ROWS + 1)), ROWS, 1, q, k, v)
        # the other layer by itself, its inputs in the same buffers
        q, k, v = layer_inputs(ROWS)
        for key, arr in (("q", q), ("k", k), ("v", v)):
            ctx.upload(arr, bufs[key])
        layer(1, ROWS, None, begins, ROWS, 1)
        check_layer(1, ROWS, None, list(range(ROWS + 1)), ROWS, 1, q, k, v)
        assert_same(ctx, c, ref)
        assert ref.consistent()
    assert ended
    if captured:
        graph.close()
    ctx.close()


@pytest.mark.parametrize("captured", [False, True])
def test_a_request_that_runs_short_leaves_the_others_alone(captured):
    """Four requests: one as ever, one without a sequence (no score is finite), one whose logits hold a NaN from some
    step on, one whose mask leaves a single token.  Their places without a continuation stay the rows that they are,
    and the forks move the others' rows and states."""
    groups, rows, vocab, state_bytes = 4, 12, 700, 208
    rng = np.random.default_rng(80)
    ctx = M.Context(0)
    ctx.reserve(rows, 256)
    ref = R.Cache(1, 60, rows, 4, seed=81)
    assert ref.resize(None, [70, 70, 70, 1, 1, 1, 64, 64, 64, 130, 130, 130]) == 0
    c = upload(ctx, ref)
    scores = np.where(np.arange(rows) % BEAMS == 0, 0, -np.inf).astype(np.float32)
    scores[3:6] = -np.inf
    done = np.zeros(rows, np.int32)
    state = rng.integers(0, 2 ** 32, (rows, state_bytes // 4), dtype=np.uint32)
    x, s, d, st = ctx.alloc(rows * vocab * 4), ctx.upload(scores), ctx.upload(done), ctx.upload(state)
    parents, tokens, res = ctx.alloc(4 * rows), ctx.alloc(4 * rows), [ints(ctx, [-77]) for _ in range(3)]
    identity, add = ints(ctx, list(range(rows))), ints(ctx, [1] * rows)

    def step():
        ctx.beam_select(groups, BEAMS, BEAMS, vocab, x, s, d, END, parents, tokens, s, d)
        ctx.kv4_fork(c, rows, parents, identity, res[0])
        ctx.state_fork([(st, state_bytes, state_bytes)], rows, rows, parents, None, res[1])
        ctx.kv4_resize(c, rows, None, add, res[2], M.QM_KV4_ADD)

    if captured:
        ctx.graph_begin()
        step()
        graph = ctx.graph_end()
    moved = short = 0
    for i in range(8):
        print(f"case: requests that run short, step {i}", flush=True)
        logits = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
        if i >= 3:
            logits[6 + i % 2, 11] = np.nan
        logits[9:, np.arange(vocab) != 5] = -np.inf
        if i == 5:
            logits[6:9] = np.nan
        ctx.upload(logits, x)
        if captured and i != 4:
            graph.launch()
        else:
            step()
        want = CR.select(groups, BEAMS, BEAMS, vocab, logits, scores, done, END)
        none = want[0] < 0
        source = np.where(none, np.arange(rows), want[0])
        got = [ctx.download(b, (rows,), t) for b, t in ((parents, np.int32), (tokens, np.int32), (s, np.float32), (d, np.int32))]
        assert np.array_equal(got[0], source) and np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
        assert (got[2][none] == -np.inf).all() and np.isfinite(got[2][~none]).all()
        scores, done = got[2], got[3]
        assert [result(ctx, r) for r in res] == [0, 0, 0]
        assert ref.fork(source, list(range(rows))) == 0 and ref.resize(None, [1] * rows, add=True) == 0
        state = state[source]
        assert np.array_equal(ctx.download(st, state.shape, np.uint32), state)
        assert_same(ctx, c, ref)
        moved += int((source[:3] != np.arange(3)).sum())
        short += int(none.sum())
    assert moved and short > 8 * 3 and ref.consistent()
    if captured:
        graph.close()
    ctx.close()

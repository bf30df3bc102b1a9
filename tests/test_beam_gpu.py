"""GPU: beam search's selection and the reordering of recurrent states, against numpy in 64 bits.

Parents, tokens and flags have to be equal.  A score is the f64 value rounded to f32 (2^-24 of itself) beside a
log-sum from f32 exponentials and sums: the exponentials' errors (some 2^-23 of each) and the sums' (16 + 6
additions of 2^-24 at most each) make at most 2^-19 of the sum, which is what its logarithm is off by.
"""
from __future__ import annotations

import numpy as np
import pytest

import chunk_reference as CR
from conftest import load_mixer
from test_kv4_gpu import ints, result

pytestmark = pytest.mark.gpu

M = load_mixer()


def run_select(ctx, groups, beams, take, logits, scores, done=None, end_id=-1, in_place=False):
    vocab = logits.shape[1]
    n = groups * take
    x, s = ctx.upload(logits), ctx.upload(scores.astype(np.float32))
    d = None if done is None else ints(ctx, done)
    parents, tokens, out = (ctx.upload(np.full(n, -9, np.int32)) for _ in range(3))
    over = ctx.upload(np.full(n, -9, np.int32))
    if in_place:
        out, over = s, d or over
    print(f"case: select groups={groups} beams={beams} take={take} vocab={vocab}", flush=True)
    ctx.beam_select(groups, beams, take, vocab, x, s, d, end_id, parents, tokens, out, over)
    got = [ctx.download(b, (n,), t) for b, t in ((parents, np.int32), (tokens, np.int32), (out, np.float32), (over, np.int32))]
    want = CR.select(groups, beams, take, vocab, logits, scores.astype(np.float32), done, end_id)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
    none = ~np.isfinite(want[2])
    assert (got[2][none] == -np.inf).all()
    off = np.abs(got[2][~none] - want[2][~none])
    assert (off <= 2.0 ** -24 * np.abs(want[2][~none]) + 2.0 ** -19).all()
    assert np.array_equal(ctx.download(x, logits.shape, np.uint32), logits.view(np.uint32))
    return got


def some(seed, groups, beams, vocab):
    rng = np.random.default_rng(seed)
    like = 2 * rng.standard_normal((groups, 1, vocab))
    logits = (like + 0.5 * rng.standard_normal((groups, beams, vocab))).astype(np.float32).reshape(groups * beams, vocab)
    return rng, logits, -5 - 3 * np.abs(rng.standard_normal(groups * beams))


@pytest.mark.parametrize("groups, beams, take, vocab", [
    (1, 1, 1, 1), (1, 1, 4, 3), (1, 4, 4, 7), (2, 3, 5, 1000), (1, 4, 8, 1023), (3, 2, 2, 1024), (1, 5, 3, 1025), (2, 8, 16, 4097), (1, 1, 64, 70),
    (1, 64, 64, 3001), (5, 1, 1, 20000), (1, 4, 4, 248320), (2, 3, 6, 262144)])
def test_select(ctx, groups, beams, take, vocab):
    _, logits, scores = some(vocab + take, groups, beams, vocab)
    run_select(ctx, groups, beams, take, logits, scores)


def test_select_with_sequences_at_their_end(ctx):
    rng, logits, scores = some(1, 3, 4, 5000)
    done = np.zeros(12, np.int32)
    done[[1, 4, 5, 6, 7, 10]] = [1, 1, -3, 2, 1, 7]
    scores[10] = -0.5                                               # the best of all
    logits[8, 77] += 30
    got = run_select(ctx, 3, 4, 8, logits, scores, done, end_id=77)
    assert got[3][:].any() and (got[1][8:12] == 77).all() and (got[1][12:16] == -1).all()
    run_select(ctx, 3, 4, 4, logits, scores, None, end_id=77)


def test_select_of_equal_values(ctx):
    """Ties within a row and between rows of the same logits: the lower row, then the lower token."""
    rng = np.random.default_rng(2)
    logits = np.tile(rng.integers(-3, 4, (1, 5000)).astype(np.float32), (4, 1))
    run_select(ctx, 1, 4, 40, logits, np.array([-1.0, -2.0, -1.0, -2.0]))
    run_select(ctx, 2, 2, 64, np.zeros((4, 70001), np.float32), np.full(4, -3.0))
    run_select(ctx, 1, 64, 64, np.full((64, 4100), -2.5, np.float32), np.zeros(64))


def test_select_leaves_out_what_is_no_sequence_and_no_continuation(ctx):
    rng, logits, scores = some(3, 2, 6, 3000)
    scores[[0, 7, 9]] = [-np.inf, np.nan, np.inf]
    logits[1, 5], logits[2, 2999], logits[3, :] = np.nan, np.inf, -np.inf
    logits[4, :] = -np.inf
    logits[4, [9, 2000]] = [3e38, -3e38]
    logits[10, rng.permutation(3000)[:2900]] = -np.inf
    run_select(ctx, 2, 6, 64, logits, scores)
    run_select(ctx, 1, 2, 3, np.full((2, 9), np.nan, np.float32), np.zeros(2))


def test_select_of_values_of_other_sizes(ctx):
    rng = np.random.default_rng(4)
    for scale in (1e-6, 1e-3, 1e2, 1e6):
        run_select(ctx, 1, 3, 10, (scale * rng.standard_normal((3, 9000))).astype(np.float32), np.array([0.0, -0.0, -1e-3]))


def test_select_of_scores_that_outweigh_the_logits(ctx):
    """A sum that is its row's score in 64 bits is every token's: the lowest are chosen, whatever their logits."""
    rng = np.random.default_rng(6)
    for vocab in (5, 700, 6000):
        logits = rng.standard_normal((4, vocab)).astype(np.float32)
        got = run_select(ctx, 1, 4, 6, logits, np.array([-1e30, -2e30, -1e30, 1.5e30]))
        assert (got[0][:5] == 3).all() and list(got[1][:5]) == [0, 1, 2, 3, 4]
    # and one row beside the others' sums
    logits = (1e30 * rng.standard_normal((2, 3000))).astype(np.float32)
    run_select(ctx, 1, 2, 20, logits, np.array([-1.0, -2e30]))


def test_select_of_logits_past_4_gib(ctx):
    """4480 rows of the largest vocabulary, all but the last request's without a score."""
    groups, beams, vocab = 70, 64, 262144
    rng = np.random.default_rng(8)
    logits = rng.standard_normal((beams, vocab)).astype(np.float32)
    scores = np.full(groups * beams, -np.inf, np.float32)
    scores[-beams:] = -np.abs(rng.standard_normal(beams))
    x = ctx.alloc(groups * beams * vocab * 4)
    try:
        ctx.upload_to(x.offset((groups - 1) * beams * vocab * 4), logits)
        parents, tokens, out = (ctx.upload(np.full(groups * 5, -9, np.int32)) for _ in range(3))
        ctx.beam_select(groups, beams, 5, vocab, x, ctx.upload(scores), None, -1, parents, tokens, out, None)
        want = CR.select(1, beams, 5, vocab, logits, scores[-beams:], None, -1)
        got = [ctx.download(b, (groups, 5), t) for b, t in ((parents, np.int32), (tokens, np.int32), (out, np.float32))]
        assert np.array_equal(got[0][-1], want[0] + (groups - 1) * beams) and np.array_equal(got[1][-1], want[1])
        assert (np.abs(got[2][-1] - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 2.0 ** -19).all()
        assert (got[0][:-1] == -1).all() and (got[1][:-1] == -1).all() and (got[2][:-1] == -np.inf).all()
    finally:
        ctx.sync()
        x.close()


def test_select_in_place(ctx):
    rng, logits, scores = some(5, 3, 4, 2500)
    done = np.array([0, 1, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1], np.int32)
    run_select(ctx, 3, 4, 4, logits, scores, done, end_id=3, in_place=True)


def test_select_log_sums_of_many_equal_logits(ctx):
    """A token in every 1024 leads equal ones d below: what a term and a sum are off by does not average out.

    In units of 2^-24: an exponential is off by 2 (1 ulp of 2^t), by d of the difference's rounding, d of its product's
    and d / 4 of log2(e)'s; equal terms, summed by halves, by nothing more, the sum of the leader's lane by 4; the rest is
    64 bits.  Scores about as large as the log-sums, so that the results are small and their own rounding, half a step,
    is next to nothing."""
    rng = np.random.default_rng(10)
    top = np.concatenate([np.zeros(9), np.round(rng.uniform(-30, 30, 40), 1), [0.1, -1.4, 1.7, 2.2, 0, 1e4]]).astype(np.float32)
    rest = top - np.concatenate([[0.01, 0.018, 0.053, 0.078, 0.107, 0.15, 0.173, 0.371, 0.6], rng.uniform(0, 9, 40),
                                 [8.8, 8.8, 7.5, 7.5, 8, 7]]).astype(np.float32)
    logits = np.repeat(rest[:, None], 262144, 1)
    logits[:, ::1024] = top[:, None]
    d = top.astype(np.float64) - rest
    sums = np.log(256 + (262144 - 256) * np.exp(-d))
    scores = sums.astype(np.float32)
    got = run_select(ctx, len(top), 1, 1, logits, scores)
    want = scores.astype(np.float64) - sums
    off = np.abs(got[2] - want) * 2 ** 24
    w, lane = 1023 * np.exp(-d) / (1 + 1023 * np.exp(-d)), (1 + 15 * np.exp(-d)) / (1 + 1023 * np.exp(-d))
    room = w * (2 + 2.25 * d) + 4 * lane + np.abs(want)
    print("largest, in 2^-24:", off.max(), "of the room:", (off / room).max())
    assert (off <= room).all()


# ---- states --------------------------------------------------------------------------------------
def run_state_fork(ctx, rows, src, dst, sizes, seed=0, refused=False):
    """sizes: (row bytes, stride) of each buffer; everything beside the rows has to stay."""
    rng = np.random.default_rng(seed)
    data = [rng.integers(0, 2 ** 32, rows * stride // 4, dtype=np.uint32) for _, stride in sizes]
    bufs = [ctx.upload(d) for d in data]
    res = ints(ctx, [-77])
    print(f"case: state fork rows={rows} count={len(src)} sizes={sizes}", flush=True)
    ctx.state_fork([(b, *s) for b, s in zip(bufs, sizes)], rows, len(src), ints(ctx, src), None if dst is None else ints(ctx, dst), res)
    assert result(ctx, res) == (-1 if refused else 0)
    for b, d, (size, stride) in zip(bufs, data, sizes):
        want = d.reshape(rows, stride // 4).copy()
        if not refused:
            at = np.arange(len(src)) if dst is None else np.asarray(dst)
            want[at, :size // 4] = d.reshape(rows, stride // 4)[np.asarray(src), :size // 4]
        assert np.array_equal(ctx.download(b, want.shape, np.uint32), want)


SIZES = [(16, 16), (4096, 4096), (4112, 8192), (98304, 98304), (49152, 49168)]


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 96, 128, 129, 200])
def test_state_fork(ctx, rows):
    """Parents at random: chains, cycles, rows that stay, several children of one."""
    rng = np.random.default_rng(rows)
    run_state_fork(ctx, rows, rng.integers(0, rows, rows), None, SIZES, rows)
    run_state_fork(ctx, rows, np.roll(np.arange(rows), 1), None, SIZES[:3], rows)


def test_state_fork_of_listed_rows(ctx):
    rng = np.random.default_rng(6)
    run_state_fork(ctx, 300, [5, 299, 7, 5], [299, 5, 7, 0], SIZES)
    run_state_fork(ctx, 65536, [65535, 3], [3, 65535], [(32, 48)])
    run_state_fork(ctx, 1100, rng.integers(0, 1100, 1024), rng.permutation(1100)[:1024], [(4112, 4112), (160, 176)])
    run_state_fork(ctx, 12, np.arange(12), None, SIZES)


def test_state_fork_of_many_buffers(ctx):
    run_state_fork(ctx, 5, [4, 4, 0, 3, 1], None, [(16 * (i + 1), 16 * (i + 2)) for i in range(64)])


def test_state_fork_of_rows_past_4_gib(ctx):
    stride, size = 2 ** 31 + 4096, 8208
    rng = np.random.default_rng(9)
    rows = rng.integers(0, 256, (3, size), dtype=np.uint8)
    buf = ctx.alloc(2 * stride + size)
    try:
        for r in range(3):
            ctx.upload_to(buf.offset(r * stride), rows[r])
        res = ints(ctx, [-77])
        ctx.state_fork([(buf, size, stride)], 3, 3, ints(ctx, [2, 0, 1]), None, res)
        assert result(ctx, res) == 0
        assert np.array_equal([ctx.download(buf.offset(r * stride), (size,), np.uint8) for r in range(3)], rows[[2, 0, 1]])
    finally:
        ctx.sync()
        buf.close()


@pytest.mark.parametrize("src, dst", [([0, 5], [1, 2]), ([0, -1], [1, 2]), ([0, 1], [5, 2]), ([0, 1], [2, 2]), ([0, 1], [-1, 2]),
                                      ([1, 1], [1, 1])])
def test_state_fork_refused_lists_change_nothing(ctx, src, dst):
    run_state_fork(ctx, 5, src, dst, SIZES, refused=True)
    run_state_fork(ctx, 70, list(range(3, 63)) + [src[0] if src[0] != 5 else 70, src[1] if src[1] != 5 else 70],
                   list(range(3, 63)) + [d if d != 5 else 70 for d in dst], SIZES, refused=True)


def test_selection_and_states_in_a_graph():
    """Captured once; replays follow the scores, flags and states that they change themselves."""
    rng, logits, scores = some(7, 2, 3, 4000)
    own = M.Context(0)
    own.reserve(6)
    state = rng.integers(0, 2 ** 32, (6, 6000), dtype=np.uint32)
    x, s, d = own.upload(logits), own.upload(scores.astype(np.float32)), own.upload(np.zeros(6, np.int32))
    st, parents, tokens, res = own.upload(state), own.alloc(24), own.alloc(24), own.alloc(4)

    def enqueue():
        own.beam_select(2, 3, 3, 4000, x, s, d, 11, parents, tokens, s, d)
        own.state_fork([(st, 24000, 24000)], 6, 6, parents, None, res)

    own.graph_begin()
    enqueue()
    graph = own.graph_end()
    at, done = scores.astype(np.float32), np.zeros(6, np.int32)
    for i in range(5):
        logits = logits + (2 * rng.standard_normal(logits.shape)).astype(np.float32)
        logits[rng.integers(0, 6), 11] += 12
        own.upload(logits, x)
        if i == 3:
            enqueue()
        else:
            graph.launch()
        want = CR.select(2, 3, 3, 4000, logits, at, done, 11)
        at = own.download(s, (6,), np.float32)
        done = own.download(d, (6,), np.int32)
        assert np.array_equal(own.download(parents, (6,), np.int32), want[0])
        assert np.array_equal(own.download(tokens, (6,), np.int32), want[1]) and np.array_equal(done, want[3])
        assert (np.abs(at - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 2.0 ** -19).all()
        state = state[want[0]]
        assert result(own, res) == 0 and np.array_equal(own.download(st, state.shape, np.uint32), state)
    assert done.any()
    graph.close()
    own.close()

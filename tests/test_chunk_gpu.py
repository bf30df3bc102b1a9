"""GPU: chunks of new tokens over the paged 4-bit KV cache against numpy in 64 bits (tests/chunk_reference.py).

What is appended has to be the reference's, byte for byte.  Attention's outputs are bf16: off by half a step,
2^-8 of themselves, beside the bound that chunk_reference.attend derives for what is rounded before.  Over all
outputs the roundings are independent: that of a bf16 is 2^-8 / sqrt(3) = 2.3e-3 of the value at most in the
2-norm, those of q, K, V and p to f16 together at most sqrt(6) 2^-11 / sqrt(3) times |score| (about 2) = 1.4e-3; the bar is 3e-3.
"""
from __future__ import annotations

import numpy as np
import pytest

import chunk_reference as CR
import kv4_reference as R
from conftest import load_mixer
from test_kv4_gpu import assert_same, ints, result, run_fork, run_resize, upload

pytestmark = pytest.mark.gpu

M = load_mixer()
FILL = 0x4141


def rope(n):
    return M.rope_table(max(n, 8))


def cache_of(lens, layers=2, spare=3, seed=0, room=0):
    """A numpy cache whose rows have these lengths, in scattered pages of values, its unused tokens random bytes."""
    most = max(1, R.pages_of(max(lens) + room))
    pages = sum(R.pages_of(n) for n in lens) + spare
    ref = R.Cache(layers, pages, len(lens), most, seed=seed)
    assert ref.resize(None, list(lens)) == 0
    perm = np.random.default_rng(seed + 1).permutation(pages)
    ref.table = np.where(ref.table >= 0, perm[np.maximum(ref.table, 0)], -1).astype(np.int32)
    refs = np.zeros_like(ref.refs)
    refs[perm] = ref.refs
    ref.refs = refs
    rng = np.random.default_rng(seed + 2)
    for r, n in enumerate(lens):
        for j in range(R.pages_of(n)):
            fill_page(ref.pages[:, ref.table[r, j]], min(R.TOKENS, n - j * R.TOKENS), rng)
    return ref


def fill_page(pages, n, rng):
    """The first n tokens of a page of every layer: scales and minima of ordinary values beside the random codes."""
    for layer in range(pages.shape[0]):
        for half in range(8):
            meta = pages[layer, half * R.HALF_BYTES + 8192:(half + 1) * R.HALF_BYTES].view(np.float16)
            for t in range(32):
                if 32 * (half % 2) + t >= n:
                    continue
                for is_v in (0, 1):
                    s = rng.uniform(0.1, 0.3, 4).astype(np.float16)
                    meta[256 * is_v + R.S_AT[t]] = s
                    meta[256 * is_v + 128 + R.LO_AT[t]] = (-7.5 * s.astype(np.float64) * rng.uniform(0.8, 1.2, 4)).astype(np.float16)


def queries(rng, tokens):
    q = CR.bf16(rng.standard_normal((tokens, 16, 512)))
    return q, (0.1 * rng.standard_normal(256)).astype(np.float16)


def begins_of(news, start=0):
    return np.concatenate([[start], start + np.cumsum(news)]).astype(np.int32)


def run_chunk(ctx, ref, news, slots=None, layer=1, max_new=None, max_len=None, res=None, tokens=None, begins=None, seed=3, c=None):
    """The call on the device and in numpy: outputs have to agree, rows of nobody to stay.  The bf16 outputs."""
    begins = begins_of(news) if begins is None else np.asarray(begins, np.int32)
    tokens = int(begins.max()) if tokens is None else tokens
    batch = len(begins) - 1
    max_new = max_new or max(1, int(np.diff(begins).max()))
    max_len = max_len or max(1, int(ref.lens.max()))
    q, gamma = queries(np.random.default_rng(seed), tokens)
    cos, sin = rope(max_len)
    c = upload(ctx, ref) if c is None else c
    out = ctx.upload(np.full((tokens, 16, 256), FILL, np.uint16))
    print(f"case: chunk lens={ref.lens[:8]} begins={begins[:9]} slots={slots} max_new={max_new} max_len={max_len}", flush=True)
    ctx.gqa_chunk_kv4(c, layer, batch, None if slots is None else ints(ctx, slots), ints(ctx, begins), tokens, max_new,
                      ctx.upload(q), ctx.upload(gamma.view(np.uint16)), ctx.upload(cos), ctx.upload(sin), len(cos), max_len,
                      None if res is None else ints(ctx, [res]), out)
    got = ctx.download(out, (tokens, 16, 256), np.uint16)
    want, bound, touched = CR.attend(ref, layer, batch, slots, begins, tokens, max_new, CR.bf16_value(q), gamma, cos, sin, max_len)
    if res:
        want[touched] = 0
    assert (got[~touched] == FILL).all()
    assert_near(CR.bf16_value(got[touched]), want[touched], bound[touched])
    return got


def assert_near(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    got, want, bound = got[fine].astype(np.float64), want[fine], bound[fine]
    if not want.size:
        return
    off = np.abs(got - want)
    room = bound + 2.0 ** -8 * (np.abs(want) + bound)
    assert (off <= room).all(), (off - room).max()
    assert np.linalg.norm(off) <= 3e-3 * np.linalg.norm(want)


# ---- appending -------------------------------------------------------------------------------
def run_append(ctx, ref, news, slots=None, layer=1, dtype="f32", max_len=None, res=None, begins=None, tokens=None, seed=5, k=None, v=None):
    begins = begins_of(news) if begins is None else np.asarray(begins, np.int32)
    tokens = int(begins.max()) if tokens is None else tokens
    max_len = max_len or max(1, int(ref.lens.max()))
    rng = np.random.default_rng(seed)
    k = rng.standard_normal((tokens, 4, 256)) * (1 + np.abs(rng.standard_normal(256))) if k is None else k
    v = 0.7 * rng.standard_normal((tokens, 4, 256)) if v is None else v
    gamma = (0.1 * rng.standard_normal(256)).astype(np.float16)
    cos, sin = rope(max_len)
    with np.errstate(over="ignore"):
        k, v = (CR.bf16(x) if dtype == "bf16" else x.astype(np.float32) for x in (k, v))
    c = upload(ctx, ref)
    print(f"case: append {dtype} lens={ref.lens[:8]} begins={begins[:9]} slots={slots}", flush=True)
    ctx.kv4_append(c, layer, len(begins) - 1, None if slots is None else ints(ctx, slots), ints(ctx, begins), tokens, ctx.upload(k),
                   ctx.upload(v), ctx.upload(gamma.view(np.uint16)), ctx.upload(cos), ctx.upload(sin), len(cos), max_len,
                   None if res is None else ints(ctx, [res]), dtype=M.QM_BF16 if dtype == "bf16" else M.QM_F32)
    if not res:
        values = [CR.bf16_value(x) if dtype == "bf16" else x for x in (k, v)]
        CR.append(ref, layer, len(begins) - 1, slots, begins, tokens, *values, gamma, cos, sin, max_len)
    assert_same(ctx, c, ref)
    return c, k, v, gamma


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens, news", [
    ([1], [1]), ([31], [31]), ([32], [1]), ([33], [2]), ([64], [64]), ([65], [1]), ([97], [34]), ([130], [66]), ([100, 40, 7], [33, 40, 1]),
    ([64, 1, 200, 65], [2, 1, 37, 64])])
def test_append(ctx, lens, news, dtype):
    """Every byte of the pool is the reference's: the new tokens', and the others of their words and pages."""
    run_append(ctx, cache_of(lens, seed=len(lens) + sum(news)), news, dtype=dtype)


def test_append_slots_and_rows_without_tokens(ctx):
    """Slots out of order; a batch row of no tokens, one outside the table, one that an earlier batch row has."""
    ref = cache_of([40, 70, 130, 9, 64], seed=8)
    run_append(ctx, ref, [5, 0, 7, 20, 3, 2], slots=[3, 1, 9, 2, 0, 2])


def test_append_of_more_rows_than_a_wave(ctx):
    rng = np.random.default_rng(9)
    lens = rng.integers(1, 80, 150).tolist()
    news = [int(rng.integers(0, n + 1)) for n in lens]
    run_append(ctx, cache_of(lens, layers=1, seed=9), news, layer=0, slots=rng.permutation(150))


def test_append_refused_rows_and_lists(ctx):
    """More new tokens than the length, a length over max_len, ranges that are none: passed over; the others written."""
    ref = cache_of([10, 90, 20, 30], seed=10)
    run_append(ctx, ref, [11, 3, 5, 6], max_len=64)
    ref = cache_of([10, 90, 20, 30], seed=11)
    run_append(ctx, ref, None, begins=[-1, 4, 4, 9, 200], tokens=12)


def test_append_after_a_refused_resize_writes_nothing(ctx):
    run_append(ctx, cache_of([10, 90], seed=12), [4, 9], res=3)


def test_append_leaves_pages_of_others_alone(ctx):
    """Pages that two rows hold, that by refs none does, and entries that are no page."""
    ref = cache_of([200, 128, 190, 70], seed=13)
    ref.table[1, 0] = ref.table[0, 1]
    ref.refs[ref.table[0, 1]] = 2
    ref.refs[ref.table[2, 1]] = 0
    ref.table[3, 0] = len(ref.refs)
    run_append(ctx, ref, [150, 100, 160, 70])


def test_append_of_infinities_and_nan(ctx):
    """A group with one reads back as NaN, the others as ever; the norm of a row with one is NaN or 0 as the formula's."""
    rng = np.random.default_rng(14)
    k, v = rng.standard_normal((2, 40, 4, 256))
    v[3, 1, 70], v[9, 2, 5], v[11, 0, 255] = np.nan, np.inf, 1e30
    k[5, 2, 100] = np.nan
    ref = cache_of([70], seed=14)
    run_append(ctx, ref, [40], k=k, v=v)


@pytest.mark.parametrize("n", [1, 64, 65, 300])
def test_append_is_what_the_decode_step_appends(ctx, n):
    ref = cache_of([n], seed=15)
    c, k, v, gamma = run_append(ctx, ref, [1], layer=1)
    cos, sin = rope(n)
    d = upload(ctx, ref)
    ctx.memset(d.pages, 0, d.pages.nbytes)
    ctx.copy(d.pages, c.pages, c.pages.nbytes)
    q = np.random.default_rng(1).standard_normal((1, 16, 512)).astype(np.float32)
    out = ctx.alloc(16 * 256 * 4)
    ctx.gqa_decode_kv4(d, 1, 1, None, ctx.upload(q), ctx.upload(k), ctx.upload(v), ctx.upload(gamma.view(np.uint16)),
                       ctx.upload(gamma.view(np.uint16)), ctx.upload(cos), ctx.upload(sin), len(cos), n, None, out)
    assert_same(ctx, d, ref)


# ---- attention ---------------------------------------------------------------------------------
@pytest.mark.parametrize("n, new", [
    (1, 1), (2, 1), (31, 2), (32, 32), (33, 1), (63, 63), (64, 1), (64, 64), (65, 1), (65, 65), (66, 3), (96, 4), (127, 5), (128, 8), (129, 16),
    (130, 17), (200, 31), (200, 33), (257, 100), (320, 256), (500, 129), (700, 1), (1000, 4)])
def test_chunk_lengths(ctx, n, new):
    run_chunk(ctx, cache_of([n], seed=n), [new])


@pytest.mark.parametrize("lens, news", [
    ([5, 70, 130], [5, 1, 64]), ([300, 1, 64, 65], [1, 1, 1, 1]), ([64, 200, 90, 33, 257], [3, 130, 90, 0, 16]), ([900, 40], [2, 40])])
def test_chunk_batches(ctx, lens, news):
    run_chunk(ctx, cache_of(lens, seed=sum(lens)), news)


def test_chunk_slots(ctx):
    """Slots out of order, outside the table, of an empty row, one slot twice; rows of nobody stay as they were."""
    ref = cache_of([100, 0, 64, 150, 10], seed=21)
    run_chunk(ctx, ref, None, slots=[3, -1, 1, 3, 0, 7], begins=[2, 22, 25, 30, 95, 100, 103], tokens=110)


@pytest.mark.parametrize("lens, news", [([900], [1]), ([900, 70], [2, 2]), ([1500, 600], [20, 5]), ([3000, 64], [32, 1]), ([1200], [33])])
def test_chunk_with_a_loose_bound_of_the_rows_new_tokens(ctx, lens, news):
    """A bound past the call's tokens, as a captured call has it: the same bits as with the least that is true."""
    ref = cache_of(lens, layers=1, seed=sum(lens))
    assert np.array_equal(run_chunk(ctx, ref, news, layer=0, max_new=4096), run_chunk(ctx, ref, news, layer=0, max_new=sum(news)))


def test_chunk_refused_rows(ctx):
    """More new tokens than max_new or than the length, a length over max_len: NaN; ranges that are none: nothing."""
    ref = cache_of([10, 90, 20, 30, 60], seed=22)
    run_chunk(ctx, ref, [11, 3, 20, 6, 70], max_len=64, max_new=19)
    run_chunk(ctx, ref, None, begins=[-1, 4, 4, 9, 200, 3], tokens=12, max_new=9)
    run_chunk(ctx, ref, [10, 4, 5, 6, 7], res=2)
    run_chunk(ctx, ref, [10, 4, 5, 6, 7], res=-1)


def test_chunk_of_more_rows_than_a_wave(ctx):
    rng = np.random.default_rng(23)
    lens = rng.integers(1, 90, 140).tolist()
    news = [int(rng.integers(0, n + 1)) for n in lens]
    run_chunk(ctx, cache_of(lens, layers=1, seed=23), news, layer=0, slots=rng.permutation(140))


@pytest.mark.parametrize("n, new", [(6001, 70), (9000, 3), (5000, 300), (20011, 1), (20011, 64)])
def test_chunk_of_long_rows(ctx, n, new):
    """Row blocks whose pages fall to several workgroups."""
    run_chunk(ctx, cache_of([n], layers=1, seed=n), [new], layer=0)


def test_chunk_ragged_and_long(ctx):
    run_chunk(ctx, cache_of([3000, 10, 700, 4097, 1], layers=1, seed=25), [65, 10, 300, 2, 1], layer=0, slots=[0, 1, 2, 3, 4])


def test_chunk_over_shared_pages(ctx):
    """Rows forked from one prompt, grown apart."""
    ref = cache_of([150, 0, 0], seed=26, spare=12, room=100)
    assert ref.fork([0, 0], [1, 2]) == 0 and ref.resize([0, 1, 2], [155, 190, 161]) == 0
    rng = np.random.default_rng(27)
    for r in range(3):
        for j in range(2, R.pages_of(int(ref.lens[r]))):
            fill_page(ref.pages[:, ref.table[r, j]], 64, rng)
    run_chunk(ctx, ref, [5, 40, 11])


def test_chunk_entries_that_are_no_page(ctx):
    """Tokens in them are not seen; a query that sees no others gives 0."""
    ref = cache_of([200, 70, 64], seed=28)
    ref.table[0, 1], ref.table[1, 0], ref.table[2, 0] = len(ref.refs), -3, -1
    run_chunk(ctx, ref, [100, 70, 64])


@pytest.mark.parametrize("at", [0, 37, 63, 64, 90, 127, 128, 139])
@pytest.mark.parametrize("is_v", [0, 1])
def test_chunk_nan_reaches_those_that_see_it(ctx, at, is_v):
    """A token's NaN group: queries before it are as without it, heads of the other kv heads too; V's only in its dims."""
    ref = cache_of([140], seed=29)
    half = ref.pages[1, ref.table[0, at // 64]][R.HEAD_BYTES * 2 + at % 64 // 32 * R.HALF_BYTES:][:R.HALF_BYTES]
    meta = half[8192:].view(np.float16)
    meta[256 * is_v + R.S_AT[at % 32, 1]] = meta[256 * is_v + 128 + R.LO_AT[at % 32, 1]] = np.nan
    got = CR.bf16_value(run_chunk(ctx, ref, [100]))
    first = max(0, at - 40)
    assert not np.isnan(got[:first]).any() and np.isnan(got[first:, 8:12, 64:128]).all()


def test_chunk_values_at_the_edges_of_f16(ctx):
    """Groups that reach to f16's largest values stay finite: a scale that would take them past it is a step less."""
    ref = cache_of([100], seed=30)
    meta = ref.pages[1, ref.table[0, 0]][R.HEAD_BYTES:][:R.HALF_BYTES][8192:].view(np.float16)
    meta[256 + R.S_AT[7]], meta[256 + 128 + R.LO_AT[7]] = np.float16(8736), np.float16(-65504)       # lo + 15 s = 65536
    meta[256 + R.S_AT[9]], meta[256 + 128 + R.LO_AT[9]] = np.float16(6e-8), np.float16(1e-7)
    run_chunk(ctx, ref, [60])


@pytest.mark.parametrize("n", [1, 40, 257, 1500])
def test_one_token_is_the_decode_steps(ctx, n):
    """The step appends and attends in f32; the call over what it appended gives the same, rounded."""
    ref = cache_of([n], seed=31)
    rng = np.random.default_rng(32)
    q, gamma = queries(rng, 1)
    k, v = rng.standard_normal((2, 1, 4, 256)).astype(np.float32)
    cos, sin = rope(n)
    c = upload(ctx, ref)
    out = ctx.alloc(16 * 256 * 4)
    norm, qf = ctx.upload(gamma.view(np.uint16)), ctx.upload(CR.bf16_value(q))
    rc, rs = ctx.upload(cos), ctx.upload(sin)
    ctx.gqa_decode_kv4(c, 1, 1, None, qf, ctx.upload(k), ctx.upload(v), norm, norm, rc, rs, len(cos), n, None, out)
    want = ctx.download(out, (1, 16, 256), np.float32)
    CR.append(ref, 1, 1, None, [0, 1], 1, k, v, gamma, cos, sin, n)
    assert_same(ctx, c, ref)
    out16 = ctx.alloc(16 * 256 * 2)
    ctx.gqa_chunk_kv4(c, 1, 1, None, ints(ctx, [0, 1]), 1, 1, ctx.upload(q), norm, rc, rs, len(cos), n, None, out16)
    _, bound, _ = CR.attend(ref, 1, 1, None, [0, 1], 1, 1, CR.bf16_value(q), gamma, cos, sin, n)
    assert_near(CR.bf16_value(ctx.download(out16, (1, 16, 256), np.uint16)), want.astype(np.float64), bound + 2e-5 * np.abs(want).max())


# ---- together, captured, elsewhere ------------------------------------------------------------
def test_prompts_in_parts_in_a_graph(ctx):
    """Grow, append, attend, captured once and replayed as the rows' lists change; every replay as the eager call."""
    rng = np.random.default_rng(40)
    rows, tokens = 3, 96
    ref = R.Cache(1, 40, rows, 8, seed=41)
    steps = [([40, 0, 7], None), ([1, 64, 31], [2, 0, 1]), ([30, 30, 36], None), ([0, 0, 90], None), ([1, 1, 1], [1, 2, 0])]
    cos, sin = rope(512)
    gamma = (0.1 * rng.standard_normal(256)).astype(np.float16)
    own = M.Context(0)
    own.reserve(rows, 512, tokens)
    c = upload(own, ref)
    bufs = {key: own.alloc(size) for key, size in (("q", tokens * 16384), ("k", tokens * 2048), ("v", tokens * 2048),
                                                    ("out", tokens * 8192), ("begins", 16), ("slots", 16), ("add", 16), ("res", 16))}
    norm, rc, rs = own.upload(gamma.view(np.uint16)), own.upload(cos), own.upload(sin)

    def enqueue():
        own.kv4_resize(c, rows, bufs["slots"], bufs["add"], bufs["res"], M.QM_KV4_ADD)
        own.kv4_append(c, 0, rows, bufs["slots"], bufs["begins"], tokens, bufs["k"], bufs["v"], norm, rc, rs, 512, 512, bufs["res"],
                       dtype=M.QM_BF16)
        own.gqa_chunk_kv4(c, 0, rows, bufs["slots"], bufs["begins"], tokens, tokens, bufs["q"], norm, rc, rs, 512, 512, bufs["res"],
                          bufs["out"])

    own.graph_begin()
    enqueue()
    graph = own.graph_end()
    for i, (news, slots) in enumerate(steps):
        slots = slots or list(range(rows))
        begins = begins_of(news)
        q = CR.bf16(rng.standard_normal((tokens, 16, 512)))
        k, v = (CR.bf16(rng.standard_normal((tokens, 4, 256))) for _ in range(2))
        for key, arr in (("q", q), ("k", k), ("v", v), ("begins", begins), ("slots", np.asarray(slots, np.int32)),
                         ("add", np.asarray(news, np.int32)), ("out", np.full((tokens, 16, 256), FILL, np.uint16))):
            own.upload(arr, bufs[key])
        print(f"case: graph step {i}", flush=True)
        if i == 2:
            enqueue()                                                   # eager in between
        else:
            graph.launch()
        assert result(own, bufs["res"]) == ref.resize(slots, news, add=True) == 0
        CR.append(ref, 0, rows, slots, begins, tokens, CR.bf16_value(k), CR.bf16_value(v), gamma, cos, sin, 512)
        assert_same(own, c, ref)
        want, bound, touched = CR.attend(ref, 0, rows, slots, begins, tokens, tokens, CR.bf16_value(q), gamma, cos, sin, 512)
        got = own.download(bufs["out"], (tokens, 16, 256), np.uint16)
        assert (got[~touched] == FILL).all()
        assert_near(CR.bf16_value(got[touched]), want[touched], bound[touched])
    graph.close()
    own.close()


def test_a_chunk_that_would_grow_the_workspace_under_capture_is_refused():
    own = M.Context(0)
    ref = cache_of([3000], layers=1, seed=42)
    c = upload(own, ref)
    z = own.alloc(70 * 16384)
    begins = ints(own, [0, 70])
    own.graph_begin()
    with pytest.raises(M.MixerError) as e:
        own.gqa_chunk_kv4(c, 0, 1, None, begins, 70, 70, z, z, z, z, 3000, 3000, None, z)
    assert e.value.code == 9
    own.graph_end().close()
    own.close()


def test_chunk_on_a_stream_of_the_callers(ctx):
    import ctypes
    s = ctypes.c_void_p(0)
    ctx._check(ctx.lib.qm_stream_create(ctx.h, ctypes.byref(s)))
    before, ctx.stream = ctx.stream, s.value
    try:
        ref = cache_of([333], seed=43)
        run_append(ctx, ref, [90], dtype="bf16")
        run_chunk(ctx, ref, [90])
    finally:
        ctx.sync()
        ctx.stream = before
        ctx._check(ctx.lib.qm_stream_destroy(ctx.h, s))


def test_a_chunk_twice_gives_the_same_bits(ctx):
    ref = cache_of([2500, 80], layers=1, seed=44)
    a = run_chunk(ctx, ref, [130, 80], layer=0)
    b = run_chunk(ctx, ref, [130, 80], layer=0)
    assert np.array_equal(a, b)


# ---- more row blocks than workgroups, and few of unequal lengths ---------------------------------
def many_rows(seed, rows, lo, hi, top, long=()):
    rng = np.random.default_rng(seed)
    lens = rng.integers(lo, hi + 1, rows).tolist()
    news = [int(rng.integers(1, min(n, top) + 1)) for n in lens]
    for at, n, new in long:
        lens[at], news[at] = n, new
    return lens, news


@pytest.mark.parametrize("seed, rows, lo, hi, top, long", [
    (50, 40, 70, 300, 129, []),                                          # runs of blocks of many tokens
    (51, 60, 1, 200, 70, [(7, 5000, 40), (30, 2500, 70)]),               # of both kinds, long ones among them
    (52, 100, 1, 130, 40, [(64, 6000, 100), (99, 3000, 1)]),             # more rows than lanes
    (53, 70, 20, 200, 20, [(3, 4000, 32)]),                              # few tokens, two operand columns
    (54, 100, 1, 100, 4, [(0, 5000, 4), (71, 2000, 3)]),                 # few tokens, one
    (55, 3, 60, 70, 60, [(0, 4200, 500), (2, 9000, 33)]),                # few blocks, cut unevenly
    (56, 14, 150, 290, 150, []),                                         # blocks of many tokens, none cut
    (57, 9, 400, 512, 250, []),                                          # and where they are
    (58, 8, 33, 64, 64, []),                                             # a call of blocks of few only
    (59, 2, 300, 400, 60, [(0, 4000, 440)])])
def test_chunk_of_many_row_blocks(ctx, seed, rows, lo, hi, top, long):
    lens, news = many_rows(seed, rows, lo, hi, top, long)
    run_chunk(ctx, cache_of(lens, layers=1, seed=seed), news, layer=0, seed=seed)


@pytest.mark.parametrize("news, max_new", [([300, 3, 2, 40], 3), ([300, 30, 2, 40], 32), ([900, 130, 2, 700], 200), ([900, 130, 2, 700], 131)])
def test_chunk_refused_rows_beside_long_ones(ctx, news, max_new):
    """Refused and idle rows of any number of tokens: theirs are NaN and 0, the others' shares are joined as ever."""
    ref = cache_of([1000, 5000, 3000, 800], layers=1, seed=62)
    run_chunk(ctx, ref, news, layer=0, max_new=max_new)
    run_chunk(ctx, ref, news, layer=0, max_new=max_new, slots=[-1, 1, 2, 7])


@pytest.mark.parametrize("n, new", [(600, 64), (1100, 40), (700, 300)])
def test_chunk_of_one_longer_row_among_many_of_a_token(ctx, n, new):
    """An even share that is less than a page of the longer row's blocks: no share of a block is empty, and what an
    earlier call left in the workspace is not joined."""
    run_chunk(ctx, cache_of([6001], layers=1, seed=61), [70], layer=0)
    run_chunk(ctx, cache_of([50] * 69 + [n], layers=1, seed=60), [1] * 69 + [new], layer=0)


def test_chunk_of_a_prompt_of_more_blocks_than_workgroups(ctx):
    run_chunk(ctx, cache_of([2200, 2100], layers=1, seed=56), [2200, 2000], layer=0)


def test_chunk_ranges_that_overlap_stay_within_the_call(ctx):
    """Ranges have to ascend; of ones that do not, nothing but their own rows is written."""
    ref = cache_of([50] * 9, layers=1, seed=57)
    q, gamma = queries(np.random.default_rng(57), 60)
    cos, sin = rope(50)
    c, out = upload(ctx, ref), ctx.upload(np.full((60, 16, 256), FILL, np.uint16))
    for max_new in (3, 20, 50):
        ctx.gqa_chunk_kv4(c, 0, 9, None, ints(ctx, [4, 50, 3, 49, 4, 50, 4, 50, 4, 50]), 50, max_new, ctx.upload(q), ctx.upload(gamma.view(np.uint16)),
                          ctx.upload(cos), ctx.upload(sin), len(cos), 50, None, out)
    got = ctx.download(out, (60, 16, 256), np.uint16)
    assert (got[50:] == FILL).all() and (got[:3] == FILL).all()
    assert_same(ctx, c, ref)
    run_chunk(ctx, ref, [5] * 9, layer=0)


@pytest.mark.parametrize("new", [1, 40])
def test_two_graphs_share_the_workspace(new):
    """Captured one after the other, replayed in turn with eager calls between: each as if alone."""
    own = M.Context(0)
    own.reserve(2, 5000, 100)
    lens = [[3000, 700], [450, 4900]]
    refs = [cache_of(n, layers=1, seed=58 + i, room=5000 - max(n)) for i, n in enumerate(lens)]
    caches = [upload(own, r) for r in refs]
    q, gamma = queries(np.random.default_rng(59), 2 * new)
    cos, sin = rope(5000)
    up = [own.upload(x) for x in (q, gamma.view(np.uint16), cos, sin)]
    begins = ints(own, [0, new, 2 * new])
    outs = [own.alloc(2 * new * 8192) for _ in refs]

    def call(i):
        own.gqa_chunk_kv4(caches[i], 0, 2, None, begins, 2 * new, new, *up, len(cos), 5000, None, outs[i])

    graphs = []
    for i in range(2):
        own.graph_begin()
        call(i)
        graphs.append(own.graph_end())
    wants = [CR.attend(r, 0, 2, None, [0, new, 2 * new], 2 * new, new, CR.bf16_value(q), gamma, cos, sin, 5000) for r in refs]
    for i in (0, 1, 1, 0, 1):
        for o in outs:
            own.upload(np.full((2 * new, 16, 256), FILL, np.uint16), o)
        call(1 - i)
        graphs[i].launch()
        for o, (want, bound, _) in zip(outs, wants):
            assert_near(CR.bf16_value(own.download(o, (2 * new, 16, 256), np.uint16)), want, bound)
    for g in graphs:
        g.close()
    own.close()


def test_pages_past_4_gib(ctx):
    """A pool of 4.5 GB, the row's pages at its end: what is appended and attended is as in a small one."""
    small = cache_of([700], layers=1, seed=63)
    pages, base = small.pages.shape[1], 61000 - small.pages.shape[1]
    c = M.Kv4Cache(ctx, 1, 61000, 1, small.table.shape[1])
    try:
        at = c.pages.offset(base * R.PAGE)
        assert at - c.pages.ptr > 2 ** 32
        refs = np.zeros(61000, np.int32)
        refs[base:] = small.refs
        ctx.upload_to(at, small.pages)
        for buf, arr in ((c.table, np.where(small.table >= 0, small.table + base, -1).astype(np.int32)), (c.lens, small.lens), (c.refs, refs)):
            ctx.upload(arr, buf)
        rng = np.random.default_rng(64)
        cos, sin = rope(700)
        rc, rs = ctx.upload(cos), ctx.upload(sin)
        for new in (3, 20, 600):
            k, v = (CR.bf16(rng.standard_normal((new, 4, 256))) for _ in range(2))
            q, gamma = queries(rng, new)
            norm, begins, out = ctx.upload(gamma.view(np.uint16)), ints(ctx, [0, new]), ctx.alloc(new * 8192)
            print(f"case: 4 GiB new={new}", flush=True)
            ctx.kv4_append(c, 0, 1, None, begins, new, ctx.upload(k), ctx.upload(v), norm, rc, rs, len(cos), 700, None, dtype=M.QM_BF16)
            ctx.gqa_chunk_kv4(c, 0, 1, None, begins, new, new, ctx.upload(q), norm, rc, rs, len(cos), 700, None, out)
            CR.append(small, 0, 1, None, [0, new], new, CR.bf16_value(k), CR.bf16_value(v), gamma, cos, sin, 700)
            assert np.array_equal(ctx.download(at, small.pages.shape, np.uint8), small.pages)
            want, bound, _ = CR.attend(small, 0, 1, None, [0, new], new, new, CR.bf16_value(q), gamma, cos, sin, 700)
            assert_near(CR.bf16_value(ctx.download(out, (new, 16, 256), np.uint16)), want, bound)
    finally:
        ctx.sync()
        c.pages.close()

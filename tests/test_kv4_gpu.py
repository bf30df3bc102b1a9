"""GPU: the paged 4-bit KV cache against its numpy form (tests/kv4_reference.py).

Codes, scales, tables, lengths and counts have to be equal.  Attention outputs (f32) are compared with
64 bits: a score is a sum of 256 products in f32, each partial sum rounded by at most 2^-24 of itself; for
the values here (|score| about 3) independent roundings add up to about 2^-24 * 16 * 3 = 3e-6, which is the
relative error of a probability and so of an output, whose own sums add about as much.  The bar is 2e-5 of
the outputs' 2-norm; a single output may be 2^-24 * 6 * (sqrt(272) * 2 A + sqrt(n)) * V off, A the sum of
the absolute products of a score and V the largest value (six deviations of the same sums, taken at their
largest terms: A up to 200, V up to 6).
"""
from __future__ import annotations

import numpy as np
import pytest

import kv4_reference as R
from conftest import load_mixer
from test_kv4 import some_steps

pytestmark = pytest.mark.gpu

M = load_mixer()


def upload(ctx, ref: R.Cache):
    """A device cache that holds what the numpy one does."""
    layers, num_pages, _ = ref.pages.shape
    c = M.Kv4Cache(ctx, layers, num_pages, *ref.table.shape)
    for buf, arr in ((c.pages, ref.pages), (c.table, ref.table), (c.lens, ref.lens), (c.refs, ref.refs)):
        ctx.upload(arr, buf)
    return c


def ints(ctx, values):
    return ctx.upload(np.asarray(values, np.int32))


def result(ctx, buf):
    return int(ctx.download(buf, (1,), np.int32)[0])


def assert_same(ctx, c, ref: R.Cache, pages=True):
    assert np.array_equal(ctx.download(c.lens, ref.lens.shape, np.int32), ref.lens)
    assert np.array_equal(ctx.download(c.refs, ref.refs.shape, np.int32), ref.refs)
    assert np.array_equal(ctx.download(c.table, ref.table.shape, np.int32), ref.table)
    if pages:
        assert np.array_equal(ctx.download(c.pages, ref.pages.shape, np.uint8), ref.pages)


def run_resize(ctx, c, rows, lens, add=False):
    res = ints(ctx, [-77])
    ctx.kv4_resize(c, len(lens), None if rows is None else ints(ctx, rows), ints(ctx, lens), res,
                   M.QM_KV4_ADD if add else M.QM_KV4_LENS)
    return result(ctx, res)


def run_fork(ctx, c, src, dst):
    res = ints(ctx, [-77])
    ctx.kv4_fork(c, len(src), ints(ctx, src), ints(ctx, dst), res)
    return result(ctx, res)


def run_compact(ctx, c):
    res = ints(ctx, [-77])
    ctx.kv4_compact(c, res)
    return result(ctx, res)


def kv_rows(rng, *lead):
    """f16 rows with channels of unequal size, and tokens that are exactly on the borders of codes."""
    k = (rng.standard_normal((*lead, 256)) * (1 + np.abs(rng.standard_normal(256)))).astype(np.float16)
    v = (0.7 * rng.standard_normal((*lead, 256))).astype(np.float16)
    v[..., ::3, :] = (rng.integers(0, 31, v[..., ::3, :].shape) * 0.25 - 2).astype(np.float16)    # steps of half a code
    v[..., ::3, ::64], v[..., ::3, 63::64] = -2.0, 5.5                                            # s = 0.5: ties
    return k, v


# ---- store and load -------------------------------------------------------------------------
@pytest.mark.parametrize("batch, n, first, spare", [
    (1, 1, None, 0), (1, 1, [63], 2), (1, 31, None, 1), (1, 32, [32], 0), (2, 33, [0, 31], 5), (1, 45, None, 0),
    (1, 64, [64], 0), (3, 100, [0, 37, 200], 3), (1, 129, [95], 0), (2, 7, [60, 28], 9)])
def test_store_and_load(ctx, batch, n, first, spare):
    """Every byte of the pool after a store is the reference's (the other tokens of a word and page with it), and a
    load gives the stored values; f16 rows past the tokens stay as they were."""
    rng = np.random.default_rng(n)
    at = first or [0] * batch
    ref = R.Cache(2, 40, batch + 2, 6, seed=n)
    lens = [f + n + (7 if b else 0) for b, f in enumerate(at)]
    assert ref.resize(list(range(1, batch + 1)), lens) == 0
    ref.table[1:batch + 1] = np.where(ref.table[1:batch + 1] >= 0, 39 - ref.table[1:batch + 1], -1)      # scattered
    ref.refs = ref.refs[::-1].copy()
    cap = n + spare
    k, v = kv_rows(rng, batch, 4, cap)
    c = upload(ctx, ref)
    print(f"case: store batch={batch} n={n} first={first}", flush=True)
    fd = None if first is None else ints(ctx, first)
    ctx.kv4_store(c, 1, 1, batch, fd, n, ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16)), cap)
    ref.store(1, 1, batch, first, n, k, v)
    assert_same(ctx, c, ref)
    kb, vb = (ctx.upload(np.full(k.shape, 0x1234, np.uint16)) for _ in range(2))
    ctx.kv4_load(c, 1, 1, batch, fd, n, kb, vb, cap)
    for buf, x in ((kb, k), (vb, v)):
        got = ctx.download(buf, x.shape, np.float16)
        want = R.value(*R.quantise(x)).astype(np.float32).astype(np.float16)
        want[:, :, n:] = np.array(0x1234, np.uint16).view(np.float16)
        assert np.array_equal(got, want)


def test_store_leaves_out_what_has_no_place(ctx):
    """Tokens past a row's length, a negative first, entries that are no page: nothing written; their f16 rows stay."""
    ref = R.Cache(1, 12, 4, 3, seed=5)
    assert ref.resize([0, 1, 2, 3], [70, 100, 128, 64]) == 0
    ref.table[2, 1], ref.table[3, 0] = 12, -5
    k, v = kv_rows(np.random.default_rng(6), 4, 4, 90)
    first = [20, -1, 50, 0]
    c = upload(ctx, ref)
    print("case: store, tokens without a place", flush=True)
    kd, vd = ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16))
    ctx.kv4_store(c, 0, 0, 4, ints(ctx, first), 90, kd, vd, 90)
    ref.store(0, 0, 4, first, 90, k, v)
    assert_same(ctx, c, ref)
    kb, vb = (ctx.upload(np.full(k.shape, 0x1234, np.uint16)) for _ in range(2))
    ctx.kv4_load(c, 0, 0, 4, ints(ctx, first), 90, kb, vb, 90)
    got = ctx.download(vb, v.shape, np.uint16)
    want = R.value(*R.quantise(v)).astype(np.float32).astype(np.float16).view(np.uint16)
    there = np.zeros((4, 90), bool)
    there[0, :50], there[2, :14] = True, True
    assert np.array_equal(got, np.where(there[:, None, :, None], want, np.uint16(0x1234)))


def test_store_of_tokens_at_the_ends_of_int32(ctx):
    """Positions near the ends of int32 (past every length, or negative) leave the pool as it was."""
    ref = R.Cache(1, 6, 6, 1, seed=9)
    assert ref.resize([0, 1, 2, 3, 4], [64] * 5) == 0
    c = upload(ctx, ref)
    k, v = kv_rows(np.random.default_rng(10), 6, 4, 70)
    kd, vd = ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16))
    first = [2 ** 31 - 1, 2 ** 31 - 33, -2 ** 31, -1, 64, 0]
    print("case: store, positions at the ends of int32", flush=True)
    ctx.kv4_store(c, 0, 0, 6, ints(ctx, first), 70, kd, vd, 70)
    assert_same(ctx, c, ref)
    ctx.kv4_load(c, 0, 0, 6, ints(ctx, first), 70, kd, vd, 70)
    assert np.array_equal(ctx.download(kd, k.shape, np.uint16), k.view(np.uint16))


def test_store_values_at_the_edges_of_f16(ctx):
    """Equal values, the widest range, subnormals, signed zeros, infinities and NaN, group by group."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((1, 4, 16, 256)).astype(np.float16)
    x[0, 0, 0, :64] = 3.5
    x[0, 0, 1, 64:128] = np.tile([-65504, 65504], 32)
    x[0, 0, 2] = (rng.integers(-9, 10, 256) * 2.0 ** -24).astype(np.float16)
    x[0, 0, 3, 5], x[0, 0, 4, 70], x[0, 0, 5, 255] = np.inf, -np.inf, np.nan
    x[0, 0, 6] = np.where(rng.random(256) < 0.5, 0.0, -0.0)
    x[0, 0, 7, ::2], x[0, 0, 7, 1::2] = 1000.0, 2.0 ** -20
    x[0, 1] = (rng.standard_normal((16, 256)) * 2.0 ** rng.integers(-24, 15, (16, 1))).clip(-65504, 65504).astype(np.float16)
    ref = R.Cache(1, 2, 1, 1, seed=8)
    assert ref.resize([0], [16]) == 0
    c = upload(ctx, ref)
    print("case: store, edges of f16", flush=True)
    d = ctx.upload(x.view(np.uint16))
    ctx.kv4_store(c, 0, 0, 1, None, 16, d, d, 16)
    kb, vb = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    ctx.kv4_load(c, 0, 0, 1, None, 16, kb, vb, 16)
    with np.errstate(over="ignore"):
        want = R.value(*R.quantise(x)).astype(np.float32).astype(np.float16)
    for buf in (kb, vb):
        got = ctx.download(buf, x.shape, np.float16)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        assert np.array_equal(got[fine], want[fine])


# ---- pages ----------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(6))
def test_pages_through_many_calls(ctx, seed):
    """Growing, freeing, forking and compacting in turn: table, lengths, counts, contents and results equal."""
    ref = R.Cache(2, 24, 7, 5, seed=seed)
    c = upload(ctx, ref)
    for step, (kind, args) in enumerate(some_steps(seed)):
        print(f"case: pages seed={seed} step={step} {kind}", flush=True)
        want = getattr(ref, kind)(*args)
        got = {"resize": run_resize, "fork": run_fork, "compact": run_compact}[kind](ctx, c, *args)
        assert got == want
        assert_same(ctx, c, ref, pages=step % 6 == 5)
    assert_same(ctx, c, ref)


def test_a_page_that_all_its_holders_write_keeps_one(ctx):
    """Three rows share a partly filled page: when two grow both copy it; when the last two grow together the first keeps it."""
    ref = R.Cache(3, 16, 5, 3, seed=1)
    c = upload(ctx, ref)
    for call, args in [(run_resize, ([0], [100])), (run_fork, ([0, 0], [3, 4])), (run_resize, ([4, 3], [101, 130])),
                       (run_fork, ([0], [1])), (run_resize, ([1, 0], [101, 101])), (run_resize, (None, [0, 0, 0, 0, 0]))]:
        print(f"case: shared page, {call.__name__} {args}", flush=True)
        want = getattr(ref, call.__name__[4:])(*args)
        assert call(ctx, c, *args) == want == 0
        assert_same(ctx, c, ref)
    assert not ref.refs.any()


def test_refused_calls_change_nothing(ctx):
    ref = R.Cache(1, 8, 4, 4, seed=2)
    assert ref.resize([0, 1], [130, 64]) == 0
    c = upload(ctx, ref)
    for call, args, want in [
            (run_resize, ([2, 3], [256, 256]), 4), (run_resize, ([0, 2], [131, 257]), -1), (run_resize, ([0, 0], [1, 2]), -1),
            (run_resize, ([4], [1]), -1), (run_resize, ([-1], [1]), -1), (run_resize, ([1], [-1]), -1),
            (run_resize, ([0, 1], [1, -65], True), -1), (run_resize, ([0], [2 ** 31 - 1], True), -1),
            (run_fork, ([0, 1], [2, 2]), -1), (run_fork, ([4], [2]), -1), (run_fork, ([0], [-1]), -1)]:
        print(f"case: refused {call.__name__} {args}", flush=True)
        assert call(ctx, c, *args) == want
        assert_same(ctx, c, ref)
    # a partly filled last page that is no page, and one that nobody is said to hold
    for entry, count in ((99, 1), (2, 0)):
        ref.table[0, 2], ref.refs[2] = entry, count
        ctx.upload(ref.table, c.table)
        ctx.upload(ref.refs, c.refs)
        assert run_resize(ctx, c, [0], [140]) == -1
        assert_same(ctx, c, ref)


def test_full_lists(ctx):
    """1024 rows in one call, each with its own new length, then all forked in reverse and freed."""
    rng = np.random.default_rng(3)
    ref = R.Cache(1, 5000, 1100, 4, fill=False)
    c = upload(ctx, ref)
    pick = rng.permutation(1100)[:1024].astype(np.int32)
    lens = rng.integers(0, 257, 1024).astype(np.int32)
    print("case: 1024 rows", flush=True)
    assert run_resize(ctx, c, pick, lens) == ref.resize(pick, lens) == 0
    assert_same(ctx, c, ref, pages=False)
    assert run_fork(ctx, c, pick[::-1].copy(), pick) == ref.fork(pick[::-1], pick) == 0
    assert_same(ctx, c, ref, pages=False)
    some = pick[::2].copy()
    want = ref.resize(some, np.ones(512, np.int32), True)
    assert run_resize(ctx, c, some, np.ones(512, np.int32), True) == want
    assert_same(ctx, c, ref, pages=False)
    assert run_resize(ctx, c, pick, np.zeros(1024, np.int32)) == ref.resize(pick, np.zeros(1024, np.int32)) == 0
    assert_same(ctx, c, ref, pages=False)


class Thin(R.Cache):
    """A cache without contents, for pools too large to compare."""

    def __init__(self, num_pages, rows, max_pages):
        super().__init__(1, 1, rows, max_pages, fill=False)
        self.refs = np.zeros(num_pages, np.int32)
        self.pages = np.zeros((1, num_pages, 1), np.uint8)


def test_large_pool(ctx):
    """70,001 pages: more than the planning workgroup holds at a time.  Free pages are found past the first 65,536, and
    pages move from there."""
    n = 70001
    ref = Thin(n, 6, 14000)
    c = M.Kv4Cache(ctx, 1, n, 6, 14000)
    ctx.upload(ref.table, c.table)
    steps = [(run_resize, (None, [13000 * 64] * 5)), (run_resize, ([5], [4900 * 64 + 5])), (run_resize, ([5, 0], [5002 * 64, 0])),
             (run_resize, ([0], [640])), (run_fork, ([5], [0])), (run_compact, ()), (run_resize, ([1, 0], [0, 64 * 13999 + 1])),
             (run_resize, ([2], [13002 * 64]))]
    for call, args in steps:
        print(f"case: large pool {call.__name__}", flush=True)
        want = getattr(ref, call.__name__[4:])(*args)
        assert call(ctx, c, *args) == want
        assert_same(ctx, c, ref, pages=False)
    for buf in (c.pages, c.table, c.lens, c.refs):
        buf.close()


# ---- attention ------------------------------------------------------------------------------
class Step:
    """A cache whose rows are full of stored tokens (and of garbage past them), and inputs of a step."""

    def __init__(self, ctx, lens, seed, layers=1, spare=3, rows=None, max_pages=None, share=0):
        rng = np.random.default_rng(seed)
        pages = [R.pages_of(n) for n in lens]
        rows, max_pages = rows or len(lens), max_pages or max(1, max(pages))
        common = [0] + [max(0, min(share, n - 1, pages[0] - 1)) for n in pages[1:]]     # first pages, those of row 0
        count = sum(pages) - sum(common) + spare
        self.ref = ref = R.Cache(layers, count, rows, max_pages, fill=False)
        # pages written in earnest, a few dozen and their copies, and garbage in the scales past each row's end
        some = np.zeros((min(count, 12), R.PAGE), np.uint8)
        for page in some:
            for head in range(4):
                k, v = kv_rows(rng, 64)
                for is_v, x in ((0, k), (1, v)):
                    _put_all(page, head, x, is_v)
        ids = rng.permutation(count).astype(np.int32)
        at = 0
        for r, n in enumerate(pages):
            own = n - common[r]
            ref.table[r, :common[r]] = ref.table[0, :common[r]]
            ref.table[r, common[r]:n] = ids[at:at + own]
            at += own
            ref.lens[r] = lens[r]
        for r in range(len(lens)):
            np.add.at(ref.refs, ref.ids(r), 1)
        ref.pages[:] = some[rng.integers(0, len(some), (layers, count))]
        for layer in range(layers):
            for r, n in enumerate(lens):
                if n % 64:
                    _spoil(ref.pages[layer, ref.table[r, pages[r] - 1]], n % 64)
        self.c = upload(ctx, ref)
        b = len(lens)
        self.q_gate = rng.standard_normal((b, 16, 512), dtype=np.float32)
        self.k_new = rng.standard_normal((b, 4, 256), dtype=np.float32)
        self.v_new = (0.7 * rng.standard_normal((b, 4, 256))).astype(np.float32)
        self.q_norm, self.k_norm = ((0.1 * rng.standard_normal(256)).astype(np.float16) for _ in range(2))

    def inputs(self, ctx):
        return [ctx.upload(x) for x in (self.q_gate, self.k_new, self.v_new, self.q_norm, self.k_norm)]

    def run(self, ctx, max_len, slots=None, layer=0, gate=None, batch=None, rope_rows=None):
        batch = batch or len(self.q_gate)
        cos, sin = M.rope_table(rope_rows or max_len)
        out = ctx.upload(np.full((batch, 16, 256), 7.0, np.float32))
        ctx.gqa_decode_kv4(self.c, layer, batch, None if slots is None else ints(ctx, slots), *self.inputs(ctx), ctx.upload(cos),
                           ctx.upload(sin), rope_rows or max_len, max_len, gate, out)
        got = ctx.download(out, (batch, 16, 256), np.float32)
        want = self.ref.decode(layer, slots, batch, self.q_gate, self.k_new, self.v_new, self.q_norm, self.k_norm, cos, sin, max_len)
        return got, want

    def check(self, got, want):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        g, w = got[fine].astype(np.float64), want[fine]
        err, norm = np.linalg.norm(g - w), np.linalg.norm(w)
        n = int(max(self.ref.lens))
        most = 2.0 ** -24 * 6 * (272 ** 0.5 * 2 * 200 + n ** 0.5) * 6
        print(f"rel={err / max(norm, 1e-30):.2e} max={np.abs(g - w).max() if g.size else 0:.2e} (bar {most:.1e})", flush=True)
        assert err <= 2e-5 * norm and (not g.size or np.abs(g - w).max() <= most)


def _put_all(page, head, x, is_v):
    """R.put of all 64 tokens at once."""
    q, s, lo = R.quantise(x)
    for half in range(2):
        h = R._half(page, head, half * 32)
        words = np.zeros(8192, np.uint8)
        part = q[half * 32:half * 32 + 32]
        for shift in (0, 4):
            m = R.CODE_SHIFT[is_v] == shift
            words[R.CODE_BYTE[is_v][m]] |= part[m] << shift
        lo8, hi8 = (0, 4096) if not is_v else (4096, 8192)
        h[lo8:hi8] = words[lo8:hi8]
        meta = h[8192:].view(np.float16)
        meta[256 * is_v + R.S_AT], meta[256 * is_v + 128 + R.LO_AT] = s[half * 32:half * 32 + 32], lo[half * 32:half * 32 + 32]


def _spoil(page, n):
    """NaN and infinities in the scales and minima of tokens n .. 63 of a page."""
    for head in range(4):
        for t in range(n, 64):
            meta = R._half(page, head, t)[8192:].view(np.float16)
            for is_v in (0, 1):
                meta[256 * is_v + R.S_AT[t % 32]] = np.inf if t % 2 else np.nan
                meta[256 * is_v + 128 + R.LO_AT[t % 32]] = np.nan if t % 3 else -np.inf


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 500, 1000])
def test_decode_lengths(ctx, n):
    """One sequence of n tokens, the last of them new: its output, and its page byte by byte."""
    s = Step(ctx, [n], seed=n)
    print(f"case: kv4 decode n={n}", flush=True)
    got, want = s.run(ctx, n)
    s.check(got, want)
    assert_same(ctx, s.c, s.ref)


@pytest.mark.parametrize("lens, share, max_len", [
    ([5000, 70, 4351, 640], 0, 5000), ([300, 64, 1, 0, 999, 128, 127, 129, 32, 33], 0, 1100), ([2000] * 9, 30, 2001),
    ([4097], 0, 4097), ([9001, 5], 0, 9001)])
def test_decode_batches(ctx, lens, share, max_len):
    """Ragged batches, empty rows, common prompts; layers beside the one stepped stay as they were."""
    s = Step(ctx, lens, seed=len(lens) + lens[0], layers=2, share=share, max_pages=R.pages_of(max_len))
    print(f"case: kv4 decode lens={lens} share={share}", flush=True)
    got, want = s.run(ctx, max_len, layer=1, rope_rows=max_len + 3)
    s.check(got, want)
    assert all((got[b] == 0).all() for b, n in enumerate(lens) if n == 0)
    assert_same(ctx, s.c, s.ref)


def test_decode_slots(ctx):
    """Slots in any order, padded rows, a slot twice (the later is refused), a row longer than max_len (refused)."""
    s = Step(ctx, [90, 0, 400, 33, 260, 64, 1, 12, 70, 5], seed=77)
    slots = [4, -1, 0, 4, 2, 10, 3, 0, 1, 8]
    print(f"case: kv4 decode slots={slots}", flush=True)
    got, want = s.run(ctx, 300, slots=slots)
    s.check(got, want)
    for b in (3, 4, 7):
        assert np.isnan(got[b]).all()
    for b in (1, 5, 8):
        assert (got[b] == 0).all()
    assert_same(ctx, s.c, s.ref)


def test_decode_more_rows_than_a_wave_looks_at(ctx):
    """130 batch rows over 66 table rows: a slot that comes again 64 and more rows later is refused there."""
    s = Step(ctx, [3 + i % 40 for i in range(66)], seed=78)
    rng = np.random.default_rng(0)
    s.q_gate, s.k_new, s.v_new = (np.concatenate([x, x[::-1]])[:130] for x in (s.q_gate, s.k_new, s.v_new))
    slots = list(rng.permutation(66)) + [0, 65, 7] + [-1] * 61
    print("case: kv4 decode 130 rows", flush=True)
    got, want = s.run(ctx, 64, slots=slots)
    s.check(got, want)
    assert all(np.isnan(got[b]).all() for b in (66, 67, 68))
    assert_same(ctx, s.c, s.ref)


def test_decode_slots_of_long_rows(ctx):
    """The same where the tokens are dealt to workgroups and joined: slots in any order, padded rows, repeats, rows longer
    than max_len, empty ones."""
    s = Step(ctx, [900, 0, 1400, 333, 2600, 64, 1, 1201, 700, 5], seed=83)
    slots = [4, -1, 0, 4, 2, 10, 3, 0, 1, 8]
    print(f"case: kv4 decode slots={slots} of long rows", flush=True)
    got, want = s.run(ctx, 1400, slots=slots)
    s.check(got, want)
    assert np.isnan(got[[0, 3, 7]]).all() and (got[[1, 5, 8]] == 0).all()
    assert_same(ctx, s.c, s.ref)


def test_decode_dealt_to_more_rows_than_a_wave(ctx):
    """150 batch rows, lengths up to 900, the tokens dealt in blocks of 64 rows; with slots, repeats in later blocks."""
    rng = np.random.default_rng(84)
    lens = rng.integers(0, 900, 150)
    lens[[0, 63, 64, 149]], lens[[1, 127, 128]] = 900, 0
    for slots in (None, list(rng.permutation(150)[:140]) + [-1, 150] + [0] * 8):
        s = Step(ctx, lens.tolist(), seed=85, max_pages=15)
        print(f"case: kv4 decode of 150 rows, slots={slots is not None}", flush=True)
        got, want = s.run(ctx, 900, slots=slots)
        s.check(got, want)
        assert_same(ctx, s.c, s.ref)


def test_decode_long_splits(ctx):
    """Enough tokens that a split has its most, 4096: 64 rows of up to 9300 tokens, some checked."""
    lens = [5000 + 70 * i for i in range(62)] + [4097, 3]
    s = Step(ctx, lens, seed=86)
    print("case: kv4 decode, the longest splits", flush=True)
    cos, sin = M.rope_table(max(lens))
    out = ctx.alloc(64 * 4096 * 4)
    ctx.gqa_decode_kv4(s.c, 0, 64, None, *s.inputs(ctx), ctx.upload(cos), ctx.upload(sin), max(lens), max(lens), None, out)
    got = ctx.download(out, (64, 16, 256), np.float32)
    some = [0, 31, 61, 62, 63]
    only = [i if i in some else -1 for i in range(64)]
    want = s.ref.decode(0, only, 64, s.q_gate, s.k_new, s.v_new, s.q_norm, s.k_norm, cos, sin, max(lens))
    s.check(got[some], want[some])


@pytest.mark.parametrize("lens", [
    [40000 - 7 * i for i in range(24)], [16000] * 60 + [3] * 9 + [1] + [12345] * 5, [200001] * 3, [70000] * 511 + [1]])
def test_decode_of_more_tokens_than_one_round_of_splits(ctx, lens):
    """So many tokens that the chip's workgroups take several rounds of splits (the last: more rounds than are dealt evenly),
    by a common prompt; some rows checked."""
    s = Step(ctx, lens, seed=87, share=10 ** 6)
    b, most = len(lens), max(lens)
    print(f"case: kv4 decode of {sum(lens)} tokens", flush=True)
    cos, sin = M.rope_table(most)
    out = ctx.upload(np.full((b, 16, 256), 7.0, np.float32))
    ctx.gqa_decode_kv4(s.c, 0, b, None, *s.inputs(ctx), ctx.upload(cos), ctx.upload(sin), most, most, None, out)
    got = ctx.download(out, (b, 16, 256), np.float32)
    some = sorted({0, b // 2, b - 2, b - 1})
    only = [i if i in some else -1 for i in range(b)]
    want = s.ref.decode(0, only, b, s.q_gate, s.k_new, s.v_new, s.q_norm, s.k_norm, cos, sin, most)
    s.check(got[some], want[some])
    assert np.isfinite(got).all() and (np.abs(got).max((1, 2)) > 0).all()


@pytest.mark.parametrize("n", [70, 1500])
def test_decode_of_rows_forked_after_they_grew(ctx, n):
    """Their last page is not one row's: neither writes there, both outputs are NaN; once they have grown again, both step."""
    s = Step(ctx, [n, 5, 20], seed=87, spare=6, max_pages=R.pages_of(n + 1))
    assert run_fork(ctx, s.c, [0], [2]) == s.ref.fork([0], [2]) == 0
    print(f"case: kv4 decode of forked rows, n={n}", flush=True)
    got, want = s.run(ctx, n)
    s.check(got, want)
    assert np.isnan(got[[0, 2]]).all() and np.isfinite(got[1]).all()
    assert_same(ctx, s.c, s.ref)
    assert run_resize(ctx, s.c, None, [1, 0, 1], True) == s.ref.resize(None, [1, 0, 1], True) == 0
    got, want = s.run(ctx, n + 1)
    s.check(got, want)
    assert np.isfinite(got).all()
    assert_same(ctx, s.c, s.ref)


def test_store_leaves_shared_pages_alone(ctx):
    ref = R.Cache(1, 9, 3, 3, seed=11)
    c = upload(ctx, ref)
    assert run_resize(ctx, c, [0], [150]) == ref.resize([0], [150]) == 0
    assert run_fork(ctx, c, [0], [1]) == ref.fork([0], [1]) == 0
    assert run_resize(ctx, c, [1], [160]) == ref.resize([1], [160]) == 0      # its third page is its own now
    k, v = kv_rows(np.random.default_rng(12), 1, 4, 160)
    print("case: store over shared pages", flush=True)
    ctx.kv4_store(c, 0, 1, 1, None, 160, ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16)), 160)
    ref.store(0, 1, 1, None, 160, k, v)
    assert_same(ctx, c, ref)


def test_decode_entries_that_are_no_page(ctx):
    """Pages outside the pool are skipped, also where the new token would go, and a row of none is zero."""
    for lens in ([300, 200, 130, 64], [1300, 200, 130, 64]):
        _no_page(ctx, lens)


def _no_page(ctx, lens):
    s = Step(ctx, lens, seed=79)
    s.ref.table[0, 1], s.ref.table[1, 3], s.ref.table[2], s.ref.table[3, 0] = 10 ** 6, -1, -1, 2 ** 31 - 1
    ctx.upload(s.ref.table, s.c.table)
    print("case: kv4 decode, entries that are no page", flush=True)
    got, want = s.run(ctx, max(lens))
    s.check(got, want)
    assert (got[2:] == 0).all()
    assert_same(ctx, s.c, s.ref)


def test_decode_nan_in_a_group_reaches_its_heads_only(ctx):
    """An infinity in the new k (kv head 1) and a NaN in the new v (head 2, dims 64 ..): NaN outputs there, none elsewhere."""
    s = Step(ctx, [40, 1], seed=80)
    s.k_new[0, 1, 200] = np.inf
    s.v_new[0, 2, 70] = np.nan
    s.v_new[1, 3, 0] = 1e6                        # beyond f16: an infinity there
    print("case: kv4 decode, NaN in groups", flush=True)
    got, _ = s.run(ctx, 40)
    bad = np.isnan(got)
    want = np.zeros_like(bad)
    want[0, 4:8], want[0, 8:12, 64:128], want[1, 12:, :64] = True, True, True
    assert np.array_equal(bad, want)


def test_decode_after_a_refused_resize_does_nothing(ctx):
    for lens in ([100, 64], [100, 1000]):
        _after_refused(ctx, lens)


def _after_refused(ctx, lens):
    s = Step(ctx, lens, seed=81)
    for gate, runs in ((ints(ctx, [3]), False), (ints(ctx, [-1]), False), (ints(ctx, [0]), True)):
        print(f"case: kv4 decode gated, runs={runs}", flush=True)
        before = R.Cache.__new__(R.Cache)
        before.__dict__ = {k: v.copy() for k, v in s.ref.__dict__.items()}
        got, want = s.run(ctx, max(lens), gate=gate)
        if runs:
            s.check(got, want)
            assert_same(ctx, s.c, s.ref)
        else:
            assert (got == 0).all()
            s.ref = before
            assert_same(ctx, s.c, s.ref)


@pytest.mark.parametrize("scale", [1e-4, 1e4])
def test_decode_values_of_other_sizes(ctx, scale):
    """V far from 1 and scores far apart: weights are not tied to a range.  The bars are relative to the values."""
    s = Step(ctx, [200], seed=82)
    for half in s.ref.pages.reshape(-1, R.HALF_BYTES):
        meta = half[8192:].view(np.float16)
        fine = np.isfinite(meta[256:])
        meta[256:][fine] = (meta[256:][fine].astype(np.float32) * scale).astype(np.float16)
    s.v_new *= scale
    ctx.upload(s.ref.pages, s.c.pages)
    print(f"case: kv4 decode V x {scale}", flush=True)
    got, want = s.run(ctx, 200)
    s.check(got / scale, want / scale)


def test_decode_steps_in_a_graph(ctx):
    """Grow by one token and step, captured once and replayed, against the same calls made eagerly on a twin cache, with
    eager work between the replays: every replay gives the eager outputs and pages bit for bit."""
    a, b = (Step(ctx, [62, 127, 0, 300], seed=90, spare=12, max_pages=6) for _ in range(2))
    for s in (a, b):
        s.ref.fork([1], [2])
        ctx.upload(s.ref.lens, s.c.lens), ctx.upload(s.ref.refs, s.c.refs), ctx.upload(s.ref.table, s.c.table)
    max_len = 6 * 64
    cos, sin = M.rope_table(max_len)
    rc, rs, one = ctx.upload(cos), ctx.upload(sin), ints(ctx, [1, 1, 1, 1])
    ctx.reserve(4, max_len)
    ia, ib = a.inputs(ctx), b.inputs(ctx)
    ra, rb = ints(ctx, [-7]), ints(ctx, [-7])
    oa, ob = (ctx.alloc(4 * 16 * 256 * 4) for _ in range(2))

    def step(s, inputs, res, out):
        ctx.kv4_resize(s.c, 4, None, one, res, M.QM_KV4_ADD)
        ctx.gqa_decode_kv4(s.c, 0, 4, None, *inputs, rc, rs, max_len, max_len, res, out)

    ctx.sync()
    ctx.graph_begin()
    step(a, ia, ra, oa)
    g = ctx.graph_end()
    rng = np.random.default_rng(91)
    for rep in range(8):
        x = rng.standard_normal(b.q_gate.shape, dtype=np.float32)
        ctx.upload(x, ia[0]), ctx.upload(x, ib[0])
        print(f"case: kv4 graph replay {rep}", flush=True)
        step(b, ib, rb, ob)
        ctx.sync()
        g.launch()
        ctx.sync()
        assert result(ctx, ra) == result(ctx, rb) == 0
        assert np.array_equal(ctx.download(oa, (4, 4096), np.float32), ctx.download(ob, (4, 4096), np.float32)), rep
        for name in ("table", "lens", "refs"):
            x, y = getattr(a.c, name), getattr(b.c, name)
            assert np.array_equal(ctx.download(x, (x.nbytes // 4,), np.int32), ctx.download(y, (y.nbytes // 4,), np.int32))
        assert np.array_equal(ctx.download(a.c.pages, a.ref.pages.shape, np.uint8), ctx.download(b.c.pages, b.ref.pages.shape, np.uint8))
    # until a row is full (300 + 84 tokens): the resize is refused, the step writes nothing
    for _ in range(76):
        g.launch()
    assert result(ctx, ra) == 0
    before = ctx.download(a.c.pages, a.ref.pages.shape, np.uint8)
    g.launch()
    assert result(ctx, ra) == -1
    assert (ctx.download(oa, (4, 4096), np.float32) == 0).all()
    assert np.array_equal(ctx.download(a.c.pages, a.ref.pages.shape, np.uint8), before)
    g.close()


def test_a_workspace_that_would_grow_under_capture_is_refused():
    with M.Context(0) as c:
        s = Step(c, [700, 300], seed=92)
        inputs = s.inputs(c)
        cos, sin = M.rope_table(700)
        rc, rs, out = c.upload(cos), c.upload(sin), c.alloc(2 * 4096 * 4)
        res = ints(c, [0])
        c.graph_begin()
        for call in (lambda: c.gqa_decode_kv4(s.c, 0, 2, None, *inputs, rc, rs, 700, 700, None, out),
                     lambda: c.kv4_resize(s.c, 2, None, res, res), lambda: c.kv4_compact(s.c, res),
                     lambda: c.kv4_fork(s.c, 1, res, res, res)):
            with pytest.raises(M.MixerError) as e:
                call()
            assert e.value.code == 9
        c.graph_end().close()
        c.reserve(2, 700)
        got, want = s.run(c, 700)
        s.check(got, want)


def test_a_conversation(ctx):
    """As they are used together: a prompt's prefill, its cache into pages, two answers forked from it, steps that copy the
    shared page and take new ones, one answer dropped, the pool compacted, more steps -- against the numpy form fed with the
    prefill's own f16 rows."""
    rng = np.random.default_rng(100)
    S, cap, max_len = 100, 128, 256
    W = __import__("conftest").load_workloads()
    p = W.gqa_prefill_workload(S, seed=101)
    cos, sin = M.rope_table(max_len)
    rc, rs = ctx.upload(cos), ctx.upload(sin)
    kf, vf = (ctx.upload(np.zeros((4, cap, 256), np.uint16)) for _ in range(2))
    out = ctx.alloc(S * 4096 * 2)
    ctx.gqa_prefill(S, *(ctx.upload(p[k]) for k in ("q_gate", "k", "v", "q_norm", "k_norm")), rc, rs, max_len, kf, vf, cap, out)
    k16, v16 = (ctx.download(x, (1, 4, cap, 256), np.float16) for x in (kf, vf))
    ref = R.Cache(2, 14, 4, 4, seed=102)
    c = upload(ctx, ref)
    s = Step.__new__(Step)
    s.ref, s.c = ref, c
    s.q_norm, s.k_norm = p["q_norm"].view(np.float16), p["k_norm"].view(np.float16)

    def both(call, *args):
        want = getattr(ref, call.__name__[4:])(*args)
        assert call(ctx, c, *args) == want
        return want

    def steps(rows, count):
        for i in range(count):
            assert both(run_resize, rows, [1] * len(rows), True) == 0
            for layer in (0, 1):
                b = len(rows)
                s.q_gate = rng.standard_normal((b, 16, 512), dtype=np.float32)
                s.k_new, s.v_new = (rng.standard_normal((b, 4, 256), dtype=np.float32) for _ in range(2))
                print(f"case: conversation rows={rows} step={i} layer={layer}", flush=True)
                s.check(*s.run(ctx, max_len, slots=rows, layer=layer))

    assert both(run_resize, [1], [S]) == 0
    for layer in (0, 1):
        ctx.kv4_store(c, layer, 1, 1, None, S, kf, vf, cap)
        ref.store(layer, 1, 1, None, S, k16, v16)
    assert_same(ctx, c, ref)
    assert both(run_fork, [1, 1], [3, 0]) == 0
    steps([3, 1, 0], 3)
    assert both(run_resize, [1], [0]) == 0
    both(run_compact)
    assert_same(ctx, c, ref)
    steps([0, 3], 30)
    assert both(run_resize, [0, 3, 1, 2], [0, 0, 0, 0]) == 0
    assert not ref.refs.any()
    assert_same(ctx, c, ref)


def test_calls_on_a_stream_of_the_callers(ctx):
    """The calls run on the stream they are given, in its order."""
    import ctypes as C
    s = Step(ctx, [150, 20], seed=103)
    h = C.c_void_p(0)
    ctx._check(ctx.lib.qm_stream_create(ctx.h, C.byref(h)))
    ctx.sync()
    before, ctx.stream = ctx.stream, h.value
    try:
        print("case: kv4 on another stream", flush=True)
        got, want = s.run(ctx, 150)
        s.check(got, want)
        assert run_fork(ctx, s.c, [0], [1]) == s.ref.fork([0], [1]) == 0
        assert run_resize(ctx, s.c, [1], [151]) == s.ref.resize([1], [151]) == 0
        run_compact(ctx, s.c), s.ref.compact()
        assert_same(ctx, s.c, s.ref)
    finally:
        ctx.sync()
        ctx.stream = before
        ctx._check(ctx.lib.qm_stream_destroy(ctx.h, h))


@pytest.mark.parametrize("n, late", [(900, False), (900, True), (1500, False), (5000, False), (5000, True)])
def test_decode_nan_in_a_split_of_no_weight(ctx, n, late):
    """A NaN group of V in a split whose scores are 300 below the others': its weight is 0, and 0 times NaN is NaN, in every
    dealing of the tokens (8, 12 and 40 splits of 128 tokens).  Scores are relative to the query's own direction: k = -300 x
    / |x| with |q| = 16 and q . k / 16."""
    s = Step(ctx, [n], seed=110 + n)
    x = np.zeros(256)
    x[64:] = np.random.default_rng(n).standard_normal(192)         # past the rotary dims
    s.q_gate[0, 8:12, :256] = x
    s.q_norm[:] = 0
    rows = np.tile((-300 * x / np.linalg.norm(x)).astype(np.float16), (64, 1))
    page0 = (n - 1) // 128 * 2 - 2 if late else 0                  # the last split but one, or the first
    for j in (page0, page0 + 1):
        _put_all(s.ref.pages[0, s.ref.table[0, j]], 2, rows, 0)
    meta = R._half(s.ref.pages[0, s.ref.table[0, page0 + 1]], 2, 40)[8192:].view(np.float16)
    meta[256 + R.S_AT[8, 1]] = meta[256 + 128 + R.LO_AT[8, 1]] = np.nan
    ctx.upload(s.ref.pages, s.c.pages)
    print(f"case: kv4 decode n={n}, NaN in a split of no weight, late={late}", flush=True)
    got, want = s.run(ctx, n)
    bad = np.zeros_like(want, bool)
    bad[0, 8:12, 64:128] = True
    assert np.array_equal(np.isnan(want), bad)
    s.check(got, want)


@pytest.mark.parametrize("count", [0, -1])
def test_pages_that_no_row_holds_are_not_written(ctx, count):
    """Where the counts say that nobody holds a row's page (the next resize may hand it to another row), a store leaves its
    tokens out, and a step over it writes nothing and gives NaN; the other rows are as ever."""
    ref = R.Cache(1, 9, 3, 3, seed=13)
    assert ref.resize([0, 1], [150, 70]) == 0
    ref.refs[ref.table[0, 1]] = count
    c = upload(ctx, ref)
    k, v = kv_rows(np.random.default_rng(14), 2, 4, 150)
    print(f"case: store to a page of count {count}", flush=True)
    ctx.kv4_store(c, 0, 0, 2, None, 150, ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16)), 150)
    before = ref.pages[0, ref.table[0, 1]].copy()
    ref.store(0, 0, 2, None, 150, k, v)
    ref.pages[0, ref.table[0, 1]] = before
    assert_same(ctx, c, ref)
    for n in (70, 1500):
        s = Step(ctx, [n, 5], seed=88, max_pages=R.pages_of(n))
        page = s.ref.table[0, (n - 1) // 64]
        s.ref.refs[page] = count
        ctx.upload(s.ref.refs, s.c.refs)
        before = s.ref.pages[:, page].copy()
        print(f"case: kv4 decode into a page of count {count}, n={n}", flush=True)
        got, want = s.run(ctx, n)
        want[0] = np.nan
        s.ref.pages[:, page] = before
        s.check(got, want)
        assert_same(ctx, s.c, s.ref)


def test_forks_and_compactions_in_a_graph_after_a_reserve():
    """All of the cache's calls captured on a new context that was reserved for exactly its table, replayed with eager work
    between: table, lengths, counts and contents are the numpy form's after every replay."""
    with M.Context(0) as c:
        ref = R.Cache(2, 40, 8, 5, fill=False)
        assert ref.resize(None, [300, 64, 130, 5, 1, 0, 0, 0]) == 0
        d = upload(c, ref)
        src, dst, sent = [0, 2, 2], [5, 6, 2], [257, 40, 0]
        rows, lens, first, res = ints(c, [2, 5, 0]), ints(c, sent), ints(c, [3, 1]), ints(c, [-7, -7, -7])
        srcs, dsts = ints(c, src), ints(c, dst)
        k, v = kv_rows(np.random.default_rng(16), 2, 4, 70)
        kd, vd, kb, vb = (c.upload(x.view(np.uint16)) for x in (k, v, k, v))
        c.reserve(8, 5 * 64)
        c.sync()
        c.graph_begin()
        c.kv4_fork(d, 3, srcs, dsts, res)
        c.kv4_resize(d, 3, rows, lens, res.ptr + 4)
        c.kv4_store(d, 1, 2, 2, first, 70, kd, vd, 70)
        c.kv4_compact(d, res.ptr + 8)
        c.kv4_load(d, 1, 2, 2, first, 70, kb, vb, 70)
        g = c.graph_end()
        for rep in range(4):
            sent = [257 - 50 * rep, 40 + 64 * rep, 0 if rep != 2 else 320]
            c.upload(np.asarray(sent, np.int32), lens)
            c.sync()
            print(f"case: kv4 calls in a graph, replay {rep}", flush=True)
            g.launch()
            c.sync()
            want = [ref.fork(src, dst), ref.resize([2, 5, 0], sent)]
            ref.store(1, 2, 2, [3, 1], 70, k, v)
            want.append(ref.compact())
            assert c.download(res, (3,), np.int32).tolist() == want and want[:2] == [0, 0]
            assert_same(c, d, ref)
            back = c.download(vb, v.shape, np.float16)
            for b, (row, first_of, n) in enumerate([(2, 3, min(70, sent[0] - 3)), (3, 1, 4)]):
                for head in range(4):
                    held = ref.rows64(1, row, head, 1)[0][first_of:first_of + n].astype(np.float32).astype(np.float16)
                    assert np.array_equal(back[b, head, :n], held, equal_nan=True)
            assert run_fork(c, d, [1], [7]) == ref.fork([1], [7]) == 0           # between the replays
            assert run_resize(c, d, [7], [0]) == ref.resize([7], [0]) == 0
        g.close()


def test_load_rounds_the_sum_to_f32_first(ctx):
    """Minima far below the scale, and values lo + s q beside a tie of f16: the sum is rounded to f32, which is the tie, and
    then to f16."""
    rng = np.random.default_rng(17)
    x = rng.uniform(0, 1, (1, 4, 64, 256)) * 2.0 ** rng.integers(6, 14, (1, 4, 64, 1))
    x[..., ::64] = 2.0 ** -24 * rng.integers(1, 9, (1, 4, 64, 4))
    x = x.astype(np.float16)
    exact = R.value(*R.quantise(x))
    want = exact.astype(np.float32).astype(np.float16)
    assert (want != exact.astype(np.float16)).sum() > 1000
    ref = R.Cache(1, 1, 1, 1, fill=False)
    assert ref.resize([0], [64]) == 0
    c = upload(ctx, ref)
    d, kb, vb = ctx.upload(x.view(np.uint16)), ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    print("case: load, sums beside a tie", flush=True)
    ctx.kv4_store(c, 0, 0, 1, None, 64, d, d, 64)
    ctx.kv4_load(c, 0, 0, 1, None, 64, kb, vb, 64)
    for buf in (kb, vb):
        assert np.array_equal(ctx.download(buf, x.shape, np.float16), want)


def test_values_a_little_past_f16(ctx):
    """Groups that reach to 65504 stand for values of up to 65536: infinity where they are loaded as f16, finite in a step (of
    one token, whose output is its v times the gate)."""
    s = Step(ctx, [1], seed=113)
    s.v_new[0, :, ::2], s.v_new[0, :, 1::2] = 65504, -65504
    s.v_new[0, 1, ::2], s.v_new[0, 1, 1::2] = 65504, 0
    print("case: values past f16", flush=True)
    got, want = s.run(ctx, 1)
    assert np.isfinite(got).all()
    s.check(got / 65536, want / 65536)
    kb, vb = (ctx.alloc(4 * 256 * 2) for _ in range(2))
    ctx.kv4_load(s.c, 0, 0, 1, None, 1, kb, vb, 1)
    held = np.stack([s.ref.rows64(0, 0, head, 1)[0] for head in range(4)])
    assert held.max() == 65536 and held[1].max() == 65520
    with np.errstate(over="ignore"):
        assert np.array_equal(ctx.download(vb, (4, 1, 256), np.float16), held.astype(np.float32).astype(np.float16))


# ---- where the forms meet: one workgroup a head, or dealt and joined -------------------------
@pytest.mark.parametrize("n", [255, 256, 257, 384, 511, 512, 513])
def test_decode_lengths_around_the_forms_border(ctx, n):
    """One row: up to 256 tokens by one workgroup a head."""
    s = Step(ctx, [n], seed=120 + n)
    print(f"case: kv4 decode n={n}", flush=True)
    got, want = s.run(ctx, n)
    s.check(got, want)
    assert_same(ctx, s.c, s.ref)


@pytest.mark.parametrize("rows", [15, 16, 17, 23, 24, 25])
@pytest.mark.parametrize("most", [256, 257, 512, 513])
def test_decode_batches_around_the_forms_border(ctx, rows, most):
    """Ragged batches: up to 512 tokens a row by one workgroup a head from 24 rows on."""
    lens = np.random.default_rng(rows * most).integers(0, most + 1, rows)
    lens[[0, 3, 7]] = most, 0, 1
    s = Step(ctx, lens.tolist(), seed=121)
    print(f"case: kv4 decode of {rows} rows of up to {most}", flush=True)
    got, want = s.run(ctx, most)
    s.check(got, want)
    assert (got[lens == 0] == 0).all()
    assert_same(ctx, s.c, s.ref)


@pytest.mark.parametrize("lens", [[500, 1], [700, 1], [5001, 1]])
def test_decode_nan_in_a_group_of_long_rows(ctx, lens):
    """An infinity in the new k (kv head 1) and a NaN in the new v (head 2, dims 64 ..) of a row of many splits: NaN in its
    outputs there, none elsewhere, and none in the other row."""
    s = Step(ctx, lens, seed=122)
    s.k_new[0, 1, 200] = np.inf
    s.v_new[0, 2, 70] = np.nan
    s.v_new[1, 3, 0] = 1e6                        # beyond f16: an infinity there
    print(f"case: kv4 decode, NaN in groups, lens={lens}", flush=True)
    got, want = s.run(ctx, lens[0])
    bad = np.zeros_like(got, bool)
    bad[0, 4:8], bad[0, 8:12, 64:128], bad[1, 12:, :64] = True, True, True
    assert np.array_equal(np.isnan(got), bad)
    fine = np.where(np.isnan(want), 0, want), np.where(bad, 0, got)
    s.check(fine[1], fine[0])


# ---- beside the f16 cache's step ------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 40, 256, 257, 1500, 5000])
def test_step_agrees_with_the_f16_caches_step_and_the_oracle(ctx, n):
    """qm_gqa_decode over f16 rows and qm_gqa_decode_kv4 over the same rows in pages: rows of multiples of 1/8 with the whole
    range in every group, which 4 bits hold exactly, and a new token whose k is 0 (gamma = -1) and whose v is such a row.
    The f16 step's own bar (its weights enter the products in 16 bits) is 1e-3.  The oracle sums in f32: a score's 256
    products with A = sum |q k| / 16 of about 6 are off by 2^-24 * 16 * 6, the output's n terms of at most 1 by 2^-24 sqrt(n);
    six deviations of both are under 6e-5 up to n = 5000.  With another gamma the new k rows agree within half a step of the
    codes, a step of f16 for the f32 norm, and the roundings of the row read back."""
    from conftest import load_oracle, load_workloads
    O, W = load_oracle(), load_workloads()
    rng = np.random.default_rng(130 + n)

    def grid(*lead):
        x = rng.integers(0, 16, (*lead, 256)) * 0.125 - 1
        x[..., ::64], x[..., 1::64] = -1, 0.875
        return x.astype(np.float16)

    k, v = grid(1, 4, n), grid(1, 4, n)
    w = {x: rng.standard_normal((1, *shape), dtype=np.float32) for x, shape in (("q_gate", (16, 512)), ("k_new", (4, 256)))}
    w["v_new"] = grid(1, 4).astype(np.float32)
    q_norm = (0.1 * rng.standard_normal(256)).astype(np.float16)
    cos, sin = M.rope_table(n)
    rc, rs, qn = ctx.upload(cos), ctx.upload(sin), ctx.upload(q_norm)
    q_gate, k_new, v_new = (ctx.upload(w[x]) for x in ("q_gate", "k_new", "v_new"))
    kf, vf = ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16))
    c = M.Kv4Cache(ctx, 1, R.pages_of(n) + 2, 1, R.pages_of(n))
    assert run_resize(ctx, c, None, [n]) == 0
    ctx.kv4_store(c, 0, 0, 1, None, n, kf, vf, n)
    a, b = ctx.alloc(4096 * 4), ctx.alloc(4096 * 4)
    for gamma in (np.full(256, -1, np.float16), (0.1 * rng.standard_normal(256)).astype(np.float16)):
        kn = ctx.upload(gamma)
        print(f"case: both steps, n={n}", flush=True)
        ctx.gqa_decode(1, q_gate, k_new, v_new, qn, kn, rc, rs, n, None, n - 1, kf, vf, n, a)
        ctx.gqa_decode_kv4(c, 0, 1, None, q_gate, k_new, v_new, qn, kn, rc, rs, n, n, None, b)
        kb, vb = (ctx.alloc(4 * 256 * 2) for _ in range(2))
        ctx.kv4_load(c, 0, 0, 1, ints(ctx, [n - 1]), 1, kb, vb, 1)
        kb, vb = (ctx.download(x, (4, 256), np.float16).astype(np.float64) for x in (kb, vb))
        k16 = ctx.download(kf, (4, n, 256), np.float16)[:, n - 1].astype(np.float64)
        assert np.array_equal(vb, w["v_new"][0])
        step = np.repeat(np.ptp(k16.reshape(4, 4, 64), axis=-1) / 15, 64, axis=-1).reshape(4, 256)
        near = step * (0.5 + 2.0 ** -9) + 2.0 ** -10 * (np.abs(k16) + 16 * step)
        assert (np.abs(kb - k16) <= near).all()
        if gamma[0] != -1:
            continue
        assert not kb.any()
        f16, kv4 = (ctx.download(x, (16, 256), np.float32) for x in (a, b))
        K, V = (np.ascontiguousarray(np.transpose(x[0].astype(np.float32), (1, 0, 2))) for x in (k, v))
        want = O.attn_decode_step(O.config(), w["q_gate"].ravel(), w["k_new"].ravel(), w["v_new"].ravel(), q_norm.view(np.uint16),
                                  gamma.view(np.uint16), cos, sin, K, V, n - 1, round_kv_f16=True, nthreads=8).reshape(16, 256)
        print(f"f16 step {np.abs(kv4 - f16).max():.2e} oracle {np.abs(kv4 - want).max():.2e}", flush=True)
        assert np.abs(kv4 - f16).max() <= 1e-3
        assert np.abs(kv4 - want).max() <= 6e-5

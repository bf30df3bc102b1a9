"""CPU: the paged 4-bit KV cache without a device -- the numpy form that the GPU tests compare with, the
layout and the host's checks of the library's own headers (tests/cpp/kv4_test.cpp), the Rust struct."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

import kv4_reference as R
import test_rust_ffi as ffi
from conftest import PKG, load_mixer


def ask(lines):
    exe = PKG / "lib" / "kv4_test"
    assert exe.exists(), "build with qora-llm-4b_amd/build.py"
    r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = r.stdout.splitlines()
    assert len(out) == len(lines)
    return out


# ---- layout ---------------------------------------------------------------------------------
def test_header_layout_is_the_reference_layout_and_uses_every_bit_once():
    got = np.array([a.split() for a in ask([f"at {t} {d}" for t in range(32) for d in range(256)])], int).reshape(32, 256, 4)
    for is_v in (0, 1):
        word, nib = got[..., 2 * is_v], got[..., 2 * is_v + 1]
        assert np.array_equal(word * 4 + nib // 2, R.CODE_BYTE[is_v])
        assert np.array_equal(nib % 2 * 4, R.CODE_SHIFT[is_v])
    bits = np.concatenate([(got[..., 0] * 8 + got[..., 1]).ravel(), (got[..., 2] * 8 + got[..., 3]).ravel()])
    assert np.array_equal(np.sort(bits), np.arange(2 * 32 * 256))          # 8192 bytes of codes, each nibble once
    meta = np.array([a.split() for a in ask([f"meta {t} {g}" for t in range(32) for g in range(4)])], int)
    assert np.array_equal(meta[:, 0].reshape(32, 4), R.S_AT) and np.array_equal(meta[:, 1].reshape(32, 4), R.LO_AT)
    for column in meta.T:
        assert np.array_equal(np.sort(column), np.arange(128))
    assert 8192 + 4 * 256 == R.HALF_BYTES and 8 * R.HALF_BYTES == R.PAGE == load_mixer().QM_KV4_PAGE_BYTES


def test_put_and_get_agree_and_leave_the_other_tokens():
    rng = np.random.default_rng(1)
    page = rng.integers(0, 256, R.PAGE, dtype=np.uint8)
    page.reshape(8, R.HALF_BYTES)[:, 8192:] = 0x30                           # finite scales and minima
    before = [[R.get(page, h, v) for v in (0, 1)] for h in range(4)]
    x = rng.standard_normal(256).astype(np.float16)
    R.put(page, 2, 45, x, 1)
    for h in range(4):
        for v in (0, 1):
            now, was = R.get(page, h, v), before[h][v]
            if (h, v) == (2, 1):
                assert np.array_equal(now[45], R.value(*R.quantise(x)))
                now, was = np.delete(now, 45, 0), np.delete(was, 45, 0)
            assert np.array_equal(now, was)


# ---- values ---------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1e-7, 1e-6, 1e-3, 1.0, 300.0, 2e4])
def test_values_are_within_half_a_step(scale):
    """Within s / 2, or within 15 2^-25 where the rounding of a subnormal s costs more."""
    x = (np.random.default_rng(2).standard_normal((50, 256)) * scale).clip(-65504, 65504).astype(np.float16)
    q, s, lo = R.quantise(x)
    err = np.abs(R.value(q, s, lo) - x.astype(np.float64)).reshape(50, 4, 64).max(-1)
    assert (err <= np.maximum(s.astype(np.float64) / 2, 15 * 2.0 ** -25)).all()


def test_values_of_odd_cus():
    x = np.zeros((1, 256), np.float16)
    x[0, :64] = 3.5                                                           # one value: exact
    x[0, 64:128] = np.tile([-65504, 65504], 32)                               # the widest range
    x[0, 130] = np.inf
    x[0, 200] = np.nan
    got = R.value(*R.quantise(x))[0]
    assert (got[:64] == 3.5).all()
    assert (np.abs(got[64:128] - x[0, 64:128]) <= 8736 / 2).all()
    assert np.isnan(got[128:]).all()


# ---- pages ----------------------------------------------------------------------------------
def some_steps(seed, count=60, rows=7, num_pages=24, max_pages=5, fill=False):
    """A seeded run of calls on a cache: yields (what, arguments) for the caller to make of its own cache too."""
    rng = np.random.default_rng(seed)
    for _ in range(count):
        kind = rng.choice(["resize", "resize", "add", "fork", "compact"], p=[0.3, 0.2, 0.25, 0.2, 0.05])
        n = int(rng.integers(1, rows + 1))
        pick = rng.permutation(rows)[:n].astype(np.int32)
        if kind == "resize":
            lens = rng.integers(0, max_pages * 64 + 1, n).astype(np.int32)
            lens[rng.random(n) < 0.3] = 0
            yield "resize", (pick, lens, False)
        elif kind == "add":
            yield "resize", (pick, rng.integers(-3, 70, n).astype(np.int32), True)
        elif kind == "fork":
            yield "fork", (rng.integers(0, rows, n).astype(np.int32), pick)
        else:
            yield "compact", ()


@pytest.mark.parametrize("seed", range(6))
def test_reference_pages_stay_consistent(seed):
    """Counts are the tables'; what a row held stays its own through forks, copies and moves."""
    c = R.Cache(1, 24, 7, 5, fill=False)
    mine = {}                                   # row -> what its pages should hold, by page index
    stamp, results = 0, set()
    for kind, args in some_steps(seed):
        old = c.lens.copy()
        got = getattr(c, kind)(*args)
        results.add(np.sign(got))
        assert c.consistent()
        if kind == "resize" and got == 0:
            for r in args[0]:
                mine[r] = mine.get(r, [])[:R.pages_of(int(c.lens[r]))]
                if c.lens[r] > old[r]:          # a step writes: into the page of the first new token, and on
                    for j in range(old[r] // 64, R.pages_of(int(c.lens[r]))):
                        assert c.refs[c.table[r, j]] == 1
                        stamp += 1
                        c.pages[0, c.table[r, j], :4] = np.frombuffer(np.int32(stamp).tobytes(), np.uint8)
                        mine[r] = mine[r][:j] + [stamp]
        if kind == "fork" and got == 0:
            was = {r: list(v) for r, v in mine.items()}
            for s, d in zip(*args):
                mine[d] = list(was.get(s, []))
        if kind == "compact":
            assert (c.refs[:got] > 0).all() and not c.refs[got:].any()
        for r, stamps in mine.items():
            held = [int(c.pages[0, p, :4].copy().view(np.int32)[0]) for p in c.ids(r)]
            assert held == stamps, (kind, r)
    assert {0, 1} <= results


# ---- the host's checks ----------------------------------------------------------------------
GOOD = "cache 4096 8192 8196 8200 8 100 16 32"


def test_refusals_of_caches():
    calls = ["resize 3 0 64 0 64", "fork 3 64 64 64", "compact 64", "rows 0 0 1 0 5 64 64 5", "decode 0 4 0 64 2048 2048 0"]
    ok = ask([GOOD] + calls)
    assert [a.split()[0] for a in ok[1:]] == ["0"] * 5
    for bad, code in [("0 8192 8196 8200 8 100 16 32", 3), ("4096 0 8196 8200 8 100 16 32", 3), ("4096 8192 0 8200 8 100 16 32", 3),
                      ("4096 8192 8196 0 8 100 16 32", 3), ("4104 8192 8196 8200 8 100 16 32", 3),
                      ("4096 8193 8196 8200 8 100 16 32", 3), ("4096 8192 8196 8202 8 100 16 32", 3),
                      ("4096 8192 8196 8200 0 100 16 32", 3), ("4096 8192 8196 8200 8 -1 16 32", 3),
                      ("4096 8192 8196 8200 8 100 0 32", 3), ("4096 8192 8196 8200 8 100 16 0", 3),
                      ("4096 8192 8196 8200 8 100 65537 32", 4), ("4096 8192 8196 8200 8 4194304 16 32", 4), ("4096 8192 8196 8200 8 100 16 33554432", 4)]:
        got = ask([f"cache {bad}"] + calls)[1:]
        assert [a.split()[0] for a in got] == [str(code)] * 5, (bad, got)
        assert all(len(a.split()) > 1 for a in got)


@pytest.mark.parametrize("call, code", [
    ("resize 0 0 64 0 64", 3), ("resize 17 0 64 0 64", 3), ("resize 3 0 0 0 64", 3), ("resize 3 0 64 0 0", 3),
    ("resize 3 0 64 2 64", 3), ("resize 3 2 64 0 64", 3), ("resize 3 0 66 0 64", 3), ("resize 3 0 64 1 65", 3),
    ("fork 0 64 64 64", 3), ("fork 3 0 64 64", 3), ("fork 3 64 0 64", 3), ("fork 3 64 64 0", 3), ("fork 3 64 62 64", 3),
    ("compact 0", 3), ("compact 2", 3),
    ("rows -1 0 1 0 5 64 64 5", 3), ("rows 8 0 1 0 5 64 64 5", 3), ("rows 0 -1 1 0 5 64 64 5", 3), ("rows 0 16 1 0 5 64 64 5", 3),
    ("rows 0 10 7 0 5 64 64 5", 3), ("rows 0 0 0 0 5 64 64 5", 3), ("rows 0 0 1 0 0 64 64 5", 3), ("rows 0 0 1 0 5 0 64 5", 3),
    ("rows 0 0 1 0 5 64 0 5", 3), ("rows 0 0 1 0 5 72 64 5", 3), ("rows 0 0 1 3 5 64 64 5", 3), ("rows 0 0 1 0 5 64 64 4", 6),
    ("rows 0 2147483647 1 0 5 64 64 5", 3), ("rows 0 0 2147483647 0 5 64 64 5", 3),
    ("decode -1 4 0 64 2048 2048 0", 3), ("decode 8 4 0 64 2048 2048 0", 3), ("decode 0 0 0 64 2048 2048 0", 3),
    ("decode 0 17 0 64 2048 2048 0", 3), ("decode 0 4 0 0 2048 2048 0", 3), ("decode 0 4 0 72 2048 2048 0", 3),
    ("decode 0 4 2 64 2048 2048 0", 3), ("decode 0 4 0 64 2048 2048 1", 3), ("decode 0 4 0 64 2048 0 0", 3),
    ("decode 0 4 0 64 2047 2048 0", 5), ("decode 0 4 0 64 4096 2049 0", 6)])
def test_refusals_of_calls(call, code):
    got = ask([GOOD, call])[1]
    assert got.split()[0] == str(code) and len(got.split()) > 1, got


def test_a_batch_may_be_larger_than_the_table_with_slots():
    assert ask([GOOD, "decode 0 17 64 64 2048 2048 0"])[1].split()[0] == "0"


def test_entries_refuse_a_null_context():
    lib = load_mixer().load_library()
    assert lib.qm_kv4_resize(None, None, None, 1, None, None, 0, None) == 3
    assert lib.qm_kv4_fork(None, None, None, 1, None, None, None) == 3
    assert lib.qm_kv4_compact(None, None, None, None) == 3
    assert lib.qm_kv4_store(None, None, None, 0, 0, 1, None, 1, None, None, 1) == 3
    assert lib.qm_kv4_load(None, None, None, 0, 0, 1, None, 1, None, None, 1) == 3
    assert lib.qm_gqa_decode_kv4(None, None, None, 0, 1, *([None] * 8), 1, 1, None, None) == 3


def dealt(lens, cus):
    """The kernel's rule (deal_chunk) on the rows' lengths: tokens per split, splits of all rows."""
    count = lambda chunk: sum(-(-n // chunk) for n in lens)

    def chunk_for(want, groups):
        chunk = (int(min(want, 4095)) + 128) // 128 * 128
        for _ in range(4 if len(lens) <= 64 else 0):
            if chunk >= 4096 or 4 * count(chunk) <= groups:
                break
            chunk += 128
        return chunk

    want = np.float32(sum(lens)) * 4 / np.float32(cus)
    rounds = max(int(np.ceil(want / 8192 - 2.0 ** -7)), 1)
    if rounds > 64:
        return 4096, count(4096)
    one, two = chunk_for(want, cus), chunk_for(want / 2 / rounds, 2 * cus * rounds)
    few = one == 128 or 10 * one <= 17 * two or max(lens) > 32 * two
    chunk = one if want < 4095 and few and one < 4096 else two
    return chunk, count(chunk)


def test_splits_fit_the_grid_and_the_reserve():
    rng = np.random.default_rng(4)
    cases = []
    for most in (129, 500, 4097, 32769, 131072, 2 ** 20, 2 ** 31 - 1):
        for batch in (1, 2, 7, 19, 64, 65, 300):
            for cus in (4, 32, 256):
                cases.append(([most] * batch, most, batch, cus))
                cases.append((rng.integers(0, most + 1, batch).tolist(), most, batch, cus))
                cases.append((np.minimum(most, rng.integers(1, 200, batch)).tolist(), most, batch, cus))
    got = [[int(x) for x in a.split()] for a in ask([f"splits {m} {b} {g}" for _, m, b, g in cases])]
    for (lens, most, batch, cus), (bound, ws, reserve) in zip(cases, got):
        chunk, n = dealt(lens, cus)
        assert chunk % 128 == 0 and 128 <= chunk <= 4096
        assert n <= bound and ws <= reserve, (most, batch, cus)
    # a reserve for the largest covers the smaller
    reserve = int(ask(["splits 32769 64 256"])[0].split()[2])
    for n in (129, 700, 4097, 32769):
        assert all(int(a.split()[1]) <= reserve for a in ask([f"splits {n} {b} 256" for b in range(1, 65)]))


def test_rust_struct_matches_the_header():
    assert ffi._c_struct_fields("qm_kv4_cache") == ffi._r_struct_fields("qm_kv4_cache")


def test_a_reserve_covers_every_call_within_its_limits():
    """Resize, fork, compaction and step at the limits that qm_reserve names, and at smaller ones."""
    exe = PKG / "lib" / "kv4_reserve_test"
    assert exe.exists(), "build with qora-llm-4b_amd/build.py"

    def sizes(cases):
        r = subprocess.run([str(exe)], input="\n".join(f"{b} {n} {g}" for b, n, g in cases) + "\n", capture_output=True,
                           text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        return [[int(x) for x in a.split()] for a in r.stdout.splitlines()]

    batches, lens = (1, 2, 19, 64, 300, 1024, 3000), (1, 64, 65, 256, 4097, 32769, 1048576)
    cases = [(b, n, g) for b in batches for n in lens for g in (4, 256)]
    got = sizes(cases)
    assert len(got) == len(cases)
    for case, (*calls, reserve) in zip(cases, got):
        assert max(calls) <= reserve, (case, calls, reserve)
    most = got[cases.index((300, 32769, 256))][-1]
    assert all(max(calls) <= most for (b, n, g), (*calls, _) in zip(cases, got) if b <= 300 and n <= 32769 and g == 256)

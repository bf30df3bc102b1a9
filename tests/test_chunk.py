"""CPU: chunks of new tokens and beam search's step without a device -- what the host refuses, the workspaces
that it asks for against what the kernels need (tests/cpp/chunk_test.cpp), and the Rust struct."""
from __future__ import annotations

import random
import subprocess

import pytest

import test_rust_ffi as ffi
from conftest import PKG

OK, INVALID, SHAPE, ROPE, CAPACITY = 0, 3, 4, 5, 6


def ask(lines):
    exe = PKG / "lib" / "chunk_test"
    assert exe.exists(), "build with qora-llm-4b_amd/build.py"
    r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = r.stdout.splitlines()
    assert len(out) == len(lines)
    return out


# ---- refusals -------------------------------------------------------------------------------
RAGGED = [
    ("", OK), ("cache=0", INVALID), ("pages=0", INVALID), ("table=0", INVALID), ("lens=0", INVALID), ("refs=0", INVALID),
    ("pages=4104", INVALID), ("table=8193", INVALID), ("lens=12290", INVALID), ("refs=16387", INVALID),
    ("layers=0", INVALID), ("num_pages=0", INVALID), ("num_pages=4194304", SHAPE), ("rows=65537", SHAPE), ("max_pages=33554432", SHAPE),
    ("layer=-1", INVALID), ("layer=2", INVALID), ("layer=1", OK),
    ("batch=0", INVALID), ("batch=9", INVALID), ("batch=9 slots=64", OK), ("batch=65536 slots=64", OK), ("batch=65537 slots=64", INVALID),
    ("slots=66", INVALID), ("begins=0", INVALID), ("begins=6", INVALID), ("result=4", OK), ("result=5", INVALID),
    ("tokens=0", INVALID), ("tokens=-1", INVALID), ("tokens=1", OK), ("tokens=1048576", OK), ("tokens=1048577", INVALID),
    ("norm=0", INVALID), ("cos=0", INVALID), ("sin=0", INVALID), ("norm=65544", INVALID), ("cos=65540", INVALID), ("sin=65538", INVALID),
    ("max_len=0", INVALID), ("max_len=-5", INVALID), ("max_len=1025", ROPE), ("max_len=1025 rope_len=1025", CAPACITY),
    ("max_len=1 rope_len=1", OK), ("max_pages=33554431 max_len=2147483584 rope_len=2147483647", OK),
    ("max_pages=33554431 max_len=2147483585 rope_len=2147483647", CAPACITY)]


@pytest.mark.parametrize("what, more", [
    ("append", [("dtype=0", OK), ("dtype=2", OK), ("dtype=1", INVALID), ("dtype=7", INVALID), ("k=0", INVALID), ("v=0", INVALID), ("k=65544", INVALID), ("v=65537", INVALID)]),
    ("chunk", [("max_new=0", INVALID), ("max_new=-1", INVALID), ("max_new=1", OK), ("max_new=2147483647", OK), ("q=0", INVALID),
               ("out=0", INVALID), ("q=65544", INVALID), ("out=65540", INVALID)])])
def test_ragged_calls_are_refused(what, more):
    cases = RAGGED + more
    for (keys, code), got in zip(cases, ask([f"{what} {keys}" for keys, _ in cases])):
        assert int(got.split()[0]) == code, (keys, got)
        assert code == OK or len(got.split()) > 3, (keys, got)


def test_selections_are_refused():
    cases = [("", OK), ("groups=0", INVALID), ("vocab=0", INVALID), ("beams=0", INVALID), ("beams=65", INVALID), ("beams=64 take=64", OK),
             ("take=0", INVALID), ("take=65", INVALID), ("take=64", OK), ("vocab=262144", OK), ("vocab=262145", SHAPE),
             ("groups=16384", OK), ("groups=16385", SHAPE), ("groups=2147483647 beams=64", SHAPE), ("logits=0", INVALID), ("scores=0", INVALID),
             ("parents=0", INVALID), ("tokens=0", INVALID), ("out_scores=0", INVALID), ("logits=258", INVALID), ("scores=513", INVALID),
             ("done=2", INVALID), ("parents=770", INVALID), ("tokens=1025", INVALID), ("out_scores=1282", INVALID), ("out_done=3", INVALID),
             ("end_id=-2", INVALID), ("end_id=1000", INVALID), ("end_id=999", OK), ("done=64", INVALID), ("done=64 end_id=0", OK),
             ("out_scores=512", OK), ("out_scores=512 take=5", INVALID), ("done=64 end_id=3 out_done=64", OK),
             ("done=64 end_id=3 out_done=64 take=3", INVALID)]
    for (keys, code), got in zip(cases, ask([f"select {keys}" for keys, _ in cases])):
        assert int(got.split()[0]) == code, (keys, got)


def test_forks_of_states_are_refused():
    cases = [("", OK), ("buffers=0", INVALID), ("buffers=64", OK), ("buffers=65", INVALID), ("list=0", INVALID), ("rows=0", INVALID),
             ("rows=65536", OK), ("rows=65537", INVALID), ("count=0", INVALID), ("count=11", INVALID), ("count=10", OK),
             ("rows=2000 count=1024", OK), ("rows=2000 count=1025", INVALID), ("src=0", INVALID), ("result=0", INVALID), ("src=258", INVALID),
             ("dst=64", OK), ("dst=66", INVALID), ("result=514", INVALID), ("rows_dev=0", INVALID), ("rows_dev=4104", INVALID),
             ("row_bytes=0", INVALID), ("row_bytes=-16", INVALID), ("row_bytes=24", INVALID), ("row_bytes=80", INVALID),
             ("row_bytes=16", OK), ("stride_bytes=72", INVALID), ("stride_bytes=48", INVALID),
             ("stride_bytes=140737488355312", OK), ("stride_bytes=140737488355328", INVALID)]
    for (keys, code), got in zip(cases, ask([f"fork {keys}" for keys, _ in cases])):
        assert int(got.split()[0]) == code, (keys, got)


# ---- workspaces ------------------------------------------------------------------------------
def test_row_blocks_and_half_pages_stay_within_what_the_host_counts():
    """Over random splits of tokens into rows: the records of all row blocks, and the grid of half pages."""
    rng = random.Random(1)
    shapes, wants, halves, touched = [], [], [], []
    for _ in range(400):
        batch = rng.choice([1, 2, 3, 7, 20, 64, 65, 150])
        top = rng.choice([1, 4, 5, 8, 32, 33, 64, 65, 200])
        news = [rng.choice([0, 1, top, rng.randrange(top + 1)]) for _ in range(batch)]
        if not any(news):
            news[0] = 1
        tokens, max_new = sum(news) + rng.choice([0, 0, 5]), max(news)
        shapes.append(f"shape {tokens} {batch} {max_new} {rng.choice([300, 5000, 1 << 20])} 256")
        wants.append((news, max_new))
        firsts = [rng.randrange(1000) for _ in news]
        halves.append(f"halves {tokens} {batch}")
        touched.append(sum((f + n - 1) // 32 - f // 32 + 1 for f, n in zip(firsts, news) if n))
    for (news, max_new), got in zip(wants, ask(shapes)):
        columns, many, split, most_many, most_few, groups, ws = (int(x) for x in got.split())
        assert columns == (1 if max_new <= 4 else 2) and (not many or max_new > 32)
        assert sum(-(-n // 64) for n in news if n > 32 and many) <= most_many
        assert sum(-(-n // (4 * columns)) for n in news if n <= 32 or not many) <= most_few
        assert 1 <= groups <= 64
        assert ws >= 16 + 32 * (most_many + most_few) + (split and groups * 4 * 2 * (16 if many else columns) * 4128 * 4)
    for want, got in zip(touched, ask(halves)):
        assert want <= int(got)


def test_a_reserve_covers_the_calls_within_it():
    rng = random.Random(2)
    for cus in (1, 64, 256, 304):
        for tokens, batch, max_len in [(1, 1, 64), (40, 3, 700), (4096, 24, 12000), (65536, 256, 1 << 20), (1 << 20, 65536, 1 << 27)]:
            reserve = int(ask([f"reserve {tokens} {batch} {max_len} {cus}"])[0])
            lines = []
            for _ in range(100):
                t = rng.choice([1, tokens, rng.randrange(1, tokens + 1)])
                b = rng.choice([1, batch, rng.randrange(1, batch + 1)])
                lines.append(f"shape {t} {b} {rng.choice([1, 4, 5, 8, 32, 33, 64, t])} {rng.choice([1, max_len, rng.randrange(1, max_len + 1)])} {cus}")
            for line, got in zip(lines, ask(lines)):
                assert int(got.split()[-1]) <= reserve, line


def test_a_loose_bound_of_a_rows_new_tokens_is_the_calls():
    """No row has more new tokens than the call: max_new past that picks no other kernel and no larger workspace."""
    for tokens, batch, max_len in [(1, 1, 100), (3, 2, 20000), (4, 1, 5000), (5, 1, 5000), (20, 4, 300000), (32, 1, 1 << 20), (33, 2, 1 << 20), (700, 3, 9000)]:
        tight, *loose = ask([f"shape {tokens} {batch} {m} {max_len} 256" for m in (tokens, tokens + 1, 64, 4096, 2147483647) if m >= tokens])
        assert all(x == tight for x in loose), (tokens, tight, loose)


def test_a_reserve_for_few_tokens_takes_no_more_than_they_need():
    """Blocks of many tokens leave 135 MB of partial sums; a reserve whose calls have none does not ask for them."""
    of = {k: int(x) for k, x in zip([(1, 32768), (4, 1 << 20), (16, 32768), (32, 1 << 20), (33, 32768), (512, 4096), (513, 4096), (33, 65536)], ask(
        ["reserve 1 1 32768 256", "reserve 4 1 1048576 256", "reserve 16 1 32768 256", "reserve 32 1 1048576 256", "reserve 33 1 32768 256",
         "reserve 512 1 4096 256", "reserve 513 1 4096 256", "reserve 33 1 65536 256"]))}
    column = 64 * 4 * 2 * 4128 * 4
    for key, columns in {(1, 32768): 1, (4, 1 << 20): 1, (16, 32768): 2, (32, 1 << 20): 2, (33, 32768): 2, (512, 4096): 2}.items():
        assert of[key] <= columns * column + 16 + 32 * 600, key
    assert of[513, 4096] >= 16 * column and of[33, 65536] >= 16 * column


def test_selections_workspaces_and_the_states_columns():
    got = [int(x) for x in ask(["slices 1 1", "slices 4 1024", "slices 4 1025", "slices 65536 262144"])]
    assert got == [16, 64, 128, 65536 * 256 * 16]
    for n, got in zip((1, 32, 33, 64, 65, 128, 129, 300, 1024), ask([f"column {n}" for n in (1, 32, 33, 64, 65, 128, 129, 300, 1024)])):
        wide = int(got)
        assert wide % 16 == 0 and 16 <= wide <= 4096 and (n <= 128 or n * wide <= 65536)
        assert n > 128 or wide == 256 * (16 if n <= 32 else 8 if n <= 64 else 4)


def test_rust_struct_matches_the_header():
    assert ffi._c_struct_fields("qm_state_rows") == ffi._r_struct_fields("qm_state_rows")

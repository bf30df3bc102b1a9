"""GPU: lists of qm_kv4_append that are filled up with entries of no tokens, byte for byte against numpy."""
from __future__ import annotations

import numpy as np
import pytest

import chunk_reference as CR
from conftest import load_mixer
from test_chunk_gpu import begins_of, cache_of, rope
from test_kv4_gpu import assert_same, ints, upload

pytestmark = pytest.mark.gpu

M = load_mixer()


def run(ctx, ref, slots, begins, dtype, seed):
    begins, batch, tokens = np.asarray(begins, np.int32), len(slots), 40 + max(begins)
    rng = np.random.default_rng(seed)
    k, v = rng.standard_normal((2, tokens, 4, 256)).astype(np.float32)
    gamma = (0.1 * rng.standard_normal(256)).astype(np.float16)
    most = int(ref.lens.max())
    cos, sin = rope(most)
    if dtype == "bf16":
        k, v = CR.bf16(k), CR.bf16(v)
    c = upload(ctx, ref)
    print(f"case: append {dtype} slots={slots[:9]} begins={begins[:9]}", flush=True)
    ctx.kv4_append(c, 0, batch, ints(ctx, slots), ints(ctx, begins), tokens, ctx.upload(k), ctx.upload(v), ctx.upload(gamma.view(np.uint16)),
                   ctx.upload(cos), ctx.upload(sin), len(cos), most, None, dtype=M.QM_BF16 if dtype == "bf16" else M.QM_F32)
    if dtype == "bf16":
        k, v = CR.bf16_value(k), CR.bf16_value(v)
    # the entries that have tokens are what is to be written
    of = [r if span else -1 for r, span in zip(slots, CR.ranges(begins, tokens, batch))]
    CR.append(ref, 0, batch, of, begins, tokens, k, v, gamma, cos, sin, most)
    assert_same(ctx, c, ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_entries_without_tokens_leave_no_row_out(ctx, dtype):
    """Idle entries that say 0, or any other row, before that row's own entry and behind it."""
    run(ctx, cache_of([40, 70, 130, 9], layers=1, seed=16), [0, 2, 2, 0, 0, 1, 0], [0, 0, 0, 7, 12, 12, 32, 32], dtype, 1)


def test_of_a_row_listed_twice_the_first_with_tokens_is_written(ctx):
    run(ctx, cache_of([40, 70], layers=1, seed=17), [1, 0, 1, 0, 1, 0], [3, 3, 20, 25, 30, 62, 90], "f32", 2)


def test_entries_whose_range_is_none_of_the_tensor_leave_no_row_out(ctx):
    run(ctx, cache_of([40, 70], layers=1, seed=18), [1, 0, 1, 0], [-2, 500, 6, 20, 30], "f32", 3)


def test_a_list_longer_than_a_wave(ctx):
    rng = np.random.default_rng(19)
    lens = rng.integers(1, 80, 150).tolist()
    slots = rng.permutation(150)
    news = [int(rng.integers(1, lens[r] + 1)) for r in slots]
    run(ctx, cache_of(lens, layers=1, seed=19), [0] * 70 + slots.tolist() + [5] * 70, begins_of([0] * 70 + news + [0] * 70), "bf16", 4)

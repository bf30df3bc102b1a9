"""GPU: attention of new tokens over the paged 4-bit cache where one key leads the others, against numpy in 64 bits.

A token whose score is 12 to 18 nats above the rest (the first one of many models' sequences) and whose V is next to
nothing leaves the output to thousands of keys of small weight.  A weight is f16: 2^-11 of itself, which
chunk_reference.attend counts, and below 2^-14 2^-25 at most.  The leading key's weight is 2^7 or more where its
row's sums are kept, so that in units of it the latter is 2^-32 a key: n 2^-32 max |V| of an output, as the leading
weight alone makes the sum 1 or more, and n 2^-32 of itself, the sum's own.  In the 2-norm of a row these are
independent: 2^-32 / sqrt(3) a key against weights of e^-18 = 2^-26 and more, 1% of a key's and, as V's signs are
random, 1% / sqrt(n) of a row's; n = 6001: 1.2e-4, nothing beside the 3e-3 that stand for the other roundings.
"""
from __future__ import annotations

import numpy as np
import pytest

import chunk_reference as CR
import kv4_reference as R
from conftest import load_mixer
from test_chunk_gpu import begins_of, cache_of, ints, rope, upload

pytestmark = pytest.mark.gpu

M = load_mixer()


def leading(rng, ref, at, beta):
    """Token `at` of the row gets K of +-beta in the dims that do not turn, and V of 0.  The signs."""
    sign = np.where(rng.random(256) < 0.5, -1.0, 1.0)
    sign[:64] = 0
    page = ref.pages[0, ref.table[0, at // R.TOKENS]]
    for head in range(R.KV):
        R.put(page, head, at % R.TOKENS, (beta * sign).astype(np.float16), 0)
        R.put(page, head, at % R.TOKENS, np.zeros(256, np.float16), 1)
    return sign


@pytest.mark.parametrize("new", [3, 20, 400])
@pytest.mark.parametrize("at", [0, 2900])
@pytest.mark.parametrize("nats", [12, 15, 18])
def test_chunk_where_one_key_leads(ctx, nats, at, new):
    n, seed = 6001, 100 + nats + at + new
    rng = np.random.default_rng(seed)
    ref = cache_of([n], layers=1, seed=seed)
    # q is unit noise and the signs, normed: the signs' share is 1 / sqrt(1 + 192 / 256) of each of 192 dims
    sign = leading(rng, ref, at, nats * 16 / 192 * (1 + 192 / 256) ** 0.5)
    x = rng.standard_normal((new, 16, 512))
    x[:, :, :256] += sign
    q, gamma = CR.bf16(x), np.zeros(256, np.float16)
    cos, sin = rope(n)
    c, out = upload(ctx, ref), ctx.alloc(new * 8192)
    print(f"case: one key leads, nats={nats} at={at} new={new}", flush=True)
    ctx.gqa_chunk_kv4(c, 0, 1, None, ints(ctx, begins_of([new])), new, new, ctx.upload(q), ctx.upload(gamma.view(np.uint16)), ctx.upload(cos),
                      ctx.upload(sin), len(cos), n, None, out)
    got = CR.bf16_value(ctx.download(out, (new, 16, 256), np.uint16)).astype(np.float64)
    want, bound, _ = CR.attend(ref, 0, 1, None, begins_of([new]), new, new, CR.bf16_value(q), gamma, cos, sin, n)
    small = max(np.abs(CR.kept(ref, 0, 0, head, 1)[0]).max() for head in range(R.KV))
    bound = bound + n * 2.0 ** -32 * (small + np.abs(want))
    off = np.abs(got - want)
    assert (off <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
    # each row as much as another, however small it is
    size = np.linalg.norm(want, axis=-1)
    rms = np.sqrt(np.mean((np.linalg.norm(got - want, axis=-1) / size) ** 2))
    print("rows' error, rms:", rms)
    assert rms <= 3e-3

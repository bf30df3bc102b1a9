"""New tokens of ragged rows over the paged 4-bit KV cache, and beam search's step, in numpy and 64 bits."""
from __future__ import annotations

import numpy as np

import kv4_reference as R


def bf16(x) -> np.ndarray:
    """f32 values rounded to bf16 (to nearest even), as uint16 bits."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(bits) -> np.ndarray:
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def ranges(begins, tokens, batch):
    """The batch rows' packed rows, None where there are none."""
    out = []
    for b in range(batch):
        lo, hi = int(begins[b]), int(begins[b + 1])
        out.append((lo, hi) if 0 <= lo < hi <= tokens else None)
    return out


def turned(x, gamma, cos, sin, at):
    """Rows [n, heads, 256] normed and rotated to positions at .. at + n - 1, f64."""
    return np.stack([R._turn(x[i], gamma, cos[at + i], sin[at + i]) for i in range(len(x))])


def append(ref: R.Cache, layer, batch, slots, begins, tokens, k, v, k_norm, cos, sin, max_len):
    """k, v values [tokens, 4, 256]."""
    seen = set()
    for b, span in enumerate(ranges(begins, tokens, batch)):
        r = b if slots is None else int(slots[b])
        repeated = r in seen
        seen.add(r)
        if span is None or repeated or not 0 <= r < len(ref.lens):
            continue
        lo, hi = span
        n, length = hi - lo, int(ref.lens[r])
        if n > length or length > max_len:
            continue
        kept = turned(k[lo:hi], k_norm, cos, sin, length - n).astype(np.float32).astype(np.float16)
        with np.errstate(over="ignore"):
            vh = v[lo:hi].astype(np.float16)
        for i in range(n):
            t = length - n + i
            p = ref.table[r, t // R.TOKENS]
            if not ref.is_page(p) or ref.refs[p] != 1:
                continue
            for head in range(R.KV):
                R.put(ref.pages[layer, p], head, t % R.TOKENS, kept[i, head], 0)
                R.put(ref.pages[layer, p], head, t % R.TOKENS, vh[i, head], 1)


def kept(ref: R.Cache, layer, r, head, is_v):
    """rows64 as attention takes it: a scale that takes its group past f16's largest value is the next lower one."""
    n = int(ref.lens[r])
    out, there = np.zeros((R.pages_of(n) * R.TOKENS, R.HD)), np.zeros(R.pages_of(n) * R.TOKENS, bool)
    for j in range(R.pages_of(n)):
        if not ref.is_page(ref.table[r, j]):
            continue
        page = ref.pages[layer, ref.table[r, j]].copy()
        for half in range(2):
            meta = R._half(page, head, half * R.HALF)[8192:].view(np.float16)
            s, lo = meta[256 * is_v + R.S_AT], meta[256 * is_v + 128 + R.LO_AT]
            with np.errstate(invalid="ignore"):
                over = lo.astype(np.float64) + 15 * s.astype(np.float64) >= 65520
            meta[256 * is_v + R.S_AT] = np.where(over, np.nextafter(s, np.float16(0)), s)
        out[j * R.TOKENS:(j + 1) * R.TOKENS] = R.get(page, head, is_v)
        there[j * R.TOKENS:(j + 1) * R.TOKENS] = True
    return out[:n], there[:n]


def attend(ref: R.Cache, layer, batch, slots, begins, tokens, max_new, q_gate, q_norm, cos, sin, max_len):
    """q_gate values [tokens, 16, 512] -> out f64 [tokens, 16, 256] (untouched rows: 7), the bound of each output's
    error before it is rounded, and which rows were touched.

    The bound: q, K and V are rounded to f16 once, p too, each by 2^-11 of itself; the f32 sums and exponentials by
    much less (2^-20 stands for them).  A score is off by a = (2^-10 + 2^-20) A at most, A the sum of its terms'
    absolute values; weights in the quotient then by e^(2 a) - 1, and with p and V's roundings an output by
    (e^(2 a) - 1 + 2^-10 + 2^-19) times its weighted sum of |V|, times the gate."""
    out = np.full((tokens, 16, 256), 7.0)
    bound = np.zeros((tokens, 16, 256))
    touched = np.zeros(tokens, bool)
    for b, span in enumerate(ranges(begins, tokens, batch)):
        if span is None:
            continue
        lo, hi = span
        touched[lo:hi] = True
        out[lo:hi] = 0.0
        r = b if slots is None else int(slots[b])
        if not 0 <= r < len(ref.lens) or ref.lens[r] <= 0:
            continue
        n, length = hi - lo, int(ref.lens[r])
        if n > length or length > max_len or n > max_new:
            out[lo:hi] = np.nan
            continue
        q = turned(q_gate[lo:hi, :, :256], q_norm, cos, sin, length - n) / 16
        gate = 1 / (1 + np.exp(-q_gate[lo:hi, :, 256:].astype(np.float64)))
        pos = length - n + np.arange(n)
        for g in range(R.KV):
            K, there = kept(ref, layer, r, g, 0)
            V, _ = kept(ref, layer, r, g, 1)
            sees = there & (np.arange(length) <= pos[:, None])
            for h in range(4 * g, 4 * g + 4):
                s = np.where(sees, q[:, h] @ np.nan_to_num(K).T, -np.inf)
                kbad = ~np.isfinite(K).all(-1)
                lost = (sees & kbad).any(-1)
                A = np.abs(q[:, h]) @ np.nan_to_num(np.abs(K)).T
                a = (2.0 ** -10 + 2.0 ** -20) * np.where(sees, A, 0).max(-1, initial=0)
                any_ = sees.any(-1)
                top = np.where(any_, s.max(-1, initial=-np.inf), 0)
                p = np.where(sees, np.exp(s - top[:, None]), 0)
                total = np.where(any_, p.sum(-1), 1)
                y = p @ np.nan_to_num(V) / total[:, None]
                # a value that is NaN reaches those that see it, whatever its weight
                y[(sees.astype(float) @ (~np.isfinite(V)).astype(float)) > 0] = np.nan
                y[lost] = np.nan
                out[lo:hi, h] = y * gate[:, h]
                size = p @ np.abs(np.nan_to_num(V)) / total[:, None]
                bound[lo:hi, h] = (np.expm1(2 * a)[:, None] + 2.0 ** -10 + 2.0 ** -19) * size * gate[:, h]
    return out, bound, touched


def select(groups, beams, take, vocab, logits, scores, done, end_id):
    """parents, tokens int32, scores f64, done int32, [groups * take] each."""
    found = []
    for g in range(groups):
        here = []
        for b in range(beams):
            r = g * beams + b
            if not np.isfinite(scores[r]):
                continue
            score = float(scores[r])
            if done is not None and done[r]:
                here.append((-score, r, end_id, 1))
                continue
            x = logits[r].astype(np.float64)
            top = x.max()
            if not np.isfinite(top) or np.isnan(x).any():
                continue
            base = score - (top + np.log(np.exp(x - top).sum()))
            order = np.argsort(-(base + x), kind="stable")[:take]          # the values', which can be equal where the logits are not
            here += [(-(base + x[t]), r, int(t), int(t == end_id)) for t in order if np.isfinite(x[t])]
        here.sort(key=lambda c: c[:3])
        found += (here + [(np.inf, -1, -1, 0)] * take)[:take]
    return (np.array([c[1] for c in found], np.int32), np.array([c[2] for c in found], np.int32),
            np.array([-c[0] for c in found]), np.array([c[3] for c in found], np.int32))

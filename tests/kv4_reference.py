"""The paged 4-bit KV cache in numpy: values, layout, pages and attention, in 64 bits and one step at a time.

What a group of 64 f16 values x is kept as: lo = min x, s = f16(f32((max x - min x) / 15)),
q = clamp(round((x - lo) / s), 0, 15) with ties to even; it stands for lo + s q.
"""
from __future__ import annotations

import numpy as np

TOKENS, HALF, HALF_BYTES, HEAD_BYTES, PAGE = 64, 32, 9216, 18432, 73728
KV, HD = 4, 256


def quantise(x: np.ndarray):
    """f16 [..., 256] -> codes u8 [..., 256], s and lo f16 [..., 4]."""
    v = x.astype(np.float16).astype(np.float64).reshape(*x.shape[:-1], 4, 64)
    fine = np.isfinite(v).all(-1)
    v = np.where(fine[..., None], v, 0.0)
    lo, hi = v.min(-1), v.max(-1)
    s = ((hi - lo) / 15).astype(np.float32).astype(np.float16)
    sd = s.astype(np.float64)[..., None]
    q = np.where(sd > 0, np.clip(np.rint((v - lo[..., None]) / np.where(sd > 0, sd, 1)), 0, 15), 0).astype(np.uint8)
    nan = np.float16(np.nan)
    return q.reshape(x.shape), np.where(fine, s, nan), np.where(fine, lo.astype(np.float16), nan)


def value(q, s, lo):
    """What codes stand for, f64."""
    g = q.reshape(*q.shape[:-1], 4, 64).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (lo.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * g).reshape(q.shape)


def nibble(e):
    return e // 2 + 4 * (e % 2)


# byte and shift of every code of a half page, f16 index of every scale and minimum
_t, _d = np.meshgrid(np.arange(HALF), np.arange(HD), indexing="ij")
_kw = ((_t // 16) * 2 + _d // 128) * 256 + (_d // 8 % 4) * 64 + (_t % 16) * 4 + _d // 32 % 4
_kn = nibble(_d % 8)
_vw = 1024 + (_d // 64) * 256 + (_t // 4 % 4) * 64 + (_d % 16) * 4 + _d // 16 % 4
_vn = nibble(4 * (_t // 16) + _t % 4)
CODE_BYTE = {0: _kw * 4 + _kn // 2, 1: _vw * 4 + _vn // 2}
CODE_SHIFT = {0: _kn % 2 * 4, 1: _vn % 2 * 4}
_tt, _g = np.meshgrid(np.arange(HALF), np.arange(4), indexing="ij")
S_AT = (_tt // 4 % 4) * 32 + (_tt // 16) * 16 + (_tt % 4) * 4 + _g
LO_AT = _g * 32 + (_tt // 4 % 4) * 8 + (_tt // 16) * 4 + _tt % 4


def _half(page, head, t):
    at = head * HEAD_BYTES + t // HALF * HALF_BYTES
    return page[at:at + HALF_BYTES]


def put(page: np.ndarray, head: int, t: int, x: np.ndarray, is_v: int):
    """Token t (0 .. 63) of a page (u8 [73728]) takes the f16 row x [256]."""
    h, i = _half(page, head, t), t % HALF
    q, s, lo = quantise(x)
    byte, shift = CODE_BYTE[is_v][i], CODE_SHIFT[is_v][i]
    for b, sh, c in zip(byte, shift, q):
        h[b] = (int(h[b]) & ~(15 << int(sh)) & 255) | (int(c) << int(sh))
    meta = h[8192:].view(np.float16)
    meta[256 * is_v + S_AT[i]] = s
    meta[256 * is_v + 128 + LO_AT[i]] = lo


def get(page: np.ndarray, head: int, is_v: int) -> np.ndarray:
    """f64 [64, 256]: what a page's tokens stand for."""
    out = []
    for half in range(2):
        h = _half(page, head, half * HALF)
        q = (h[CODE_BYTE[is_v]] >> CODE_SHIFT[is_v].astype(np.uint8)) & 15
        meta = h[8192:].view(np.float16)
        out.append(value(q, meta[256 * is_v + S_AT], meta[256 * is_v + 128 + LO_AT]))
    return np.concatenate(out)


def pages_of(n: int) -> int:
    return -(-n // TOKENS)


class Cache:
    """pages u8 [layers, num_pages, PAGE], table [rows, max_pages], lens [rows], refs [num_pages]."""

    def __init__(self, layers, num_pages, rows, max_pages, seed=0, fill=True):
        rng = np.random.default_rng(seed)
        self.pages = (rng.integers(0, 256, (layers, num_pages, PAGE), dtype=np.uint8) if fill
                      else np.zeros((layers, num_pages, PAGE), np.uint8))
        self.table = np.full((rows, max_pages), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.refs = np.zeros(num_pages, np.int32)

    def ids(self, r):
        return self.table[r, :pages_of(int(self.lens[r]))]

    def consistent(self):
        want = np.zeros_like(self.refs)
        for r in range(len(self.lens)):
            np.add.at(want, self.ids(r), 1)
        return np.array_equal(want, self.refs)

    def resize(self, rows, lens, add=False):
        most = self.table.shape[1] * TOKENS
        rows = list(range(len(lens))) if rows is None else [int(r) for r in rows]
        if any(not 0 <= r < len(self.lens) for r in rows) or len(set(rows)) < len(rows):
            return -1
        lens = [int(n) + (int(self.lens[r]) if add else 0) for r, n in zip(rows, lens)]
        if any(not 0 <= n <= most for n in lens):
            return -1
        old = [int(self.lens[r]) for r in rows]
        partial = [int(self.table[r, o // TOKENS]) if n > o and o % TOKENS else None for r, n, o in zip(rows, lens, old)]
        copies, kept = [], set()
        for i, p in enumerate(partial):
            if p is None:
                continue
            if partial.count(p) == self.refs[p] and p not in kept:
                kept.add(p)
                continue
            copies.append(i)
        free = [int(p) for p in np.flatnonzero(self.refs == 0)]
        need = sum(max(0, pages_of(n) - pages_of(o)) + (i in copies) for i, (n, o) in enumerate(zip(lens, old)))
        if need > len(free):
            return need - len(free)
        drop, fresh = [], []
        for i, (r, n, o) in enumerate(zip(rows, lens, old)):
            if i in copies:
                p, at = free.pop(0), o // TOKENS
                self.pages[:, p] = self.pages[:, partial[i]]
                drop.append(partial[i])
                self.table[r, at] = p
                fresh.append(p)
            for at in range(pages_of(o), pages_of(n)):
                self.table[r, at] = free.pop(0)
                fresh.append(int(self.table[r, at]))
            drop += [int(self.table[r, at]) for at in range(pages_of(n), pages_of(o))]
            self.lens[r] = n
        np.subtract.at(self.refs, np.asarray(drop, int), 1)
        self.refs[np.asarray(fresh, int)] = 1
        return 0

    def fork(self, src, dst):
        n = len(self.lens)
        if any(not 0 <= r < n for r in list(src) + list(dst)) or len(set(dst)) < len(dst):
            return -1
        was = [(self.ids(s).copy(), int(self.lens[s])) for s in src]
        for (ids, length), d in zip(was, dst):
            np.add.at(self.refs, ids, 1)
            np.subtract.at(self.refs, self.ids(d).copy(), 1)
            self.table[d, :len(ids)] = ids
            self.lens[d] = length
        return 0

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = {m: h for m, h in zip(movers, holes)}
        for m, h in to.items():
            self.pages[:, h] = self.pages[:, m]
            self.refs[h], self.refs[m] = self.refs[m], 0
        for r in range(len(self.lens)):
            for j in range(pages_of(int(self.lens[r]))):
                self.table[r, j] = to.get(int(self.table[r, j]), self.table[r, j])
        return live

    def is_page(self, p):
        return 0 <= p < len(self.refs)

    def store(self, layer, row, batch, first, n, k, v):
        """k, v f16 values [batch, 4, >= n, 256]."""
        for b in range(batch):
            f = 0 if first is None else int(first[b])
            if f < 0:
                continue
            for i in range(n):
                t = f + i
                if t >= self.lens[row + b] or not self.is_page(self.table[row + b, t // TOKENS]):
                    continue
                if self.refs[self.table[row + b, t // TOKENS]] > 1:
                    continue
                page = self.pages[layer, self.table[row + b, t // TOKENS]]
                for head in range(KV):
                    put(page, head, t % TOKENS, k[b, head, i], 0)
                    put(page, head, t % TOKENS, v[b, head, i], 1)

    def rows64(self, layer, r, head, is_v):
        """f64 [len, 256] of a row; pages that are none of the pool: None in the mask returned beside it."""
        n = int(self.lens[r])
        out, there = np.zeros((pages_of(n) * TOKENS, HD)), np.zeros(pages_of(n) * TOKENS, bool)
        for j in range(pages_of(n)):
            if self.is_page(self.table[r, j]):
                out[j * TOKENS:(j + 1) * TOKENS] = get(self.pages[layer, self.table[r, j]], head, is_v)
                there[j * TOKENS:(j + 1) * TOKENS] = True
        return out[:n], there[:n]

    def decode(self, layer, slots, batch, q_gate, k_new, v_new, q_norm, k_norm, cos, sin, max_len):
        """One step; q_norm, k_norm f16 values.  Appends to the pages; f64 [batch, 16, 256]."""
        out = np.zeros((batch, 16, HD))
        seen = set()
        for b in range(batch):
            r = b if slots is None else int(slots[b])
            if not 0 <= r < len(self.lens):
                continue
            n = int(self.lens[r])
            if r in seen or n > max_len:
                out[b] = np.nan
                continue
            seen.add(r)
            if n <= 0:
                continue
            pos = n - 1
            if self.is_page(self.table[r, pos // TOKENS]) and self.refs[self.table[r, pos // TOKENS]] > 1:
                out[b] = np.nan
                continue
            if self.is_page(self.table[r, pos // TOKENS]):
                page = self.pages[layer, self.table[r, pos // TOKENS]]
                k = _turn(k_new[b], k_norm, cos[pos], sin[pos]).astype(np.float32).astype(np.float16)
                with np.errstate(over="ignore"):
                    vh = v_new[b].astype(np.float16)
                for head in range(KV):
                    put(page, head, pos % TOKENS, k[head], 0)
                    put(page, head, pos % TOKENS, vh[head], 1)
            q = _turn(q_gate[b, :, :HD], q_norm, cos[pos], sin[pos])
            for head in range(KV):
                K, there = self.rows64(layer, r, head, 0)
                V, _ = self.rows64(layer, r, head, 1)
                if not there.any():
                    continue
                K, V = K[there], V[there]
                s = q[4 * head:4 * head + 4] @ K.T / 16
                p = np.exp(s - s.max(-1, keepdims=True))
                out[b, 4 * head:4 * head + 4] = p @ V / p.sum(-1, keepdims=True)
            out[b] /= 1 + np.exp(-q_gate[b, :, HD:].astype(np.float64))
        return out


def _turn(x, gamma, cos, sin):
    """Per-head RMSNorm (1 + gamma) and RoPE of rows [..., 256] at one position, f64."""
    x, cos, sin = x.astype(np.float64), cos.astype(np.float64), sin.astype(np.float64)
    with np.errstate(invalid="ignore"):
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * (1 + gamma.astype(np.float64))
    y = x.copy()
    y[..., :32] = x[..., :32] * cos - x[..., 32:64] * sin
    y[..., 32:64] = x[..., 32:64] * cos + x[..., :32] * sin
    return y

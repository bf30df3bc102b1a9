"""Timed cases of the paged 4-bit KV cache: attention over it, writing and reading it, and its pages.

One layer's page holds 64 tokens of the 4 kv heads' K and V (256 dims each) in 4 bits: per token,
head and group of 64 dims the minimum `lo` and a scale `s` (f16) and 64 codes, the value being
lo + s * code.  A cache is a pool [layers][num_pages][73728 bytes], a table of page ids per row
(sequence), the rows' lengths and a reference count per page.  Kinds (`case["kind"]`):

  store    `tokens` f16 K/V rows of each of `batch` sequences into the pages, and read back
  decode   one attention step of `batch` sequences: append, softmax over the row's tokens, gate
  resize   `rows` sequences take `draft` more tokens and give them back
  fork     `beams` rows go back a token, are forked, and all of them take the next token
  compact  the live pages of a pool move to its front

`own` false: elementary torch operations.  `own` true: the calls of `qora_mixer.Context`.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DEV = "cuda"
F32, F64 = torch.float32, torch.float64
HEADS, KV, HD = 16, 4, 256
TOKENS, HALF, HALF_BYTES, PAGE = 64, 32, 9216, 73728
LAYERS = 8           # attention layers of the 4B model: they share one table
ROPE_ROWS = 32896


# ---- the cases -----------------------------------------------------------------------------
def listed():
    return [
        # a one-line question's cache goes from the prompt's f16 rows to the pages
        {"name": "store_t45", "kind": "store", "batch": 1, "tokens": 45, "first": 0},
        # four long caches move over; they begin inside a page
        {"name": "store_b4_t32701", "kind": "store", "batch": 4, "tokens": 32701, "first": 37},
        # the first token of a sequence
        {"name": "decode_b1_t1", "kind": "decode", "batch": 1, "len": 1, "ragged": False, "shared": 0, "idle": 0},
        # one chat, a few pages of context
        {"name": "decode_b1_t4097", "kind": "decode", "batch": 1, "len": 4097, "ragged": False, "shared": 0, "idle": 0},
        # a serving batch: odd lengths, a common prompt, three rows empty
        {"name": "decode_b19_ragged", "kind": "decode", "batch": 19, "len": 7001, "ragged": True, "shared": 1024, "idle": 3},
        # the benchmark's serving step: 64 sequences at 32K context
        {"name": "decode_b64_t32769", "kind": "decode", "batch": 64, "len": 32769, "ragged": False, "shared": 0, "idle": 0},
        # one chat drafts four tokens and loses them
        {"name": "resize_r1", "kind": "resize", "rows": 1, "pages": 512, "draft": 4},
        # a serving batch does, in a large pool
        {"name": "resize_r64", "kind": "resize", "rows": 64, "pages": 32768, "draft": 5},
        # four beams of a short answer
        {"name": "fork_b4", "kind": "fork", "beams": 4, "len": 300, "shared": 256},
        # a wide search after a long prompt
        {"name": "fork_b32", "kind": "fork", "beams": 32, "len": 2100, "shared": 1920},
        # a small pool, half of it freed
        {"name": "compact_p64", "kind": "compact", "pages": 64, "live": 32},
        # a large pool after many sequences ended
        {"name": "compact_p4096", "kind": "compact", "pages": 4096, "live": 2051},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "decode", "resize", "fork", "compact"])
    if kind == "store":
        return {"kind": kind, "batch": _spread(rng, 1, 4), "tokens": _spread(rng, 1, 32701), "first": rng.randrange(0, 64)}
    if kind == "decode":
        n, batch = _spread(rng, 1, 32769), _spread(rng, 1, 64)
        return {"kind": kind, "batch": batch, "len": n, "ragged": rng.random() < 0.5,
                "shared": n // 2 // TOKENS * TOKENS if rng.random() < 0.3 else 0, "idle": rng.randrange(0, max(1, batch // 4))}
    if kind == "resize":
        rows = _spread(rng, 1, 64)
        return {"kind": kind, "rows": rows, "pages": _spread(rng, 4 * rows, 32768), "draft": rng.randrange(1, 200)}
    if kind == "fork":
        n = _spread(rng, 20, 2100)
        return {"kind": kind, "beams": _spread(rng, 1, 32), "len": n, "shared": n // 2 // TOKENS * TOKENS}
    pages = _spread(rng, 64, 4096)
    return {"kind": kind, "pages": pages, "live": rng.randrange(pages // 4, 3 * pages // 4)}


# ---- the library ---------------------------------------------------------------------------
_made = {}


def _binding():
    if "qora_mixer" not in sys.modules:
        spec = importlib.util.spec_from_file_location("qora_mixer", ROOT / "qora-llm-4b_amd" / "qora_mixer.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules["qora_mixer"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["qora_mixer"]


def _context():
    """One context for the process, on a torch stream, reserved for the largest case."""
    if "ctx" not in _made:
        M = _binding()
        ctx = M.Context(0)
        _made["stream"] = torch.cuda.Stream()
        ctx.stream = _made["stream"].cuda_stream
        ctx.reserve(64, ROPE_ROWS, 0)
        _made["ctx"] = ctx
    return _made["ctx"], _made["stream"]


def _handle(s):
    """The library's description of the state's cache."""
    return _binding().Kv4Cache.of(
        pages=s["pages"].data_ptr(), table=s["table"].data_ptr(), lens=s["lens"].data_ptr(), refs=s["refs"].data_ptr(),
        layers=s["pages"].shape[0], num_pages=s["pages"].shape[1], rows=s["table"].shape[0], max_pages=s["table"].shape[1])


# ---- the format ----------------------------------------------------------------------------
# Half a page of one head: K codes [2 runs of 16 tokens][2][4 quarters g][16 tokens][4 words], V codes
# [4 groups][4 g][16 dims][4 words], then per half page the scales and minima of K and of V.  A word's
# nibble n is element e = 2 (n & 3) + (n >> 2) of eight: dims 32 s + 8 g + e of K (s = 4 * second index
# + word), tokens 16 (e >> 2) + 4 g + (e & 3) of V.  Scales are [g][run][4 tokens][group], minima
# [group][g][run][4 tokens], for token 16 run + 4 g + i.
def _quantise(x):
    """f16 values [..., 256] (any float type) -> codes u8 [..., 256], s and lo f16 [..., 4]."""
    x = x.to(F32).unflatten(-1, (4, 64))
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi.to(F64) - lo.to(F64)) / 15).to(F32).half()
    ratio = (x.to(F64) - lo.to(F64).unsqueeze(-1)) / s.to(F64).unsqueeze(-1)
    q = torch.where(s.unsqueeze(-1) > 0, ratio.round().clamp(0, 15), torch.zeros_like(ratio))
    return q.to(torch.uint8).flatten(-2), s, lo.half()


def _value(codes, s, lo):
    """f32 [..., 256]: lo + s * code."""
    v = s.to(F32).unsqueeze(-1) * codes.unflatten(-1, (4, 64)).to(F32)
    return v.add_(lo.to(F32).unsqueeze(-1)).flatten(-2)


_K_VIEW, _K_ORDER = (2, 2, 4, 16, 4, 2, 4), (0, 3, 1, 4, 2, 6, 5)           # run half g token word n>>2 n&3
_V_VIEW, _V_ORDER = (4, 4, 16, 4, 2, 2, 2), (5, 1, 6, 4, 0, 3, 2)           # group g dim word n2 n1 n0


def _permuted(t, view, order):
    lead = t.dim() - 1
    return t.unflatten(-1, view).permute(*range(lead), *(lead + i for i in order))


def _inverse(order):
    back = [0] * len(order)
    for i, o in enumerate(order):
        back[o] = i
    return back


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _split(t):
    """Half pages u8 [..., 9216] -> (codes u8 [..., 32, 256], s, lo f16 [..., 32, 4]) of K and of V."""
    lead = t.shape[:-1]
    kc = _permuted(_nibbles(t[..., :4096]), _K_VIEW, _K_ORDER).reshape(*lead, HALF, HD)
    vc = _permuted(_nibbles(t[..., 4096:8192]), _V_VIEW, _V_ORDER).reshape(*lead, HALF, HD)
    meta = t[..., 8192:].contiguous().view(torch.float16).unflatten(-1, (4, 128))
    s = [_permuted(meta[..., i, :], (4, 2, 4, 4), (1, 0, 2, 3)).reshape(*lead, HALF, 4) for i in (0, 2)]
    lo = [_permuted(meta[..., i, :], (4, 4, 2, 4), (2, 1, 3, 0)).reshape(*lead, HALF, 4) for i in (1, 3)]
    return (kc, s[0], lo[0]), (vc, s[1], lo[1])


def _join(k, v):
    """The inverse of _split."""
    lead = k[0].shape[:-2]

    def packed(codes, view, order):
        shape = [view[o] for o in order]
        n = codes.reshape(*lead, *shape).permute(*range(len(lead)), *(len(lead) + i for i in _inverse(order)))
        n = n.reshape(*lead, 4096, 2)
        return n[..., 0] | (n[..., 1] << 4)

    def halves(x, shape, order):
        n = x.reshape(*lead, *shape).permute(*range(len(lead)), *(len(lead) + i for i in order))
        return n.reshape(*lead, 128).contiguous().view(torch.uint8)

    parts = [packed(k[0], _K_VIEW, _K_ORDER), packed(v[0], _V_VIEW, _V_ORDER)]
    for _, s, lo in (k, v):
        parts.append(halves(s, (2, 4, 4, 4), (1, 0, 2, 3)))
        parts.append(halves(lo, (2, 4, 4, 4), (3, 1, 0, 2)))
    return torch.cat(parts, -1)


def _halves_of(pages):
    """[layers, pages, 73728] -> [layers, pages, 4 heads, 2, 9216], the same memory."""
    return pages.view(*pages.shape[:2], KV, 2, HALF_BYTES)


# ---- inputs --------------------------------------------------------------------------------
class _Gen:
    """Seeded device tensors; every draw is another part of the same stream of numbers."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, shape, std=1.0, dtype=F32):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=dtype).mul_(std)

    def ints(self, shape, lo, hi):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=torch.int32)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV).to(torch.int32)

    def kv(self, *lead):
        """Normed K rows (channels of unequal size) and V rows, f16."""
        k = self.normal((*lead, HD)) * (1 + 0.5 * self.normal((HD,)).abs())
        return k.half(), self.normal((*lead, HD), 0.7).half()

    def pool(self, layers, count):
        """Pages as they stand in a used pool: random ones of 96 written in earnest."""
        some = []
        for _ in range(3):
            k, v = self.kv(32, KV, 2, HALF)
            some.append(_join(_quantise(k), _quantise(v)).reshape(32, PAGE))
        at = torch.randint(0, 96, (layers * count,), generator=self.g, device=DEV)
        return torch.cat(some)[at].view(layers, count, PAGE)


def _rope(rows):
    freq = 1.0 / 10_000_000.0 ** (torch.arange(32, device=DEV, dtype=F64) / 32)
    angle = torch.arange(rows, device=DEV, dtype=F64).unsqueeze(1) * freq
    return angle.cos().float(), angle.sin().float()


def _cdiv(a, b):
    return -(-a // b)


def _table(g, pages_of, num_pages, max_pages, prefix=0, keep=0):
    """Scattered pages for rows of pages_of (a list) pages, the first `prefix` the same in every row that has them,
    but the last `keep` pages of a row its own."""
    ids = g.perm(num_pages)
    table = torch.full((len(pages_of), max_pages), -1, device=DEV, dtype=torch.int32)
    at = prefix
    for i, n in enumerate(pages_of):
        p = max(0, min(prefix, n - keep))
        table[i, :p] = ids[:p]
        table[i, p:n] = ids[at:at + n - p]
        at += n - p
    refs = torch.zeros(num_pages, device=DEV, dtype=torch.int32)
    used = table[table >= 0].long()
    return table, refs.scatter_add_(0, used, torch.ones_like(used, dtype=torch.int32))


def _ints(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _inputs(case, seed):
    g, kind = _Gen(seed), case["kind"]
    pick = torch.Generator().manual_seed(int(seed))          # lengths: the host plans with them too

    def lengths(count, lo, hi):
        return torch.randint(lo, hi, (count,), generator=pick).tolist()

    if kind == "store":
        b, n, first = case["batch"], case["tokens"], case["first"]
        lens = [first + n] * b
        pages = _cdiv(first + n, TOKENS)
        table, refs = _table(g, [pages] * b, b * pages + 3, pages)
        k, v = g.kv(b, KV, n)
        return {"pages": g.pool(1, b * pages + 3), "table": table, "refs": refs, "lens": _ints(lens),
                "k": k, "v": v, "first": _ints([first] * b)}
    if kind == "decode":
        b, n = case["batch"], case["len"]
        lens = lengths(b, 1, n + 1) if case["ragged"] else [n] * b
        lens[0] = n
        if case["idle"]:
            lens[-case["idle"]:] = [0] * case["idle"]
        prefix, most = case["shared"] // TOKENS, _cdiv(n, TOKENS)
        count = prefix + sum(max(1, _cdiv(m, TOKENS) - prefix) for m in lens) + 3
        # a row's last page is its own: the step writes there
        table, refs = _table(g, [_cdiv(m, TOKENS) for m in lens], count, most, prefix, keep=1)
        return {"pages": g.pool(1, count), "table": table, "refs": refs, "lens": _ints(lens),
                "q_gate": g.normal((b, HEADS, 2 * HD)), "k_new": g.normal((b, KV, HD)), "v_new": g.normal((b, KV, HD), 0.7),
                "q_norm": g.normal((HD,), 0.1).half(), "k_norm": g.normal((HD,), 0.1).half(),
                "first": _ints([max(0, m - 1) for m in lens])}
    if kind == "resize":
        rows, count, draft = case["rows"], case["pages"], case["draft"]
        most = max(1, (count - rows * _cdiv(draft, TOKENS) - rows) // rows) * TOKENS
        lens = lengths(rows, 1, max(2, most))
        more = lengths(rows, 0, draft + 1)
        more[0] = draft
        max_pages = _cdiv(most + draft, TOKENS) + 1
        table, refs = _table(g, [_cdiv(m, TOKENS) for m in lens], count, max_pages)
        return {"pages": g.pool(1, count), "table": table, "refs": refs, "lens": _ints(lens), "back": _ints(lens),
                "up": _ints([m + d for m, d in zip(lens, more)]), "result": _ints([-7, -7])}
    if kind == "fork":
        beams, n, prefix = case["beams"], case["len"], case["shared"] // TOKENS
        lens = [n - m for m in lengths(beams, 0, max(1, n // 8))]
        count = prefix + 2 * beams * (_cdiv(n, TOKENS) + 2 - prefix) + 5
        held = [_cdiv(m + 1, TOKENS) for m in lens]
        table, refs = _table(g, held + [0] * beams, count, _cdiv(n, TOKENS) + 2, prefix)
        src = g.ints((beams,), 0, beams)
        base = _ints(lens)
        return {"pages": g.pool(LAYERS, count), "table": table, "refs": refs, "lens": torch.cat([base + 1, torch.zeros_like(base)]),
                "base": base, "src": src, "dst": torch.arange(beams, 2 * beams, device=DEV, dtype=torch.int32),
                "next": torch.cat([base, base[src.long()]]) + 1, "result": _ints([-7, -7, -7])}
    count, live = case["pages"], case["live"]
    rows = 16
    each = [live // rows + (i < live % rows) for i in range(rows)]
    table, refs = _table(g, each, count, max(each) + 1)
    lens = _ints([m * TOKENS - (i if m else 0) for i, m in enumerate(each)])
    return {"pages": g.pool(LAYERS, count), "table": table, "refs": refs, "lens": lens, "table0": table.clone(),
            "refs0": refs.clone(), "live": _ints([-7])}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], kind = dict(case), case["kind"]
    if kind == "store":
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    if kind == "decode":
        b = case["batch"]
        s["rope"] = _rope(case["len"])
        s["out"] = torch.empty((b, HEADS, HD), device=DEV)
        s["k_row"], s["v_row"] = (torch.zeros((b, KV, 1, HD), device=DEV, dtype=torch.float16) for _ in range(2))
    if own:
        _context()
        s["handle"] = _handle(s)
    return s


# ---- the plain forms -----------------------------------------------------------------------
def _rms(x, gain):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain


def _rotate(x, cos, sin):
    lo, hi = x[..., :32], x[..., 32:64]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 64:]], -1)


def _write(s, rows, first, k, v):
    """Tokens first[i] .. of table rows `rows` take the f16 rows k, v [b, 4, n, 256]; past the length none."""
    n = k.shape[2]
    lens = s["lens"][rows].long().unsqueeze(1)
    # the half pages that the tokens touch, whole
    tile0 = first.long() // HALF
    tiles = tile0.unsqueeze(1) + torch.arange((n + HALF - 1) // HALF + 1, device=DEV)
    tok = (tiles.unsqueeze(-1) * HALF + torch.arange(HALF, device=DEV)).flatten(1)
    src = tok - first.long().unsqueeze(1)
    valid = (src >= 0) & (src < n) & (tok < lens)
    b_at, t_at = valid.unflatten(1, (-1, HALF)).any(-1).nonzero(as_tuple=True)
    page = s["table"].long()[rows[b_at], tiles[b_at, t_at] // 2]
    half = tiles[b_at, t_at] % 2
    pool = _halves_of(s["pages"])[0]
    old = _split(pool[page, :, half])                                       # [m, 4, 32, ...]
    take = valid.unflatten(1, (-1, HALF))[b_at, t_at].unsqueeze(1).unsqueeze(-1)
    src = src.clamp(0, n - 1).unflatten(1, (-1, HALF))[b_at, t_at]
    new = [_quantise(x[b_at.unsqueeze(1), :, src].transpose(1, 2)) for x in (k, v)]
    pool[page, :, half] = _join(*([torch.where(take, a, o) for a, o in zip(x, y)] for x, y in zip(new, old)))


def _read(s, rows, first, n, into_k, into_v):
    """The inverse: f16 rows, positions past the length left as they were."""
    tok = first.long().unsqueeze(1) + torch.arange(n, device=DEV)
    valid = (tok < s["lens"][rows].long().unsqueeze(1)).unsqueeze(1).unsqueeze(-1)
    tile = tok // HALF
    most = s["table"].shape[1]
    tile0 = first.long() // HALF
    tiles = (tile0.unsqueeze(1) + torch.arange((n + HALF - 1) // HALF + 1, device=DEV)).clamp(max=2 * most - 1)
    page = s["table"].long()[rows.unsqueeze(1), tiles // 2].clamp(min=0)
    got = _split(_halves_of(s["pages"])[0][page, :, tiles % 2])             # [b, t, 4, 32, ...]
    at = ((tile - tile0.unsqueeze(1)) * HALF + tok % HALF).unsqueeze(1).unsqueeze(-1)
    for (codes, sc, lo), into in zip(got, (into_k, into_v)):
        flat = _value(codes, sc, lo).half().transpose(1, 2).flatten(2, 3)
        into.copy_(torch.where(valid, flat.gather(2, at.expand(-1, KV, -1, HD)), into))


def _attend(s):
    b, rows = s["case"]["batch"], torch.arange(s["case"]["batch"], device=DEV)
    lens = s["lens"].long()
    pos = (lens - 1).clamp(min=0)
    cos, sin = (r[pos].unsqueeze(1) for r in s["rope"])
    q = _rotate(_rms(s["q_gate"][..., :HD], 1 + s["q_norm"].to(F32)), cos, sin)
    k = _rotate(_rms(s["k_new"].to(F64), 1 + s["k_norm"].to(F64)), cos.to(F64), sin.to(F64))
    _write(s, rows, pos, k.to(F32).half().unsqueeze(2), s["v_new"].half().unsqueeze(2))
    page = s["table"].long().clamp(min=0)
    got = _split(_halves_of(s["pages"])[0][page].permute(0, 2, 1, 3, 4).flatten(2, 3))   # [b, 4, halves, 32, ...]
    keys = _value(*got[0]).flatten(2, 3)
    seen = (torch.arange(keys.shape[2], device=DEV) < lens.unsqueeze(1)).view(b, 1, 1, -1)
    score = torch.matmul(q.view(b, KV, 4, HD), keys.transpose(-1, -2)) / 16
    del keys
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros_like(score))
    values = torch.where(seen.transpose(-1, -2), _value(*got[1]).flatten(2, 3), torch.zeros((), device=DEV))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    out = y.view(b, HEADS, HD) * torch.sigmoid(s["q_gate"][..., HD:])
    _read(s, rows, pos, 1, s["k_row"], s["v_row"])
    return {"out": out, "k_row": s["k_row"], "v_row": s["v_row"]}


def _resize(s, rows, new, result, at):
    """Rows (all different) take the lengths `new`; result[at]: 0, or how many pages are lacking."""
    table, refs, lens = s["table"], s["refs"], s["lens"]
    rows, new, old = rows.long(), new.long(), lens[rows].long()
    had, want = (old + TOKENS - 1) // TOKENS, (new + TOKENS - 1) // TOKENS
    last = table.long()[rows, (old // TOKENS).clamp(max=table.shape[1] - 1)]
    partial = (new > old) & (old % TOKENS != 0)
    # a partly filled last page that others hold is copied; if every holder grows, the first of them keeps it
    same = (last.unsqueeze(1) == last.unsqueeze(0)) & partial.unsqueeze(1) & partial.unsqueeze(0)
    first = ~torch.tril(same, -1).any(1)
    held = refs.long()[last.clamp(min=0)]
    copy = partial & ~((same.sum(1) == held) & first)
    need = torch.where(new > old, want - had + copy.long(), torch.zeros_like(new))
    free = refs == 0
    ok = need.sum() <= free.sum()
    result[at] = torch.where(ok, torch.zeros_like(ok, dtype=torch.int32), (need.sum() - free.sum()).int())
    order = torch.argsort((~free).to(torch.uint8), stable=True)              # free ids first, ascending
    begin = torch.where(copy, old // TOKENS, had)
    slot = torch.arange(table.shape[1], device=DEV).unsqueeze(0)
    fresh = ok & (new > old).unsqueeze(1) & (slot >= begin.unsqueeze(1)) & (slot < want.unsqueeze(1))
    number = (need.cumsum(0) - need - begin).unsqueeze(1) + slot
    page = order[number.clamp(0, order.numel() - 1)]
    gone = ok & (slot >= want.unsqueeze(1)) & (slot < had.unsqueeze(1))
    was = table[rows]
    # contents of the copied pages
    at_copy = (copy & ok).nonzero().squeeze(1)
    s["pages"][:, page[at_copy, begin[at_copy]]] = s["pages"][:, last[at_copy]]
    table[rows] = torch.where(fresh, page.int(), was)
    drop = torch.where(gone, was, -1).flatten().long()
    drop = torch.cat([drop, torch.where(copy & ok, last, -1)])
    refs.scatter_add_(0, drop.clamp(min=0), -(drop >= 0).int())
    add = torch.where(fresh, page, -1).flatten()
    refs.scatter_add_(0, add.clamp(min=0), (add >= 0).int())
    lens[rows] = torch.where(ok, new, old).int()


def _fork(s, src, dst, result, at):
    table, refs, lens = s["table"], s["refs"], s["lens"]
    src, dst = src.long(), dst.long()
    slot = torch.arange(table.shape[1], device=DEV).unsqueeze(0)
    had = (lens[dst].long() + TOKENS - 1) // TOKENS
    want = (lens[src].long() + TOKENS - 1) // TOKENS
    old, new, length = table[dst], table[src], lens[src]
    for keep, ids, sign in ((slot < want.unsqueeze(1), new, 1), (slot < had.unsqueeze(1), old, -1)):
        ids = torch.where(keep, ids, -1).flatten().long()
        refs.scatter_add_(0, ids.clamp(min=0), sign * (ids >= 0).int())
    table[dst] = torch.where(slot < want.unsqueeze(1), new, old)
    lens[dst] = length
    result[at] = 0


def _compact(s):
    table, refs, pages = s["table"], s["refs"], s["pages"]
    used = refs > 0
    live = used.sum()
    ids = torch.arange(refs.numel(), device=DEV)
    holes = ids[~used & (ids < live)]
    movers = ids[used & (ids >= live)]
    pages[:, holes] = pages[:, movers]
    to = ids.clone()
    to[movers] = holes
    held = torch.arange(table.shape[1], device=DEV) < ((s["lens"] + TOKENS - 1) // TOKENS).unsqueeze(1)
    table.copy_(torch.where(held, to[table.long().clamp(min=0)].int(), table))
    refs[holes] = refs[movers]
    refs[movers] = 0
    s["live"][0] = live


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "store":
        rows = torch.arange(case["batch"], device=DEV)
        _write(s, rows, s["first"], s["k"], s["v"])
        _read(s, rows, s["first"], case["tokens"], s["k_back"], s["v_back"])
        return {"k": s["k_back"], "v": s["v_back"]}
    if kind == "decode":
        return _attend(s)
    if kind == "resize":
        rows = torch.arange(case["rows"], device=DEV)
        _resize(s, rows, s["up"], s["result"], 0)
        _resize(s, rows, s["back"], s["result"], 1)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "result": s["result"]}
    if kind == "fork":
        beams = case["beams"]
        _resize(s, torch.arange(beams, device=DEV), s["base"], s["result"], 0)
        _fork(s, s["src"], s["dst"], s["result"], 1)
        _resize(s, torch.arange(2 * beams, device=DEV), s["next"], s["result"], 2)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "result": s["result"],
                "pages": s["pages"].view(torch.int32)}
    # a pool as it was before it was compacted: the moved pages still stand where they were
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    _compact(s)
    return {"table": s["table"], "refs": s["refs"], "live": s["live"], "pages": s["pages"].view(torch.int32)}


# ---- the framework's calls -----------------------------------------------------------------
def _p(t):
    return t.data_ptr()


def _library(s):
    ctx, stream = _context()
    case, kind, h = s["case"], s["case"]["kind"], s["handle"]
    if kind == "store":
        b, n = case["batch"], case["tokens"]
        ctx.kv4_store(h, 0, 0, b, _p(s["first"]), n, _p(s["k"]), _p(s["v"]), n)
        ctx.kv4_load(h, 0, 0, b, _p(s["first"]), n, _p(s["k_back"]), _p(s["v_back"]), n)
        return {"k": s["k_back"], "v": s["v_back"]}
    if kind == "decode":
        b, n = case["batch"], case["len"]
        ctx.gqa_decode_kv4(h, 0, b, None, _p(s["q_gate"]), _p(s["k_new"]), _p(s["v_new"]), _p(s["q_norm"]), _p(s["k_norm"]),
                           _p(s["rope"][0]), _p(s["rope"][1]), n, n, None, _p(s["out"]))
        ctx.kv4_load(h, 0, 0, b, _p(s["first"]), 1, _p(s["k_row"]), _p(s["v_row"]), 1)
        return {"out": s["out"], "k_row": s["k_row"], "v_row": s["v_row"]}
    if kind == "resize":
        ctx.kv4_resize(h, case["rows"], None, _p(s["up"]), _p(s["result"]))
        ctx.kv4_resize(h, case["rows"], None, _p(s["back"]), _p(s["result"]) + 4)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "result": s["result"]}
    if kind == "fork":
        beams = case["beams"]
        ctx.kv4_resize(h, beams, None, _p(s["base"]), _p(s["result"]))
        ctx.kv4_fork(h, beams, _p(s["src"]), _p(s["dst"]), _p(s["result"]) + 4)
        ctx.kv4_resize(h, 2 * beams, None, _p(s["next"]), _p(s["result"]) + 8)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "result": s["result"],
                "pages": s["pages"].view(torch.int32)}
    with torch.cuda.stream(stream):
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
    ctx.kv4_compact(h, _p(s["live"]))
    return {"table": s["table"], "refs": s["refs"], "live": s["live"], "pages": s["pages"].view(torch.int32)}


def run(state):
    return _library(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------
TOKEN = PAGE // TOKENS                # 1152 bytes
F16_TOKEN = 2 * 2 * KV * HD           # 4096 bytes


def work(case):
    kind = case["kind"]
    if kind == "store":
        n = case["batch"] * case["tokens"]
        return {"bytes": 2 * n * (TOKEN + F16_TOKEN), "flops": n * 2 * KV * HD * 8}
    if kind == "decode":
        b, n = case["batch"] - case["idle"], case["len"]
        keys = b * ((n + 1) / 2 if case["ragged"] else n)
        shared = min(case["shared"], n) * (b - 1) * (0.5 if case["ragged"] else 1.0)   # read once, roughly
        return {"bytes": max(b, keys - shared) * TOKEN + b * 4 * (HEADS * 3 * HD + 2 * KV * HD), "flops": keys * HEADS * HD * 4}
    if kind == "resize":
        # two calls: counts of the pages, lengths and entries of the rows
        return {"bytes": 2 * (4 * case["pages"] + case["rows"] * 24), "flops": 0}
    if kind == "fork":
        beams, pages = case["beams"], _cdiv(case["len"], TOKENS)
        # the table rows, and a copy of the last page per row but one of each beam
        return {"bytes": beams * pages * 20 + 2 * beams * PAGE * LAYERS, "flops": 0}
    count, live = case["pages"], case["live"]
    return {"bytes": 2 * live * (1 - live / count) * PAGE * LAYERS + 8 * count, "flops": 0}


# ---- the same in 64 bits, from the format's formulas ---------------------------------------
def _code_at(half, t, d, is_v):
    """Byte offset in a page and shift of the code of token t (0 .. 63), dim d; head 0."""
    u, c = t % 32 // 16, t % 16
    if is_v:
        g, e = c // 4, 4 * u + c % 4
        word = (d // 64 * 64 + g * 16 + d % 16) * 4 + d % 64 // 16
        base = 4096
    else:
        g, e = d % 32 // 8, d % 8
        word = ((u * 2 + d // 128) * 64 + g * 16 + c) * 4 + d % 128 // 32
        base = 0
    n = e // 2 + 4 * (e % 2)
    return half * HALF_BYTES + base + word * 4 + n // 2, n % 2 * 4


def _meta_at(half, t, group, which):
    """Byte offset of the scale (which 0 / 2) or minimum (1 / 3) of token t."""
    u, g, i = t % 32 // 16, t % 16 // 4, t % 4
    at = ((g * 2 + u) * 4 + i) * 4 + group if which % 2 == 0 else ((group * 4 + g) * 2 + u) * 4 + i
    return half * HALF_BYTES + 8192 + which * 256 + at * 2


def _rows64(pages, ids, n):
    """K and V f64 [4, n, 256] of the first n tokens of the pages `ids`."""
    t = torch.arange(TOKENS, device=DEV).view(-1, 1)
    d = torch.arange(HD, device=DEV).view(1, -1)
    head = torch.arange(KV, device=DEV).view(-1, 1, 1) * 2 * HALF_BYTES
    found = []
    raw = pages[ids]
    for is_v in (False, True):
        at, shift = _code_at(t // HALF, t, d, is_v)
        q = (raw[:, head + at].to(torch.int32) >> shift) & 15
        s, lo = (raw[:, head + _meta_at(t // HALF, t, torch.arange(4, device=DEV).view(1, -1), 2 * is_v + w)].to(torch.int32) |
                 raw[:, head + _meta_at(t // HALF, t, torch.arange(4, device=DEV).view(1, -1), 2 * is_v + w) + 1].to(torch.int32) << 8
                 for w in (0, 1))
        s, lo = (x.to(torch.int16).view(torch.float16).to(F64).repeat_interleave(64, -1) for x in (s, lo))
        found.append((lo + s * q).transpose(0, 1).reshape(KV, -1, HD)[:, :n])
    return found


def _stand_for(x):
    """What f64 rows [..., 256] (f16 values) read back as."""
    groups = []
    for i in range(4):
        y = x[..., 64 * i:64 * i + 64]
        lo = y.min(-1, keepdim=True).values
        s = ((y.max(-1, keepdim=True).values - lo) / 15).to(F32).to(torch.float16).to(F64)
        steps = torch.clamp(torch.round((y - lo) / torch.where(s == 0, torch.ones_like(s), s)), 0, 15)
        groups.append(lo + s * torch.where(s == 0, torch.zeros_like(steps), steps))
    return torch.cat(groups, -1)


def exact(case, seed):
    kind = case["kind"]
    if kind not in ("store", "decode"):
        return None                                                          # whole numbers and copies
    s = _inputs(case, seed)
    if kind == "store":
        return {"k": _stand_for(s["k"].to(F64)), "v": _stand_for(s["v"].to(F64))}
    lens = s["lens"].tolist()
    out = torch.zeros((case["batch"], HEADS, HD), device=DEV, dtype=F64)
    k_row, v_row = (torch.zeros((case["batch"], KV, 1, HD), device=DEV, dtype=F64) for _ in range(2))
    cos, sin = (r.to(F64) for r in _rope(case["len"]))

    def turned(x, gain, at):
        x = x.to(F64)
        x = x / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + 1e-6) * (1 + gain.to(F64))
        y = x.clone()
        y[..., :32] = x[..., :32] * cos[at] - x[..., 32:64] * sin[at]
        y[..., 32:64] = x[..., 32:64] * cos[at] + x[..., :32] * sin[at]
        return y

    for i, n in enumerate(lens):
        if not n:
            continue
        K, V = _rows64(s["pages"][0], s["table"][i, :_cdiv(n, TOKENS)].long(), n)
        K[:, n - 1] = _stand_for(turned(s["k_new"][i], s["k_norm"], n - 1).to(F32).to(torch.float16).to(F64))
        V[:, n - 1] = _stand_for(s["v_new"][i].to(torch.float16).to(F64))
        q = turned(s["q_gate"][i, :, :HD], s["q_norm"], n - 1).view(KV, 4, HD)
        p = torch.softmax(torch.bmm(q, K.transpose(1, 2).contiguous()) / 16, -1)
        out[i] = torch.bmm(p, V).view(HEADS, HD) * torch.sigmoid(s["q_gate"][i, :, HD:].to(F64))
        k_row[i, :, 0], v_row[i, :, 0] = K[:, n - 1], V[:, n - 1]
    return {"out": out, "k_row": k_row, "v_row": v_row}

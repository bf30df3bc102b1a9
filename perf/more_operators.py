"""Timed cases of chunks of new tokens over the paged 4-bit KV cache, and of beam search's step.

A cache is a pool [layers][num_pages][73728 bytes], a table of page ids per row (sequence), the rows'
lengths and a reference count per page; a page holds 64 tokens of the 4 kv heads' K and V (256 dims
each) in 4 bits: per token, head and group of 64 dims the minimum `lo` and a scale `s` (f16) and 64
codes, the value being lo + s * code.  A batch row's new tokens are rows begins[b] .. begins[b + 1]
of packed tensors, and the last ones of the length that its cache row has been grown to.  Kinds
(`case["kind"]`):

  append  the new tokens' K (RMSNorm, RoPE) and V into the pages, and read back
  chunk   attention of the new tokens over their row's pages up to their own position, and the gate
  beam    the best `take` continuations of each request's `beams` sequences by summed log-probability
  states  the recurrent states of sequences become those of their parents, in place

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
VOCAB = 248320                       # the 4B model's
DN_LAYERS, DN_STATE, DN_CONV = 24, 32 * 128 * 128, 8192 * 3      # its recurrent layers; f32 a sequence and layer


# ---- the cases -----------------------------------------------------------------------------
def listed():
    return [
        # one token of one chat, f32 projections
        {"name": "append_t1", "kind": "append", "batch": 1, "new": 1, "len": 300, "ragged": False, "dtype": "f32"},
        # prompts of several requests in one pass, bf16 projections, some behind a prompt that is there already
        {"name": "append_b5_ragged", "kind": "append", "batch": 5, "new": 4099, "len": 6001, "ragged": True, "dtype": "bf16"},
        # one token over a few pages
        {"name": "chunk_t1", "kind": "chunk", "batch": 1, "new": 1, "len": 260, "ragged": False},
        # one chat checks four drafted tokens
        {"name": "chunk_t5_len4101", "kind": "chunk", "batch": 1, "new": 5, "len": 4101, "ragged": False},
        # a serving batch checks up to three drafted tokens a row
        {"name": "chunk_b24_draft", "kind": "chunk", "batch": 24, "new": 4, "len": 12001, "ragged": True},
        # a short prompt, whole
        {"name": "chunk_t700", "kind": "chunk", "batch": 1, "new": 700, "len": 700, "ragged": False},
        # prompts of several requests, some behind a prompt that is there already
        {"name": "chunk_b6_ragged", "kind": "chunk", "batch": 6, "new": 513, "len": 9001, "ragged": True},
        # the last part of a long prompt
        {"name": "chunk_t2048_len32768", "kind": "chunk", "batch": 1, "new": 2048, "len": 32768, "ragged": False},
        # four beams of one answer
        {"name": "beam_w4", "kind": "beam", "groups": 1, "beams": 4, "take": 4, "vocab": VOCAB, "done": 0},
        # eight beams of each of twelve answers, twice as many candidates, some beams at their end
        {"name": "beam_g12_w8", "kind": "beam", "groups": 12, "beams": 8, "take": 16, "vocab": VOCAB, "done": 9},
        # the beams' recurrent states follow: one answer
        {"name": "states_r4", "kind": "states", "rows": 4, "layers": DN_LAYERS},
        # and a wide search
        {"name": "states_r24", "kind": "states", "rows": 24, "layers": DN_LAYERS},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "chunk", "chunk", "chunk", "beam", "states"])
    if kind == "append":
        new, ragged = _spread(rng, 1, 4099), rng.random() < 0.5
        batch = _spread(rng, 1, 5 if ragged else max(1, min(5, 10000 // new)))
        return {"kind": kind, "batch": batch, "new": new, "len": new + _spread(rng, 1, 1902) - 1, "ragged": ragged,
                "dtype": rng.choice(["f32", "bf16"])}
    if kind == "chunk":
        n = _spread(rng, 1, 32768)
        new = _spread(rng, 1, min(n, 2048))
        batch = _spread(rng, 1, max(1, min(24, 2048 * 32768 // (n * new), 24 * 12001 // n)))
        return {"kind": kind, "batch": batch, "new": new, "len": n, "ragged": rng.random() < 0.5}
    if kind == "beam":
        groups, beams = _spread(rng, 1, 12), _spread(rng, 1, 16)
        vocab = VOCAB if rng.random() < 0.4 else _spread(rng, 1000, 262144)
        while groups * beams * vocab > 12 * 8 * VOCAB:
            groups -= 1
        return {"kind": kind, "groups": groups, "beams": beams, "take": rng.choice([beams, 2 * beams, rng.randrange(1, 33)]),
                "vocab": vocab, "done": rng.randrange(0, beams)}
    return {"kind": kind, "rows": _spread(rng, 2, 24), "layers": rng.randrange(1, DN_LAYERS + 1)}


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
    """One context for the process, on a torch stream; its workspace grows with the first calls."""
    if "ctx" not in _made:
        M = _binding()
        ctx = M.Context(0)
        _made["stream"] = torch.cuda.Stream()
        ctx.stream = _made["stream"].cuda_stream
        _made["ctx"] = ctx
    return _made["ctx"]


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
    return sorted(range(len(order)), key=order.__getitem__)


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


def _codes_out(codes, view, order):
    lead = codes.shape[:-2]
    n = codes.reshape(*lead, *(view[o] for o in order))
    n = n.permute(*range(len(lead)), *(len(lead) + i for i in _inverse(order))).reshape(*lead, 4096, 2)
    return n[..., 0] | (n[..., 1] << 4)


def _meta_out(x, shape, order):
    lead = x.shape[:-2]
    n = x.reshape(*lead, *shape).permute(*range(len(lead)), *(len(lead) + i for i in order))
    return n.reshape(*lead, 128).contiguous().view(torch.uint8)


def _join(k, v):
    """The inverse of _split."""
    return torch.cat([_codes_out(k[0], _K_VIEW, _K_ORDER), _codes_out(v[0], _V_VIEW, _V_ORDER),
                      _meta_out(k[1], (2, 4, 4, 4), (1, 0, 2, 3)), _meta_out(k[2], (2, 4, 4, 4), (3, 1, 0, 2)),
                      _meta_out(v[1], (2, 4, 4, 4), (1, 0, 2, 3)), _meta_out(v[2], (2, 4, 4, 4), (3, 1, 0, 2))], -1)


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

    def pool(self, count):
        """One layer's pages as they stand in a used pool: random ones of 96 written in earnest."""
        some = []
        for _ in range(3):
            k = self.normal((32, KV, 2, HALF, HD)) * (1 + 0.5 * self.normal((HD,)).abs())
            v = self.normal((32, KV, 2, HALF, HD), 0.7)
            some.append(_join(_quantise(k.half()), _quantise(v.half())).reshape(32, PAGE))
        at = torch.randint(0, 96, (count,), generator=self.g, device=DEV)
        return torch.cat(some)[at].view(1, count, PAGE)


def _rope(rows):
    freq = 1.0 / 10_000_000.0 ** (torch.arange(32, device=DEV, dtype=F64) / 32)
    angle = torch.arange(rows, device=DEV, dtype=F64).unsqueeze(1) * freq
    return angle.cos().float(), angle.sin().float()


def _cdiv(a, b):
    return -(-a // b)


def _ints(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _sequences(g, case, seed):
    """A cache of batch + 2 rows in scattered pages; the batch rows' slots, lengths and new tokens."""
    b, n, new = case["batch"], case["len"], case["new"]
    pick = torch.Generator().manual_seed(int(seed))          # lengths: the host plans with them too

    def between(lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=pick))

    lens, news = [n] * b, [new] * b
    if case["ragged"]:
        # how many new tokens is the case's own, how much stands before them the seed's
        news = [new] + torch.randint(1, new + 1, (b - 1,), generator=torch.Generator().manual_seed(n + new)).tolist()
        lens = [n] + [between(k, n) for k in news[1:]]
    slots = torch.randperm(b + 2, generator=pick).tolist()[:b]
    row_lens, row_first = [0] * (b + 2), [-1] * (b + 2)
    for r, m, k in zip(slots, lens, news):
        row_lens[r], row_first[r] = m, m - k
    begins = [0]
    for k in news:
        begins.append(begins[-1] + k)
    most = _cdiv(n, TOKENS)
    count = sum(_cdiv(m, TOKENS) for m in row_lens) + 3
    ids, at = g.perm(count), 0
    table = torch.full((b + 2, most), -1, device=DEV, dtype=torch.int32)
    refs = torch.zeros(count, device=DEV, dtype=torch.int32)
    for r, m in enumerate(row_lens):
        held = ids[at:at + _cdiv(m, TOKENS)]
        table[r, :held.numel()] = held
        refs[held.long()] = 1
        at += held.numel()
    return {"pages": g.pool(count), "table": table, "refs": refs, "lens": _ints(row_lens), "first": _ints(row_first),
            "slots": _ints(slots), "begins": _ints(begins), "rope": _rope(n), "total": begins[-1]}


def _inputs(case, seed):
    g, kind = _Gen(seed), case["kind"]
    if kind == "append":
        s = _sequences(g, case, seed)
        t, dtype = s["total"], torch.bfloat16 if case["dtype"] == "bf16" else F32
        s["k"] = (g.normal((t, KV, HD)) * (1 + 0.5 * g.normal((HD,)).abs())).to(dtype)
        s["v"] = g.normal((t, KV, HD), 0.7).to(dtype)
        s["k_norm"] = g.normal((HD,), 0.1).half()
        return s
    if kind == "chunk":
        s = _sequences(g, case, seed)
        s["q_gate"] = g.normal((s["total"], HEADS, 2 * HD)).to(torch.bfloat16)
        s["q_norm"] = g.normal((HD,), 0.1).half()
        return s
    if kind == "beam":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        # the beams of one answer see nearly the same text: like logits, a few tokens far ahead
        like = g.normal((groups, 1, vocab), 2.0) + 12.0 * (torch.rand((groups, 1, vocab), generator=g.g, device=DEV) > 1 - 20 / vocab)
        logits = like + g.normal((groups, beams, vocab), 0.5)
        scores = -g.normal((groups, beams), 3.0).abs() - 5.0
        done = torch.zeros((groups * beams,), device=DEV, dtype=torch.int32)
        done[g.perm(groups * beams)[:case["done"]].long()] = 1
        return {"logits": logits.view(groups * beams, vocab), "scores": scores.view(-1), "done": done, "end": vocab - 3}
    rows, layers = case["rows"], case["layers"]
    return {"state": g.normal((layers, rows, DN_STATE), 0.1), "conv": g.normal((layers, rows, DN_CONV)),
            "src": g.ints((rows,), 0, rows), "dst": torch.arange(rows, device=DEV, dtype=torch.int32), "result": _ints([-7])}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], kind = dict(case), case["kind"]
    if kind == "append":
        rows = s["table"].shape[0]
        s["k_back"], s["v_back"] = (torch.zeros((rows, KV, case["new"], HD), device=DEV, dtype=torch.float16) for _ in range(2))
    if kind == "chunk":
        s["out"] = torch.empty((s["total"], HEADS, HD), device=DEV, dtype=torch.bfloat16)
    if kind == "beam":
        n = case["groups"] * case["take"]
        s["parents"], s["tokens"], s["ended"] = (torch.empty((n,), device=DEV, dtype=torch.int32) for _ in range(3))
        s["best"] = torch.empty((n,), device=DEV)
    if own:
        _context()
        if kind in ("append", "chunk"):
            s["handle"] = _handle(s)
        if kind == "states":
            s["buffers"] = [(s[key][i].data_ptr(), 4 * s[key].shape[2], 4 * s[key].shape[2])
                            for key in ("state", "conv") for i in range(case["layers"])]
    return s


# ---- the plain forms -----------------------------------------------------------------------
def _rms(x, gain):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain


def _rotate(x, cos, sin):
    lo, hi = x[..., :32], x[..., 32:64]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 64:]], -1)


def _places(s):
    """Batch row and position of each packed token."""
    begins, t = s["begins"].long(), torch.arange(s["total"], device=DEV)
    row = torch.searchsorted(begins[1:], t, right=True)
    return row, s["lens"].long()[s["slots"].long()[row]] - begins[row + 1] + t


def _append(s):
    row, pos = _places(s)
    cos, sin = (r[pos].to(F64).unsqueeze(1) for r in s["rope"])
    k = _rotate(_rms(s["k"].to(F64), 1 + s["k_norm"].to(F64)), cos, sin).to(F32).half()
    v = s["v"].half()
    # the half pages that the new tokens touch, whole: tokens tok of batch rows
    begins, slots, lens = s["begins"].long(), s["slots"].long(), s["lens"].long()
    first = lens[slots] - (begins[1:] - begins[:-1])
    tiles = first.unsqueeze(1) // HALF + torch.arange((s["case"]["new"] + HALF - 1) // HALF + 1, device=DEV)
    tok = tiles.unsqueeze(-1) * HALF + torch.arange(HALF, device=DEV)
    valid = (tok >= first.view(-1, 1, 1)) & (tok < lens[slots].view(-1, 1, 1))
    b_at, t_at = valid.any(-1).nonzero(as_tuple=True)
    page, half = s["table"].long()[slots[b_at], tiles[b_at, t_at] // 2], tiles[b_at, t_at] % 2
    pool = _halves_of(s["pages"])[0]
    old = _split(pool[page, :, half])                                       # [m, 4, 32, ...]
    take = valid[b_at, t_at].unsqueeze(1).unsqueeze(-1)
    src = (begins[:-1].view(-1, 1, 1) + tok - first.view(-1, 1, 1)).clamp(0, s["total"] - 1)[b_at, t_at]
    new = [_quantise(x[src].transpose(1, 2)) for x in (k, v)]
    pool[page, :, half] = _join(*([torch.where(take, a, o) for a, o in zip(x, y)] for x, y in zip(new, old)))
    # and the new tokens as they read back, at the cache rows' own places
    got = _split(pool[page, :, half])
    at = (tok - first.view(-1, 1, 1))[b_at, t_at]
    m, e = valid[b_at, t_at].nonzero(as_tuple=True)
    s["k_back"][slots[b_at[m]], :, at[m, e]] = _value(*got[0]).half()[m, :, e]
    s["v_back"][slots[b_at[m]], :, at[m, e]] = _value(*got[1]).half()[m, :, e]
    return {"k": s["k_back"], "v": s["v_back"]}


def _chunk(s):
    row, pos = _places(s)
    cos, sin = (r[pos].unsqueeze(1) for r in s["rope"])
    q = _rotate(_rms(s["q_gate"][..., :HD].to(F32), 1 + s["q_norm"].to(F32)), cos, sin)
    # queries and keys of a batch row side by side, shorter rows filled up
    b, most = s["case"]["batch"], s["case"]["new"]
    at = torch.arange(s["total"], device=DEV) - s["begins"].long()[row]
    dense = torch.zeros((b, most, HEADS, HD), device=DEV)
    dense[row, at] = q
    last = torch.full((b, most), -1, device=DEV)
    last[row, at] = pos
    page = s["table"].long()[s["slots"].long()].clamp(min=0)
    got = _split(_halves_of(s["pages"])[0][page].permute(0, 2, 1, 3, 4).flatten(2, 3))   # [b, 4, halves, 32, ...]
    keys, values = (_value(*x).flatten(2, 3) for x in got)
    seen = (torch.arange(keys.shape[2], device=DEV) <= last.unsqueeze(-1)).view(b, 1, 1, most, -1)
    score = torch.matmul(dense.permute(0, 2, 1, 3).reshape(b, KV, 4 * most, HD), keys.transpose(-1, -2))
    score = score.div_(16).view(b, KV, 4, most, -1).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_().flatten(2, 3)
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    y = y.view(b, HEADS, most, HD).transpose(1, 2)[row, at]
    s["out"].copy_(y * torch.sigmoid(s["q_gate"][..., HD:].to(F32)))
    return {"out": s["out"]}


def _beam(s):
    case = s["case"]
    groups, beams, take, vocab = (case[k] for k in ("groups", "beams", "take", "vocab"))
    x = s["logits"].to(F64)
    top = x.amax(-1, keepdim=True)
    value = s["scores"].to(F64).unsqueeze(1) + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    del x
    ended = s["done"].unsqueeze(1) != 0
    end = torch.arange(vocab, device=DEV) == s["end"]
    value = torch.where(ended, torch.where(end, s["scores"].to(F64).unsqueeze(1), -math.inf), value)
    best, order = torch.sort(value.view(groups, beams * vocab), dim=1, descending=True, stable=True)
    best, order = best[:, :take], order[:, :take]
    there = best > -math.inf
    parent = order // vocab + torch.arange(groups, device=DEV).unsqueeze(1) * beams
    token = order % vocab
    s["parents"].copy_(torch.where(there, parent, -1).flatten())
    s["tokens"].copy_(torch.where(there, token, -1).flatten())
    s["best"].copy_(best.flatten())
    s["ended"].copy_((there & ((s["done"][parent] != 0) | (token == s["end"]))).flatten())
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["best"], "done": s["ended"]}


def _states(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["state"][:, dst] = s["state"][:, src]
    s["conv"][:, dst] = s["conv"][:, src]
    s["result"].zero_()
    return {"state": s["state"], "conv": s["conv"], "result": s["result"]}


_PLAIN = {"append": _append, "chunk": _chunk, "beam": _beam, "states": _states}


# ---- the framework's calls -----------------------------------------------------------------
def _p(t):
    return t.data_ptr()


def _library(s):
    ctx, case, kind = _context(), s["case"], s["case"]["kind"]
    if kind == "append":
        b, n = case["batch"], case["new"]
        ctx.kv4_append(s["handle"], 0, b, _p(s["slots"]), _p(s["begins"]), s["total"], _p(s["k"]), _p(s["v"]), _p(s["k_norm"]),
                       _p(s["rope"][0]), _p(s["rope"][1]), case["len"], case["len"], None,
                       dtype=_binding().QM_BF16 if case["dtype"] == "bf16" else _binding().QM_F32)
        ctx.kv4_load(s["handle"], 0, 0, b + 2, _p(s["first"]), n, _p(s["k_back"]), _p(s["v_back"]), n)
        return {"k": s["k_back"], "v": s["v_back"]}
    if kind == "chunk":
        ctx.gqa_chunk_kv4(s["handle"], 0, case["batch"], _p(s["slots"]), _p(s["begins"]), s["total"], case["new"], _p(s["q_gate"]),
                          _p(s["q_norm"]), _p(s["rope"][0]), _p(s["rope"][1]), case["len"], case["len"], None, _p(s["out"]))
        return {"out": s["out"]}
    if kind == "beam":
        ctx.beam_select(case["groups"], case["beams"], case["take"], case["vocab"], _p(s["logits"]), _p(s["scores"]), _p(s["done"]),
                        s["end"], _p(s["parents"]), _p(s["tokens"]), _p(s["best"]), _p(s["ended"]))
        return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["best"], "done": s["ended"]}
    ctx.state_fork(s["buffers"], case["rows"], case["rows"], _p(s["src"]), _p(s["dst"]), _p(s["result"]))
    return {"state": s["state"], "conv": s["conv"], "result": s["result"]}


def run(state):
    return _library(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------
TOKEN = PAGE // TOKENS                # 1152 bytes


def work(case):
    kind = case["kind"]
    if kind in ("append", "chunk"):
        # a ragged batch: the first row as listed, the others about half of it
        b = 1 + (case["batch"] - 1) * (0.5 if case["ragged"] else 1.0)
        keys = b * case["len"]
        new = 1 + (case["batch"] - 1) * (0.5 if case["ragged"] else 1.0)
        new *= case["new"]
    if kind == "append":
        size = 2 if case["dtype"] == "bf16" else 4
        # projections in, 4-bit rows out and in, f16 rows out
        return {"bytes": new * (2 * KV * HD * (size + 2) + 2 * TOKEN + 256), "flops": new * 2 * KV * HD * 10}
    if kind == "chunk":
        mean = max(1.0, case["len"] * (0.6 if case["ragged"] else 1.0) - case["new"] / 2)
        return {"bytes": keys * TOKEN + new * HEADS * HD * 6, "flops": new * mean * HEADS * HD * 4}
    if kind == "beam":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * n, "flops": 4 * n}
    # rows whose parent is another one: read and written
    rows = case["rows"]
    return {"bytes": 2 * 4 * case["layers"] * (rows - 1) * (DN_STATE + DN_CONV), "flops": 0}


# ---- the same in 64 bits, from the formulas ------------------------------------------------
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


def _rows64(raw, n):
    """K and V f64 [4, n, 256] of the first n tokens of the pages u8 [m, 73728]."""
    t = torch.arange(TOKENS, device=DEV).view(-1, 1)
    d = torch.arange(HD, device=DEV).view(1, -1)
    group = torch.arange(4, device=DEV).view(1, -1)
    head = torch.arange(KV, device=DEV).view(-1, 1, 1) * 2 * HALF_BYTES
    found = []
    for is_v in (False, True):
        at, shift = _code_at(t // HALF, t, d, is_v)
        q = (raw[:, head + at].to(torch.int32) >> shift) & 15
        parts = []
        for w in (0, 1):
            m = head + _meta_at(t // HALF, t, group, 2 * is_v + w)
            bits = raw[:, m].to(torch.int32) | raw[:, m + 1].to(torch.int32) << 8
            parts.append(bits.to(torch.int16).view(torch.float16).to(F64).repeat_interleave(64, -1))
        found.append((parts[1] + parts[0] * q).transpose(0, 1).reshape(KV, -1, HD)[:, :n])
    return found


def _stand_for(x):
    """What f64 rows [..., 256] (f16 values) read back as, f16."""
    groups = []
    for i in range(4):
        y = x[..., 64 * i:64 * i + 64]
        lo = y.min(-1, keepdim=True).values
        s = ((y.max(-1, keepdim=True).values - lo) / 15).to(F32).to(torch.float16).to(F64)
        steps = torch.clamp(torch.round((y - lo) / s), 0, 15)
        groups.append(torch.where(s > 0, lo + s * steps, lo))
    return torch.cat(groups, -1).to(F32).to(torch.float16)


def _turned(x, norm, rope, at):
    """Rows [m, heads, 256] normed and rotated to the positions at [m], f64."""
    x = x.to(F64)
    x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / HD + 1e-6) * (norm.to(F64) + 1)
    cos, sin = (r[at].to(F64).view(-1, 1, 32) for r in rope)
    y = x.clone()
    y[..., :32] = x[..., :32] * cos - x[..., 32:64] * sin
    y[..., 32:64] = x[..., 32:64] * cos + x[..., :32] * sin
    return y


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "states":
        return None                                       # moved, not computed
    if kind == "beam":
        groups, beams, take, vocab = (case[k] for k in ("groups", "beams", "take", "vocab"))
        found = {"parents": [], "tokens": [], "scores": [], "done": []}
        for i in range(groups):
            here = []
            for r in range(i * beams, (i + 1) * beams):
                score, x = float(s["scores"][r]), s["logits"][r].to(F64)
                if int(s["done"][r]):
                    here.append((-score, r, s["end"], 1))
                else:
                    least = x.topk(min(take, vocab)).values[-1]
                    ids = (x >= least).nonzero().squeeze(1)
                    for v, t in zip((score + x[ids] - torch.logsumexp(x, 0)).tolist(), ids.tolist()):
                        here.append((-v, r, t, int(t == s["end"])))
            here = (sorted(here) + [(math.inf, -1, -1, 0)] * take)[:take]
            for key, j in (("parents", 1), ("tokens", 2), ("done", 3)):
                found[key] += [h[j] for h in here]
            found["scores"] += [-h[0] for h in here]
        return {key: torch.tensor(v, device=DEV, dtype=F64 if key == "scores" else torch.int32) for key, v in found.items()}
    slots, begins, lens = s["slots"].tolist(), s["begins"].tolist(), s["lens"].tolist()
    if kind == "append":
        k, v = (torch.zeros((len(lens), KV, case["new"], HD), device=DEV, dtype=F64) for _ in range(2))
    else:
        out = torch.zeros((s["total"], HEADS, HD), device=DEV, dtype=F64)
    for b, r in enumerate(slots):
        lo, hi, n = begins[b], begins[b + 1], lens[r]
        at = torch.arange(n - (hi - lo), n, device=DEV)
        if kind == "append":
            kept = _turned(s["k"][lo:hi], s["k_norm"], s["rope"], at).to(F32).to(torch.float16).to(F64)
            k[r, :, :hi - lo] = _stand_for(kept).to(F64).transpose(0, 1)
            v[r, :, :hi - lo] = _stand_for(s["v"][lo:hi].to(torch.float16).to(F64)).to(F64).transpose(0, 1)
            continue
        K, V = _rows64(s["pages"][0][s["table"][r, :_cdiv(n, TOKENS)].long()], n)
        q = _turned(s["q_gate"][lo:hi, :, :HD], s["q_norm"], s["rope"], at)
        gate = torch.sigmoid(s["q_gate"][lo:hi, :, HD:].to(F64))
        hidden = torch.arange(n, device=DEV) > at.unsqueeze(1)
        for h in range(HEADS):
            p = torch.softmax((torch.mm(q[:, h], K[h // 4].T.contiguous()) / 16).masked_fill(hidden, -math.inf), -1)
            out[lo:hi, h] = torch.mm(p, V[h // 4]) * gate[:, h]
    return {"k": k, "v": v} if kind == "append" else {"out": out}

"""The operators of beam search over DeepSeek-V2-Lite's latent cache: choosing the
beams, forking and moving the pages of a cache, the cache rows in 8 bits, and the
attention over them, each in plain torch and through `fleet_moe`.

A page holds 64 positions of every layer. One layer of it is 36,992 bytes: four
blocks of 16 positions, each [36 chunks][16 positions][16 bytes] of e4m3 codes
(dimension 16 * chunk + byte), then fp32 scales [4 blocks][2] for dimensions
0..511 (c) and 512..575 (k_pe), powers of two. `table` [sequences][max_pages]
names a sequence's pages (-1 behind the last), `lens` its positions, `refs` how
many sequences hold a page.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
if str(_ROOT / "fleet-mi300x_amd") not in sys.path:
    sys.path.insert(0, str(_ROOT / "fleet-mi300x_amd"))

_DEV = "cuda"
_HEADS, _LORA, _ROPE = 16, 512, 64
_ROW = _LORA + _ROPE
_LAYERS, _VOCAB = 27, 102400
_PAGE, _BLOCK = 64, 16                      # positions of a page, of a block
_CODES = _PAGE * _ROW                       # code bytes of one layer of a page
_BYTES = 36992                              # with its scales
_E_MIN, _E4M3_MAX = -110, 448.0
_FLT_MAX = 3.4028234663852886e38
# (qk_nope + qk_rope)^-0.5 * mscale(40, 0.707)^2
_SCALE = 192.0 ** -0.5 * (0.1 * 0.707 * math.log(40.0) + 1.0) ** 2


def listed():
    return [
        # one request's beams, one decode step: all latency
        {"name": "beam_4", "kind": "beam", "groups": 1, "beams": 4, "out": 4, "vocab": _VOCAB},
        # a full server: 32 requests of 8 beams, twice as many candidates kept
        {"name": "beam_256", "kind": "beam", "groups": 32, "beams": 8, "out": 16,
         "vocab": _VOCAB},
        # one layer's new rows of 17 sequences in one decode step
        {"name": "append_17", "kind": "append", "layers": 1, "seqs": 17, "len": 1000, "new": 1},
        # a prompt's cache of the whole model moves into pages
        {"name": "append_1000", "kind": "append", "layers": _LAYERS, "seqs": 1, "len": 1000,
         "new": 1000},
        # a sequence's cache goes back to the batch-1 decoder
        {"name": "read_1000", "kind": "read", "layers": _LAYERS, "seqs": 1, "len": 1000,
         "new": 1000},
        # the step between two tokens of 16 beams: states follow their parents, and
        # pages that two beams would now write are copied
        {"name": "fork_16", "kind": "fork", "layers": _LAYERS, "groups": 4, "beams": 4,
         "len": 1000},
        # a pool that is half empty after requests have ended
        {"name": "compact_128", "kind": "compact", "layers": _LAYERS, "seqs": 8, "len": 1024},
        # one sequence, one token
        {"name": "attend_1", "kind": "attend", "seqs": 1, "len": 1024, "new": 1, "window": 0,
         "sinks": 0},
        # a large decode batch of ragged, long sequences
        {"name": "attend_64", "kind": "attend", "seqs": 64, "len": 8192, "new": 1, "window": 0,
         "sinks": 0},
        # streams far longer than their window, four first positions kept
        {"name": "window_8", "kind": "attend", "seqs": 8, "len": 32000, "new": 1,
         "window": 4096, "sinks": 4},
        # a prompt from its first token on
        {"name": "prompt_384", "kind": "attend", "seqs": 1, "len": 384, "new": 384, "window": 0,
         "sinks": 0},
        # the last chunks of four long prompts together
        {"name": "prompt_2000", "kind": "attend", "seqs": 4, "len": 4096, "new": 500,
         "window": 0, "sinks": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["beam", "append", "read", "fork", "compact", "decode", "window", "prompt"])
    if kind == "beam":
        beams = _log_int(rng, 1, 16)
        return {"kind": kind, "groups": _log_int(rng, 1, 256 // beams), "beams": beams,
                "out": min(64, beams * rng.choice([1, 2])),
                "vocab": _log_int(rng, 500, _VOCAB)}
    if kind in ("append", "read"):
        n = _log_int(rng, 1, 1000)
        return {"kind": kind, "layers": rng.choice([1, 3, _LAYERS]), "seqs": _log_int(rng, 1, 16),
                "len": n + rng.randrange(0, 500), "new": n}
    if kind == "fork":
        return {"kind": kind, "layers": rng.choice([1, 3, _LAYERS]), "groups": _log_int(rng, 1, 8),
                "beams": _log_int(rng, 1, 8), "len": _log_int(rng, 2, 2000)}
    if kind == "compact":
        return {"kind": kind, "layers": rng.choice([1, 3, _LAYERS]), "seqs": _log_int(rng, 1, 8),
                "len": _log_int(rng, 2, 2000)}
    if kind == "decode":
        return {"kind": "attend", "seqs": _log_int(rng, 1, 64), "len": _log_int(rng, 2, 8192),
                "new": 1, "window": 0, "sinks": 0}
    if kind == "window":
        return {"kind": "attend", "seqs": _log_int(rng, 1, 8), "len": _log_int(rng, 16, 32000),
                "new": rng.choice([1, 1, 3]), "window": _log_int(rng, 1, 4096),
                "sinks": rng.choice([0, 1, 4, 64])}
    n = _log_int(rng, 2, 500)
    return {"kind": "attend", "seqs": _log_int(rng, 1, 4), "len": n + rng.randrange(0, 3500),
            "new": n, "window": rng.choice([0, 0, 700]), "sinks": rng.choice([0, 4])}


# ---------------------------------------------------------------- sizes

def _pages(n):
    return -(-n // _PAGE)


def _lens(case):
    """Every sequence's positions: ragged, from 5/8 of `len` up to it, and what is
    new of them: from `new` on down."""
    n, top = case["seqs"], case["len"]
    lens = [max(1, top - (top * 3 * i) // (8 * n)) for i in range(n)]
    new = [max(1, case["new"] - (case["new"] * i) // (4 * n)) for i in range(n)]
    return lens, [min(a, b) for a, b in zip(new, lens)]


def _beam_lens(case):
    """Positions of each beam, the same within a request, and the pages that a
    request's beams share."""
    lens = [max(1, case["len"] - 7 * (g % 8)) for g in range(case["groups"])]
    return lens, [(3 * n) // (4 * _PAGE) for n in lens]


# ---------------------------------------------------------------- inputs

def _gen(seed, stream):
    g = torch.Generator(device=_DEV)
    g.manual_seed((int(seed) * 1_000_003 + stream) & (2**62 - 1))
    return g


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return _int32(out)


def _pool(seed, n_pages, layers):
    """A pool whose every block holds normal values under scales of its own."""
    g = _gen(seed, 1)
    pool = torch.zeros((n_pages, layers, _BYTES), dtype=torch.uint8, device=_DEV)
    codes = pool[..., :_CODES].view(torch.float8_e4m3fn)
    for a in range(0, n_pages, 64):
        n = min(64, n_pages - a)
        v = torch.randn((n, layers, _CODES), generator=g, device=_DEV, dtype=torch.bfloat16)
        codes[a: a + n] = v.mul_(100.0).clamp_(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    e = torch.randint(-8, -5, (n_pages, layers, 8), generator=g, device=_DEV)
    pool[..., _CODES: _CODES + 32].view(torch.float32).copy_(torch.exp2(e.float()))
    return pool


def _table(seed, owned, n_pages, max_pages):
    """Rows of `owned` page numbers (lists of 0..), which are dealt the pool's pages
    in a shuffled order, and how many rows hold each page."""
    perm = torch.randperm(n_pages, generator=_gen(seed, 2), device=_DEV).to(torch.int32)
    rows = torch.full((len(owned), max_pages), -1, dtype=torch.int64)
    for i, o in enumerate(owned):
        rows[i, : len(o)] = torch.tensor(o, dtype=torch.int64)
    rows = rows.to(_DEV)
    table = torch.where(rows >= 0, perm[rows.clamp(min=0)], -1).to(torch.int32)
    refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)
    return table, refs


def _book(s, table, lens, refs):
    """Table, lengths and counts of holders in one buffer, and a copy of it."""
    s["book"] = torch.cat([table.reshape(-1), lens, refs])
    s["book0"] = s["book"].clone()
    n, m = table.numel(), table.numel() + lens.numel()
    s["table"], s["lens"], s["refs"] = (s["book"][:n].view(table.shape), s["book"][n:m],
                                        s["book"][m:])


def prepare(case, seed):
    kind = case["kind"]
    s = {"kind": kind}
    if kind == "beam":
        g, b = case["groups"], case["beams"]
        x = torch.randn((g * b, case["vocab"]), generator=_gen(seed, 3), device=_DEV)
        s["logits"] = (3.0 * x).bfloat16().float()        # as lm_head leaves them
        s["scores"] = -12.0 * torch.rand((g, b), generator=_gen(seed, 4), device=_DEV)
        u = torch.rand((g, b), generator=_gen(seed, 5), device=_DEV)
        s["finished"] = (u < 0.1).to(torch.uint8)
        s["out"], s["eos"] = case["out"], 1
        if own:
            from fleet_moe import ops
            s["select"] = ops.BeamSelector(g, b, case["out"], case["vocab"], eos=1, device=_DEV)
        return s
    if kind == "fork":
        lens, shared = _beam_lens(case)
        owned, at = [], 0
        for n, k in zip(lens, shared):
            common = list(range(at, at + k))
            at += k
            for _ in range(case["beams"]):
                owned.append(common + list(range(at, at + _pages(n) - k)))
                at += _pages(n) - k
        rows = len(owned)
        n_pages, max_pages = at + 2 * rows + 5, _pages(case["len"]) + 2
        s["lens0"] = [n for n in lens for _ in range(case["beams"])]
        group = torch.arange(rows, device=_DEV) // case["beams"] * case["beams"]
        pick = torch.randint(0, case["beams"], (rows,), generator=_gen(seed, 6), device=_DEV)
        s["parents"] = (group + pick).to(torch.int32)
        s["new"] = torch.ones(rows, dtype=torch.int32, device=_DEV)
    else:
        lens, new = _lens(case) if kind != "compact" else ([case["len"]] * case["seqs"], None)
        owned, at = [], 0
        for n in lens:
            owned.append(list(range(at, at + _pages(n))))
            at += _pages(n)
        n_pages, max_pages = (2 * at + 3 if kind == "compact" else at + 2), _pages(case["len"])
        s["lens0"] = lens
    s["pool"] = _pool(seed, n_pages, case.get("layers", 1))
    table, refs = _table(seed, owned, n_pages, max_pages)
    _book(s, table, _int32(s["lens0"]), refs)
    if kind in ("append", "read"):
        s["start"] = _starts(new)
        shape = (case["layers"], sum(new), _ROW)
        x = torch.randn(shape, generator=_gen(seed, 7), device=_DEV)
        x[..., _LORA:] *= 5.0                             # k_pe is not normalised
        s["rows"] = x.bfloat16() if kind == "append" else torch.zeros_like(x).bfloat16()
    if kind == "attend":
        s["start"] = _starts(new)
        s["window"], s["sinks"], s["top"] = case["window"], case["sinks"], case["len"]
        s["most"] = max(new)
        q = torch.randn((sum(new), _HEADS, _ROW), generator=_gen(seed, 8), device=_DEV)
        s["q"] = (0.5 * q).bfloat16()
    if own:
        from fleet_moe import paged
        s["cache"] = paged.PagedCache(s["pool"], s["table"], s["lens"], s["refs"])
    return s


# ---------------------------------------------------------------- run

def run(s):
    return _run_own(s) if own else _PLAIN[s["kind"]](s)


def _run_own(s):
    kind = s["kind"]
    if kind == "beam":
        return s["select"].select(s["logits"], s["scores"], s["finished"])
    c = s["cache"]
    if kind == "append":
        c.append(s["rows"].view(torch.int16), s["start"])
        return _held(s)
    if kind == "read":
        c.read(s["rows"].view(torch.int16), s["start"])
        return {"rows": s["rows"]}
    if kind == "attend":
        out, lse = c.attend(s["q"].view(torch.int16), s["start"], max_len=s["top"],
                            window=s["window"], sinks=s["sinks"])
        return {"out": out.view(torch.bfloat16), "lse": lse}
    s["book"].copy_(s["book0"])
    if kind == "fork":
        c.remap(s["parents"])
        c.grow(s["new"])
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "pool": s["pool"]}
    used = c.compact()
    return {"table": s["table"], "refs": s["refs"], "used": used, "pool": s["pool"]}


def _held(s):
    """What the pool holds: e4m3 values and their scales."""
    return {"codes": s["pool"][..., :_CODES].view(torch.float8_e4m3fn),
            "scales": s["pool"][..., _CODES: _CODES + 32].view(torch.float32)}


# ---------------------------------------------------------------- plain forms

def _unpack(pool, table):
    """The values and the exponents of the scales that a table's pages hold, by
    sequence and position: fp32 [layers][seqs][positions][576] without their scales, and
    fp32 [layers][seqs][blocks][2]."""
    pages = pool[table.clamp(min=0).long()].permute(2, 0, 1, 3)   # layers, seqs, pages, bytes
    n, b, p = pages.shape[:3]
    v = pages[..., :_CODES].view(torch.float8_e4m3fn).float()
    v = v.view(n, b, p, 4, _ROW // 16, _BLOCK, 16).permute(0, 1, 2, 3, 5, 4, 6)
    scales = pages[..., _CODES: _CODES + 32].contiguous().view(torch.float32)
    return v.reshape(n, b, p * _PAGE, _ROW), scales.view(n, b, p * 4, 2)


def _values(pool, table):
    """fp32 [layers][seqs][positions][576]: what the pages stand for."""
    v, scales = _unpack(pool, table)
    per = scales.repeat_interleave(_BLOCK, 2)
    return torch.cat([v[..., :_LORA] * per[..., :1], v[..., _LORA:] * per[..., 1:]], -1)


def _places(start, lens, n):
    """The sequence and the position of each of the n rows that `start` deals out."""
    i = torch.arange(n, device=_DEV)
    seq = torch.searchsorted(start[1:].long(), i, right=True)
    return seq, lens.long()[seq] - (start.long()[seq + 1] - i)


def _plain_append(s):
    pool, table, rows = s["pool"], s["table"], s["rows"].float()
    n, total = rows.shape[0], rows.shape[1]
    seq, pos = _places(s["start"], s["lens"], total)
    v, scales = _unpack(pool, table)
    b, t = v.shape[1], v.shape[2]
    new = torch.zeros((b, t), dtype=torch.bool, device=_DEV)
    new[seq, pos] = True
    first = s["lens"].long() - (s["start"][1:] - s["start"][:-1]).long()
    old = torch.arange(t, device=_DEV) < first[:, None]
    by_block = lambda m: m.view(b, t // _BLOCK, _BLOCK).any(-1)    # noqa: E731
    touched, kept = by_block(new), by_block(old)
    # the largest finite magnitude of a block's new rows, per part
    mag = torch.where(rows.isfinite(), rows.abs(), 0.0)
    mag = torch.stack([mag[..., :_LORA].amax(-1), mag[..., _LORA:].amax(-1)], -1)
    dense = torch.zeros((n, b, t, 2), device=_DEV)
    dense[:, seq, pos] = mag
    m, x = torch.frexp(dense.view(n, b, t // _BLOCK, _BLOCK, 2).amax(3))
    e = torch.where(m <= 0.875, x - 9, x - 8)                     # 448 = 0.875 * 2^9
    e = torch.where(m == 0, _E_MIN, e).clamp(min=_E_MIN)
    e_old = torch.frexp(scales)[1] - 1
    e = torch.where(kept[None, :, :, None], torch.maximum(e, e_old), e)
    e = torch.where(touched[None, :, :, None], e, e_old)
    spread = lambda a: torch.cat([a[..., :1].expand(*a.shape[:-1], _LORA),   # noqa: E731
                                  a[..., 1:].expand(*a.shape[:-1], _ROPE)], -1)
    per = lambda a: a.repeat_interleave(_BLOCK, 2)                # noqa: E731
    v = v * spread(per(torch.exp2((e_old - e).float())))
    step = torch.exp2(-e.float())[:, seq, pos // _BLOCK]
    fresh = (rows * spread(step)).clamp(-_E4M3_MAX, _E4M3_MAX)
    v[:, seq, pos] = torch.where(rows.isinf(), rows.sign() * _E4M3_MAX, fresh)
    # back into the pages: new rows, and the older ones of their blocks
    codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    codes = codes.view(n, b, t // _PAGE, 4, _BLOCK, _ROW // 16, 16).permute(1, 2, 0, 3, 5, 4, 6)
    write = (new | (old & touched.repeat_interleave(_BLOCK, 1))).view(b, t // _PAGE, 1, 4, 1,
                                                                       _BLOCK, 1)
    held = pool[table.clamp(min=0).long()]
    was = held[..., :_CODES].reshape(codes.shape)
    held[..., :_CODES] = torch.where(write, codes, was).reshape(held.shape[:-1] + (_CODES,))
    held[..., _CODES: _CODES + 32] = torch.exp2(e.float()).view(n, b, t // _PAGE, 8).permute(
        1, 2, 0, 3).contiguous().view(torch.uint8)
    pool[table[table >= 0].long()] = held[table >= 0]
    return _held(s)


def _plain_read(s):
    rows = s["rows"]
    seq, pos = _places(s["start"], s["lens"], rows.shape[1])
    rows.copy_(_values(s["pool"], s["table"])[:, seq, pos].bfloat16())
    return {"rows": rows}


def _plain_attend(s):
    q, start, lens = s["q"].float(), s["start"].long(), s["lens"].long()
    n, b, most = q.shape[0], lens.numel(), s["most"]
    k = _values(s["pool"], s["table"])[0]                         # [b][t][576]
    t = k.shape[1]
    at = torch.arange(t, device=_DEV)
    k = torch.where((at < lens[:, None])[..., None], k, 0.0)
    seq, pos = _places(s["start"], s["lens"], n)
    slot = torch.arange(n, device=_DEV) - start[seq]
    dense = torch.zeros((b, most, _HEADS, _ROW), device=_DEV)
    dense[seq, slot] = q
    where = torch.full((b, most), -1, dtype=torch.int64, device=_DEV)
    where[seq, slot] = pos
    z = torch.matmul(dense.view(b, most * _HEADS, _ROW), k.transpose(1, 2)) * _SCALE
    seen = at <= where[..., None]
    if s["window"] > 0:
        seen = seen & ((at > where[..., None] - s["window"]) | (at < s["sinks"]))
    z = z.view(b, most, _HEADS, t).masked_fill_(~seen[:, :, None], -math.inf)
    m = z.amax(-1, keepdim=True).clamp_(min=-_FLT_MAX)
    p = z.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, most * _HEADS, t), k[..., :_LORA]).view(b, most, _HEADS, _LORA)
    o = torch.where(total > 0, o / total, 0.0)[seq, slot]
    return {"out": o.bfloat16(), "lse": (m + total.log())[seq, slot, :, 0]}


def _plain_fork(s):
    s["book"].copy_(s["book0"])
    table, lens, refs, pool = s["table"], s["lens"], s["refs"], s["pool"]
    parents = s["parents"].long()
    alive = parents >= 0
    table.copy_(torch.where(alive[:, None], table[parents.clamp(min=0)], -1))
    lens.copy_(torch.where(alive, lens[parents.clamp(min=0)], 0))
    refs.zero_().index_add_(0, table.clamp(min=0).view(-1).long(),
                            (table >= 0).view(-1).to(torch.int32))
    # pages for the new positions; a shared last page that is not full is copied
    rows = torch.arange(lens.numel(), device=_DEV)
    n, new = lens.long(), s["new"].long()
    have, want = (n + _PAGE - 1) // _PAGE, (n + new + _PAGE - 1) // _PAGE
    last = table[rows, (have - 1).clamp(min=0)].long()
    open_ = (new > 0) & (n % _PAGE > 0)
    rank = ((last[:, None] == last) & open_ & (rows < rows[:, None])).sum(1)
    copy = open_ & (refs[last.clamp(min=0)] - rank > 1)
    need = want - have + copy
    before = need.cumsum(0) - need
    free = torch.sort((refs > 0).to(torch.int8), stable=True)[1]  # the free pages first
    at = torch.arange(table.shape[1], device=_DEV)
    lo = (have - copy.long())[:, None]
    fresh = (at >= lo) & (at < want[:, None])
    given = free[(before[:, None] + at - lo).clamp(0, refs.numel() - 1)]
    table.copy_(torch.where(fresh, given.to(torch.int32), table))
    refs.zero_().index_add_(0, table.clamp(min=0).view(-1).long(),
                            (table >= 0).view(-1).to(torch.int32))
    src, dst = last[copy], free[before[copy]]
    filled = (n[copy] % _PAGE + _BLOCK - 1) // _BLOCK * (_BLOCK * _ROW)
    byte = torch.arange(_BYTES, device=_DEV)
    moved = ((byte < filled[:, None]) | (byte >= _CODES))[:, None]
    pool[dst] = torch.where(moved, pool[src], pool[dst])
    lens.add_(s["new"])
    return {"table": table, "lens": lens, "refs": refs, "pool": pool}


def _plain_compact(s):
    s["book"].copy_(s["book0"])
    table, refs, pool = s["table"], s["refs"], s["pool"]
    held = refs > 0
    used = held.sum()
    page = torch.arange(refs.numel(), device=_DEV)
    from_, to = page[held & (page >= used)], page[~held & (page < used)]
    pool[to] = pool[from_]
    new = page.clone()
    new[from_] = to
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].to(torch.int32), -1))
    refs[to] = refs[from_]
    refs[from_] = 0
    return {"table": table, "refs": refs, "used": used.to(torch.int32).view(1), "pool": pool}


def _plain_beam(s):
    x, (g, b), out = s["logits"], s["scores"].shape, s["out"]
    vocab = x.shape[1]
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=_FLT_MAX)
    score, done = s["scores"].reshape(-1).double(), s["finished"].reshape(-1) > 0
    m = x.amax(1).double()
    z = (x.double() - m[:, None]).exp_().sum(1).log_()
    top, token = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(out, vocab)
    top, token = top[:, :k].double(), token[:, :k]
    cand = score[:, None] + ((top - m[:, None]) - z[:, None])
    cand = torch.where(top > -math.inf, cand, -math.inf)
    first = torch.arange(k, device=_DEV) == 0
    cand = torch.where(done[:, None], torch.where(first, score[:, None], -math.inf), cand)
    token = torch.where(done[:, None], s["eos"], token)
    cand = torch.where(cand.isnan(), -math.inf, cand).view(g, b * k)
    if b * k < out:
        cand = torch.cat([cand, torch.full((g, out - b * k), -math.inf, device=_DEV,
                                           dtype=cand.dtype)], 1)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    best, at = best[:, :out], at[:, :out]
    there = best > -math.inf
    at = torch.where(there, at, 0)
    parent = at // k + torch.arange(g, device=_DEV)[:, None] * b
    token = token.reshape(g, b * k).gather(1, at)
    ended = there & (done[parent] | (token == s["eos"]))
    return {"scores": best.float(), "parents": torch.where(there, parent, -1).to(torch.int32),
            "tokens": torch.where(there, token, -1).to(torch.int32),
            "finished": ended.to(torch.uint8)}


_PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend,
          "fork": _plain_fork, "compact": _plain_compact, "beam": _plain_beam}


# ---------------------------------------------------------------- work

def _seen(case):
    """Positions that some query reads, and the pairs of query and position."""
    union = pairs = 0
    for n, m in zip(*_lens(case)):
        w = case["window"] or n
        lo = max(0, n - m - w + 1)
        union += n - lo + min(case["sinks"], lo)
        for p in range(n - m, n):
            a = max(0, p - w + 1)
            pairs += p + 1 - a + min(case["sinks"], a)
    return union, pairs


def work(case):
    kind = case["kind"]
    if kind == "beam":
        n = case["groups"] * case["beams"]
        return {"bytes": 4 * n * case["vocab"] + 13 * case["groups"] * case["out"],
                "flops": 4 * n * case["vocab"]}
    if kind in ("append", "read"):
        n = case["layers"] * sum(_lens(case)[1])
        return {"bytes": n * (3 * _ROW + 0.5), "flops": n * _ROW}
    layer = 2 * case.get("layers", 1)
    if kind == "fork":
        lens, _ = _beam_lens(case)
        beams = case["beams"]
        # beams that share a parent: the mean of beams - distinct parents
        twins = beams - beams * (1 - (1 - 1 / beams) ** beams)
        copied = sum(twins * -(-(n % _PAGE) // _BLOCK) * _BLOCK * _ROW for n in lens)
        rows = case["groups"] * beams
        return {"bytes": layer * copied + 8 * rows * _pages(case["len"]), "flops": rows}
    if kind == "compact":
        used = case["seqs"] * _pages(case["len"])
        total = 2 * used + 3
        return {"bytes": layer * _BYTES * used * (total - used) / total + 8 * total,
                "flops": total}
    union, pairs = _seen(case)
    rows = sum(_lens(case)[1]) * _HEADS
    return {"bytes": union * (_ROW + 0.5) + rows * (2 * _ROW + 2 * _LORA + 4),
            "flops": 2 * _HEADS * pairs * (_ROW + _LORA)}


# ---------------------------------------------------------------- 64-bit values

def _row_exact(s, layer, i, p):
    """The cache row of sequence i at positions p, in 64 bits."""
    page = s["table"][i].long()[p // _PAGE]
    blk, tok = p % _PAGE // _BLOCK, p % _BLOCK
    dim = torch.arange(_ROW, device=_DEV)
    byte = (blk * _BLOCK * _ROW + tok * 16)[:, None] + dim // 16 * 256 + dim % 16
    bits = s["pool"][page, layer].gather(1, byte).long()
    sign, ex, man = bits >> 7, bits >> 3 & 15, (bits & 7).double()
    mag = torch.where(ex > 0, (8 + man) * torch.exp2(ex.double() - 10), man * 2.0**-9)
    mag = torch.where((bits & 127) == 127, math.nan, mag)
    scales = s["pool"][page, layer, _CODES: _CODES + 32].contiguous().view(torch.float32)
    part = blk[:, None] * 2 + (dim >= _LORA)
    return torch.where(sign > 0, -mag, mag) * scales.double().gather(1, part)


def exact(case, seed):
    kind = case["kind"]
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if kind == "beam":
        return _beam_exact(s)
    if kind == "attend":
        return _attend_exact(s)
    if kind == "append":
        return _append_exact(s)
    if kind == "read":
        lens, new = _lens(case)
        rows = [torch.cat([_row_exact(s, layer, i, torch.arange(n - m, n, device=_DEV))
                           for i, (n, m) in enumerate(zip(lens, new))])
                for layer in range(case["layers"])]
        return {"rows": torch.stack(rows)}
    return None            # whole numbers and moved bytes: nothing is computed


def _attend_exact(s):
    start = s["start"].tolist()
    outs, lses = [], []
    for i, n in enumerate(s["lens0"]):
        k = _row_exact(s, 0, i, torch.arange(n, device=_DEV))
        at = torch.arange(n, device=_DEV)
        q = s["q"][start[i]: start[i + 1]].double()
        for a in range(0, q.shape[0], 64):
            part = q[a: a + 64]
            p = n - q.shape[0] + a + torch.arange(part.shape[0], device=_DEV)
            z = _SCALE * (part.reshape(-1, _ROW) @ k.T).view(part.shape[0], _HEADS, n)
            gone = at[None] > p[:, None]
            if s["window"]:
                gone = gone | ((p[:, None] - at[None] >= s["window"]) & (at[None] >= s["sinks"]))
            z.masked_fill_(gone[:, None], -math.inf)
            lse = torch.logsumexp(z, -1)
            w = torch.exp(z - lse[..., None])
            outs.append((w.view(-1, n) @ k[:, :_LORA]).view(part.shape[0], _HEADS, _LORA))
            lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _append_exact(s):
    """The codes and scales after the rows are in, block by block. Rounding to
    e4m3 is part of the definition: it is done here on 64-bit values."""
    start = s["start"].tolist()
    if s["rows"].shape[0] * start[-1] > 30000:
        return None
    codes = s["pool"][..., :_CODES].view(torch.float8_e4m3fn).double()
    scales = s["pool"][..., _CODES: _CODES + 32].contiguous().view(torch.float32).double()
    rows = s["rows"].double()
    table = s["table"].tolist()
    byte = torch.arange(_BLOCK * _ROW, device=_DEV).view(_ROW // 16, _BLOCK, 16)
    byte = byte.transpose(0, 1).reshape(_BLOCK, _ROW)             # [position][dimension]
    for i, n in enumerate(s["lens0"]):
        first = n - (start[i + 1] - start[i])
        for b0 in range(first // _BLOCK * _BLOCK, n, _BLOCK):
            page, blk = table[i][b0 // _PAGE], b0 % _PAGE // _BLOCK
            a, z = max(first, b0) - b0, min(n, b0 + _BLOCK) - b0
            at = start[i] + b0 + a - first
            for c, (lo, hi) in enumerate(((0, _LORA), (_LORA, _ROW))):
                place = blk * _BLOCK * _ROW + byte[:, lo:hi]
                fresh = rows[:, at: at + z - a, lo:hi]
                scale = torch.full((rows.shape[0],), 2.0**_E_MIN, dtype=torch.float64,
                                   device=_DEV)
                big = fresh.abs().amax((1, 2))
                # the least power of two that takes the largest within 448
                e = torch.log2(big / _E4M3_MAX).round().clamp(min=_E_MIN + 2)
                for d in (1, 0, -1):
                    ok = big <= _E4M3_MAX * torch.exp2(e + d)
                    scale = torch.where(ok & (big > 0), torch.exp2(e + d), scale)
                kept = codes[page][:, place[:a]] * scales[page, :, 2 * blk + c, None, None]
                if a:
                    scale = torch.maximum(scale, scales[page, :, 2 * blk + c])
                both = torch.cat([kept, fresh], 1) / scale[:, None, None]
                codes[page][:, place[:z]] = _e4m3(both)
                scales[page, :, 2 * blk + c] = scale
    return {"codes": codes, "scales": scales}


def _e4m3(v):
    """The nearest values of 4 significant bits and exponents from -6 on, ties to even."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _beam_exact(s):
    g, b = s["scores"].shape
    best = []
    for i in range(g):
        x = s["logits"][i * b: (i + 1) * b].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        c = s["scores"][i].double()[:, None] + lp
        done = s["finished"][i] > 0
        c[done] = -math.inf
        c[done, 0] = s["scores"][i].double()[done]
        c = c.reshape(-1).sort(descending=True)[0][: s["out"]]
        best.append(torch.nn.functional.pad(c, (0, s["out"] - c.numel()), value=-math.inf))
    return {"scores": torch.stack(best), "parents": None, "tokens": None, "finished": None}

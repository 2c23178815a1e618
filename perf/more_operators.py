"""The operators between the layers' products and DeepSeek-V2-Lite's paged latent
cache, for several sequences at once, each in plain torch and through `fleet_moe`:
the norms around a block with its gate and residual, the rotation of queries, the
projected rows' way into the pages (norm of c, rotation of k_pe, 8 bits), and the
attention of sequences that share their first pages.

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
_HIDDEN, _HEADS, _NOPE, _LORA, _ROPE = 2048, 16, 128, 512, 64
_ROW = _LORA + _ROPE
_QKV = _HEADS * (_NOPE + _ROPE) + _ROW      # a row of the fused projection
_PAGE, _BLOCK = 64, 16                      # positions of a page, of a block
_CODES = _PAGE * _ROW                       # code bytes of one layer of a page
_BYTES = 36992                              # with its scales
_E_MIN, _E4M3_MAX, _EPS = -110, 448.0, 1e-6
# (qk_nope + qk_rope)^-0.5 * mscale(40, 0.707)^2
_SCALE = 192.0 ** -0.5 * (0.1 * 0.707 * math.log(40.0) + 1.0) ** 2


def listed():
    return [
        # between two layers' halves, one token: latency
        {"name": "norm_1", "kind": "norm", "tokens": 1, "hidden": _HIDDEN, "x": "fp32",
         "post": False, "gate": ""},
        # a decode batch whose block ends in a norm and a gate for each channel
        {"name": "norm_250", "kind": "norm", "tokens": 250, "hidden": _HIDDEN, "x": "bf16",
         "post": True, "gate": "channel"},
        # the prompts of a full server, gated for each token
        {"name": "norm_16000", "kind": "norm", "tokens": 16000, "hidden": _HIDDEN, "x": "bf16",
         "post": False, "gate": "token"},
        # one token's queries, out of the projection's row into the absorbed ones
        {"name": "rope_1", "kind": "rope", "tokens": 1, "heads": _HEADS, "width": _ROPE, "at": 0,
         "dim": _ROPE, "type": "bf16", "halves": False, "seqs": 1, "far": 1024},
        # the last 500 tokens of four prompts, their positions taken from the cache
        {"name": "rope_2000", "kind": "rope", "tokens": 2000, "heads": _HEADS, "width": _ROPE,
         "at": 0, "dim": _ROPE, "type": "bf16", "halves": False, "seqs": 4, "far": 4096},
        # whole heads with their part that is not rotated, in fp32, at positions far out
        {"name": "rope_8001", "kind": "rope", "tokens": 8001, "heads": _HEADS,
         "width": _NOPE + _ROPE, "at": _NOPE, "dim": _ROPE, "type": "fp32", "halves": True,
         "seqs": 0, "far": 1 << 20},
        # 17 sequences' new row in one decode step of one layer
        {"name": "latent_17", "kind": "latent", "seqs": 17, "len": 1000, "new": 1, "norm": True},
        # three ragged prompts at once
        {"name": "latent_4001", "kind": "latent", "seqs": 3, "len": 5000, "new": 4001,
         "norm": True},
        # one request's four hypotheses
        {"name": "shared_4", "kind": "shared", "groups": 1, "seqs": 4, "prefix": 1000, "own": 40,
         "new": 1},
        # 64 requests behind one long instruction
        {"name": "shared_64", "kind": "shared", "groups": 1, "seqs": 64, "prefix": 8192,
         "own": 500, "new": 1},
        # eight documents, 16 hypotheses each, four proposed tokens looked at together
        {"name": "drafts_128", "kind": "shared", "groups": 8, "seqs": 16, "prefix": 4000,
         "own": 300, "new": 4},
        # a full server on two long documents
        {"name": "shared_256", "kind": "shared", "groups": 2, "seqs": 128, "prefix": 16300,
         "own": 1000, "new": 1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "rope", "latent", "shared", "shared"])
    if kind == "norm":
        hidden = rng.choice([_HIDDEN, _log_int(rng, 16, 8192), 8 * _log_int(rng, 8, 1024)])
        x, gate = rng.choice(["bf16", "fp32"]), rng.choice(["", "channel", "token"])
        each = 2 * hidden * ((4 if x == "bf16" else 6) + (gate == "token"))
        return {"kind": kind, "hidden": hidden,
                "tokens": _log_int(rng, 1, min(16000, 320_000_000 // each)),
                "x": x, "post": rng.random() < 0.5, "gate": gate}
    if kind == "rope":
        dim = rng.choice([_ROPE, 2 * rng.randrange(1, 65)])
        at = rng.choice([0, _NOPE, rng.randrange(0, 130)])
        heads, tokens = _log_int(rng, 1, 128), _log_int(rng, 1, 8001)
        most = 8001 * _HEADS * (_NOPE + _ROPE) // (heads * (at + dim + 8))
        return {"kind": kind, "tokens": min(tokens, most), "heads": heads,
                "width": at + dim + rng.choice([0, 0, 8]), "at": at, "dim": dim,
                "type": rng.choice(["bf16", "fp32"]), "halves": rng.random() < 0.5,
                "seqs": rng.choice([0, 1, 4]), "far": _log_int(rng, 1024, 1 << 20)}
    if kind == "latent":
        n = _log_int(rng, 1, 4001)
        return {"kind": kind, "seqs": _log_int(rng, 1, max(1, min(32, 10000 // n))),
                "len": n + rng.randrange(0, 900), "new": n, "norm": rng.random() < 0.8}
    groups, seqs, new = _log_int(rng, 1, 8), _log_int(rng, 1, 64), rng.choice([1, 1, 2, 5])
    most = 16300 * 256 // (groups * seqs * new)
    return {"kind": kind, "groups": groups, "seqs": seqs,
            "prefix": _log_int(rng, 10, max(10, min(16300, most - 500))),
            "own": _log_int(rng, new, 500), "new": new}


# ---------------------------------------------------------------- sizes

def _pages(n):
    return -(-n // _PAGE)


def _lens(case):
    """Every sequence's positions, ragged: from 5/8 of `len` up to it (shared: of what is
    its own behind the prefix), and what is new of them, from `new` on down."""
    if case["kind"] == "shared":
        n, own_ = case["groups"] * case["seqs"], case["own"]
        # neighbours differ, the groups do not
        lens = [case["prefix"] + max(case["new"], own_ - (own_ * 3 * (i % 16)) // (8 * 16))
                for i in range(n)]
        return lens, [case["new"]] * n
    n, top = case["seqs"], case["len"]
    lens = [max(1, top - (top * 3 * i) // (8 * n)) for i in range(n)]
    new = [max(1, case["new"] - (case["new"] * i) // (4 * n)) for i in range(n)]
    return lens, [min(a, b) for a, b in zip(new, lens)]


def _rope_lens(case):
    """The tokens of each sequence and its positions, where the cache has them."""
    n = case["seqs"]
    new = [case["tokens"] // n + (i < case["tokens"] % n) for i in range(n)]
    return [max(case["far"] - 7 * i, m) for i, m in enumerate(new)], new


# ---------------------------------------------------------------- inputs

def _gen(seed, stream):
    g = torch.Generator(device=_DEV)
    g.manual_seed((int(seed) * 1_000_003 + stream) & (2**62 - 1))
    return g


def _normal(seed, stream, *shape):
    return torch.randn(shape, generator=_gen(seed, stream), device=_DEV)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return _int32(out)


def _frequencies(dim):
    """Radians a position of each pair: base 10,000, the slow ones stretched 40 times, as
    for a context of 4,096 that is extended."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / dim)
    turns = 4096.0 * f / (2.0 * math.pi)
    keep = ((turns.log2() - 0.0) / 5.0).clamp(0.0, 1.0)    # 1 .. 32 turns in the context
    return f * keep + f / 40.0 * (1.0 - keep)


def _pool(seed, n_pages):
    """A pool of one layer whose every block holds normal values under scales of its own."""
    g = _gen(seed, 1)
    pool = torch.zeros((n_pages, 1, _BYTES), dtype=torch.uint8, device=_DEV)
    v = torch.randn((n_pages, 1, _CODES), generator=g, device=_DEV, dtype=torch.bfloat16)
    pool[..., :_CODES].view(torch.float8_e4m3fn).copy_(
        v.mul_(100.0).clamp_(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn))
    e = torch.randint(-8, -5, (n_pages, 1, 8), generator=g, device=_DEV)
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


def _cache(s):
    from fleet_moe import paged
    return paged.PagedCache(s["pool"], s["table"], s["lens"], s["refs"])


def prepare(case, seed):
    kind = case["kind"]
    s = {"kind": kind}
    if kind == "norm":
        t, h = case["tokens"], case["hidden"]
        x = 4.0 * _normal(seed, 3, t, h)
        s["x"] = x.bfloat16() if case["x"] == "bf16" else x
        s["y"] = _normal(seed, 4, t, h).bfloat16()
        s["w"] = (1.0 + 0.1 * _normal(seed, 5, h)).bfloat16()
        s["post"] = (0.5 + 0.1 * _normal(seed, 6, h)).bfloat16() if case["post"] else None
        gate = {"": (), "channel": (h,), "token": (t, h)}[case["gate"]]
        s["gate"] = torch.sigmoid(_normal(seed, 7, *gate)).bfloat16() if gate else None
        s["scale"] = 0.7
        return s
    if kind == "rope":
        t, n, w, dim = case["tokens"], case["heads"], case["width"], case["dim"]
        # a part of wider heads in a longer row, and a place in wider heads
        dt = torch.bfloat16 if case["type"] == "bf16" else torch.float32
        row = _normal(seed, 3, t, n * (w + _NOPE) + _ROW).to(dt)
        s["x"] = row[:, : n * (w + _NOPE)].view(t, n, w + _NOPE)[..., _NOPE:]
        s["out"] = torch.zeros((t, n, _LORA + w), dtype=dt, device=_DEV)[..., _LORA:]
        s["at"], s["dim"], s["halves"] = case["at"], dim, case["halves"]
        s["freq"] = _frequencies(dim).to(_DEV)
        if case["seqs"]:
            lens, new = _rope_lens(case)
            s["lens"], s["start"] = _int32(lens), _starts(new)
        else:
            s["pos"] = torch.randint(0, case["far"], (t,), generator=_gen(seed, 4),
                                     device=_DEV).to(torch.int32)
        if own:
            from fleet_moe import ops
            s["rope"] = ops.Rotary(s["freq"], halves_in=case["halves"], halves_out=True)
            if case["seqs"]:
                pages = _pages(max(lens))
                s["table"] = torch.zeros((case["seqs"], pages), dtype=torch.int32, device=_DEV)
                s["refs"] = torch.full((1,), case["seqs"] * pages, dtype=torch.int32, device=_DEV)
                s["pool"] = torch.zeros((1, 1, _BYTES), dtype=torch.uint8, device=_DEV)
                s["cache"] = _cache(s)
        return s
    lens, new = _lens(case)
    owned, at = [], 0
    if kind == "shared":
        k = case["prefix"] // _PAGE                        # what is left of it is copied
        for i, n in enumerate(lens):
            if i % case["seqs"] == 0:
                common = list(range(at, at + k))
                at += k
            owned.append(common + list(range(at, at + _pages(n) - k)))
            at += _pages(n) - k
        s["groups"] = _int32([i * case["seqs"] for i in range(case["groups"] + 1)])
        s["shared"] = k * _PAGE
    else:
        for n in lens:
            owned.append(list(range(at, at + _pages(n))))
            at += _pages(n)
    s["lens0"], s["new0"], s["lens"], s["start"] = lens, new, _int32(lens), _starts(new)
    s["pool"] = _pool(seed, at + 2)
    s["table"], s["refs"] = _table(seed, owned, at + 2, _pages(max(lens)))
    if kind == "latent":
        # the last part of the fused projection's rows
        s["rows"] = _normal(seed, 7, sum(new), _QKV).bfloat16()[:, _QKV - _ROW:]
        s["w"] = (1.0 + 0.1 * _normal(seed, 8, _LORA)).bfloat16() if case["norm"] else None
        s["freq"] = _frequencies(_ROPE).to(_DEV)
    else:
        s["q"] = (0.5 * _normal(seed, 8, sum(new), _HEADS, _ROW)).bfloat16()
    if own:
        from fleet_moe import ops, paged
        s["cache"] = _cache(s)
        if kind == "latent":
            s["rope"] = ops.Rotary(s["freq"], halves_in=False, halves_out=True)
        else:
            s["plan"] = paged.SharedPrefix(s["cache"], s["groups"], sum(new), _HEADS)
            s["plan"].update()
    return s


# ---------------------------------------------------------------- run

def run(s):
    return _run_own(s) if own else _PLAIN[s["kind"]](s)


def _bits(t):
    return t if t is None or t.dtype == torch.float32 else t.view(torch.int16)


def _run_own(s):
    kind = s["kind"]
    if kind == "norm":
        from fleet_moe import ops
        x, h = ops.residual_norm(_bits(s["x"]), _bits(s["y"]), norm=_bits(s["w"]),
                                 post_norm=_bits(s["post"]), gate=_bits(s["gate"]),
                                 scale=s["scale"], eps=_EPS)
        return {"x": x.view(s["x"].dtype), "h": h.view(torch.bfloat16)}
    if kind == "rope":
        x, out = _bits(s["x"]), _bits(s["out"])
        if "pos" in s:
            s["rope"].rotate(x, s["pos"], out=out, at=s["at"])
        else:
            s["cache"].rotate(s["rope"], x, s["start"], out=out, at=s["at"])
        return {"out": s["out"]}
    if kind == "latent":
        s["cache"].append_latent(_bits(s["rows"]), s["rope"], norm=_bits(s["w"]),
                                 start=s["start"], eps=_EPS)
        return _held(s)
    out, lse = s["plan"].attend(_bits(s["q"]), s["start"])
    return {"out": out.view(torch.bfloat16), "lse": lse}


def _held(s):
    """What the pool holds: e4m3 values and their scales."""
    return {"codes": s["pool"][..., :_CODES].view(torch.float8_e4m3fn),
            "scales": s["pool"][..., _CODES: _CODES + 32].view(torch.float32)}


# ---------------------------------------------------------------- plain forms

def _rms(v):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)


def _plain_norm(s):
    u = s["y"].float()
    if s["post"] is not None:
        u = _rms(u) * s["post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    x = s["x"].float() + s["scale"] * u
    return {"x": x.to(s["x"].dtype), "h": (_rms(x) * s["w"].float()).bfloat16()}


def _turned(x, pos, freq, halves):
    """x [n][heads][dim] at positions pos [n], the pairs' first values and then their second."""
    a = pos.double()[:, None] * freq
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    half = x.shape[-1] // 2
    u, v = (x[..., :half], x[..., half:]) if halves else (x[..., 0::2], x[..., 1::2])
    return torch.cat([u * cos - v * sin, v * cos + u * sin], -1)


def _plain_rope(s):
    x, at, end = s["x"], s["at"], s["at"] + s["dim"]
    pos = s["pos"] if "pos" in s else _places(s["start"], s["lens"], x.shape[0])[1]
    out = s["out"]
    out[..., :at] = x[..., :at]
    out[..., end:] = x[..., end:]
    out[..., at:end] = _turned(x[..., at:end].float(), pos, s["freq"], s["halves"]).to(out.dtype)
    return {"out": out}


def _unpack(pool, table):
    """The values and the scales that a table's pages hold, by sequence and position:
    fp32 [seqs][positions][576] without their scales, and fp32 [seqs][blocks][2]."""
    pages = pool[table.clamp(min=0).long(), 0]                    # seqs, pages, bytes
    b, p = pages.shape[:2]
    v = pages[..., :_CODES].view(torch.float8_e4m3fn).float()
    v = v.view(b, p, 4, _ROW // 16, _BLOCK, 16).transpose(3, 4)
    scales = pages[..., _CODES: _CODES + 32].contiguous().view(torch.float32)
    return v.reshape(b, p * _PAGE, _ROW), scales.view(b, p * 4, 2)


def _values(pool, table):
    """fp32 [seqs][positions][576]: what the pages stand for."""
    v, scales = _unpack(pool, table)
    per = scales.repeat_interleave(_BLOCK, 1)
    return torch.cat([v[..., :_LORA] * per[..., :1], v[..., _LORA:] * per[..., 1:]], -1)


def _places(start, lens, n):
    """The sequence and the position of each of the n rows that `start` deals out."""
    i = torch.arange(n, device=_DEV)
    seq = torch.searchsorted(start[1:].long(), i, right=True)
    return seq, lens.long()[seq] - (start.long()[seq + 1] - i)


def _plain_latent(s):
    pool, table, rows = s["pool"], s["table"], s["rows"].float()
    seq, pos = _places(s["start"], s["lens"], rows.shape[0])
    c = _rms(rows[:, :_LORA])
    if s["w"] is not None:
        c = c * s["w"].float()
    pe = _turned(rows[:, None, _LORA:], pos, s["freq"], False)[:, 0]
    rows = torch.cat([c, pe], -1)
    v, scales = _unpack(pool, table)
    b, t = v.shape[:2]
    new = torch.zeros((b, t), dtype=torch.bool, device=_DEV)
    new[seq, pos] = True
    first = s["lens"].long() - (s["start"][1:] - s["start"][:-1]).long()
    old = torch.arange(t, device=_DEV) < first[:, None]
    by_block = lambda m: m.view(b, t // _BLOCK, _BLOCK).any(-1)    # noqa: E731
    touched, kept = by_block(new), by_block(old)
    dense = torch.zeros((b, t, 2), device=_DEV)
    dense[seq, pos] = torch.stack([rows[:, :_LORA].abs().amax(-1), rows[:, _LORA:].abs().amax(-1)],
                                  -1)
    m, x = torch.frexp(dense.view(b, t // _BLOCK, _BLOCK, 2).amax(2))
    e = torch.where(m <= 0.875, x - 9, x - 8)                     # 448 = 0.875 * 2^9
    e = torch.where(m == 0, _E_MIN, e).clamp(min=_E_MIN)
    e_old = torch.frexp(scales)[1] - 1
    e = torch.where(kept[..., None], torch.maximum(e, e_old), e)
    e = torch.where(touched[..., None], e, e_old)
    spread = lambda a: torch.cat([a[..., :1].expand(*a.shape[:-1], _LORA),   # noqa: E731
                                  a[..., 1:].expand(*a.shape[:-1], _ROPE)], -1)
    v = v * spread(torch.exp2((e_old - e).float()).repeat_interleave(_BLOCK, 1))
    step = torch.exp2(-e.float())[seq, pos // _BLOCK]
    v[seq, pos] = (rows * spread(step)).clamp(-_E4M3_MAX, _E4M3_MAX)
    # back into the pages: new rows, and the older ones of their blocks
    codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    codes = codes.view(b, t // _PAGE, 4, _BLOCK, _ROW // 16, 16).transpose(3, 4)
    write = (new | (old & touched.repeat_interleave(_BLOCK, 1))).view(b, t // _PAGE, 4, 1, _BLOCK,
                                                                       1)
    held = pool[table.clamp(min=0).long(), 0]
    was = held[..., :_CODES].reshape(codes.shape)
    held[..., :_CODES] = torch.where(write, codes, was).reshape(held.shape[:-1] + (_CODES,))
    held[..., _CODES: _CODES + 32] = torch.exp2(e.float()).view(b, t // _PAGE, 8).view(torch.uint8)
    pool[table[table >= 0].long(), 0] = held[table >= 0]
    return _held(s)


def _plain_shared(s):
    """A group's common positions in one product, what is each sequence's own in another."""
    q, lens, n_shared = s["q"].float(), s["lens"].long(), s["shared"]
    n, b = q.shape[0], lens.numel()
    groups, k = s["groups"].numel() - 1, s["new0"][0]
    common = n_shared // _PAGE
    front = _values(s["pool"], s["table"][:: b // groups, :common])   # [groups][shared][576]
    back = _values(s["pool"], s["table"][:, common:])                 # [b][t][576]
    at = n_shared + torch.arange(back.shape[1], device=_DEV)
    back = torch.where((at < lens[:, None])[..., None], back, 0.0)
    pos = (lens - k)[:, None] + torch.arange(k, device=_DEV)          # [b][k]
    z0 = torch.matmul(q.view(groups, -1, _ROW), front.transpose(1, 2)) * _SCALE
    z1 = torch.matmul(q.view(b, k * _HEADS, _ROW), back.transpose(1, 2)) * _SCALE
    z1 = z1.view(b, k, _HEADS, -1).masked_fill_((at > pos[..., None])[:, :, None], -math.inf)
    rows = n * _HEADS
    z0, z1 = z0.view(rows, n_shared), z1.view(rows, back.shape[1])
    m = z1.amax(-1, keepdim=True)
    if n_shared:
        m = torch.maximum(m, z0.amax(-1, keepdim=True))
    p0, p1 = z0.sub_(m).exp_(), z1.sub_(m).exp_()
    total = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
    o = torch.matmul(p0.view(groups, rows // groups, n_shared), front[..., :_LORA])
    o = o.view(rows, _LORA) + torch.matmul(p1.view(b, k * _HEADS, -1), back[..., :_LORA]).view(
        rows, _LORA)
    return {"out": (o / total).view(n, _HEADS, _LORA).bfloat16(),
            "lse": (m + total.log()).view(n, _HEADS)}


_PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "latent": _plain_latent,
          "shared": _plain_shared}


# ---------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, h = case["tokens"] * case["hidden"], case["hidden"]
        x = 2 if case["x"] == "bf16" else 4
        gate = {"": 0, "channel": 2 * h, "token": 2 * n}[case["gate"]]
        return {"bytes": n * (2 * x + 4) + gate + 2 * h * (1 + case["post"]),
                "flops": n * (6 + 4 * case["post"] + bool(gate))}
    if kind == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["width"] * (2 if case["type"] == "bf16" else 4),
                "flops": 3 * n * case["dim"]}
    lens, new = _lens(case)
    if kind == "latent":
        return {"bytes": sum(new) * (3 * _ROW + 0.5), "flops": sum(new) * (5 * _LORA + 4 * _ROPE)}
    common = case["prefix"] // _PAGE * _PAGE
    held = case["groups"] * common + sum(n - common for n in lens)
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))
    rows = sum(new) * _HEADS
    return {"bytes": held * (_ROW + 0.5) + rows * (2 * _ROW + 2 * _LORA + 4),
            "flops": 2 * _HEADS * pairs * (_ROW + _LORA)}


# ---------------------------------------------------------------- 64-bit values

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norm": _norm_exact, "rope": _rope_exact, "latent": _latent_exact,
            "shared": _shared_exact}[case["kind"]](s)


def _norm_exact(s):
    unit = lambda v: v / torch.sqrt(torch.linalg.vecdot(v, v)[:, None] / v.shape[1]   # noqa: E731
                                    + _EPS)
    u = s["y"].double()
    if s["post"] is not None:
        u = unit(u) * s["post"].double()
    if s["gate"] is not None:
        u = u * s["gate"].double()
    x = s["x"].double() + 0.7 * u
    return {"x": x, "h": unit(x) * s["w"].double()}


def _exact_turn(x, pos, freq, halves):
    """The pairs as complex numbers, by powers of e^(i angle)."""
    d = x.shape[-1]
    pairs = x.reshape(*x.shape[:-1], 2, d // 2).transpose(-1, -2) if halves else \
        x.reshape(*x.shape[:-1], d // 2, 2)
    z = torch.view_as_complex(pairs.double().contiguous())
    z = z * torch.polar(torch.ones((), dtype=torch.float64, device=_DEV),
                        pos.double().view(-1, *[1] * (x.dim() - 1)) * freq)
    return torch.cat([z.real, z.imag], -1)


def _exact_positions(s):
    start, lens = s["start"].tolist(), s["lens"].tolist()
    return torch.cat([torch.arange(n - (start[i + 1] - start[i]), n, device=_DEV)
                      for i, n in enumerate(lens)])


def _rope_exact(s):
    pos = s["pos"] if "pos" in s else _exact_positions(s)
    out, end = s["x"].double().clone(), s["at"] + s["dim"]
    out[..., s["at"]: end] = _exact_turn(s["x"][..., s["at"]: end], pos, s["freq"], s["halves"])
    return {"out": out}


def _block_bytes():
    """The byte of a block's [position][dimension]."""
    byte = torch.arange(_BLOCK * _ROW, device=_DEV).view(_ROW // 16, _BLOCK, 16)
    return byte.transpose(0, 1).reshape(_BLOCK, _ROW)


def _latent_exact(s):
    """What the codes stand for after the rows are in, block by block, before each is
    rounded to 8 bits, and the scales."""
    start = s["start"].tolist()
    x = s["rows"].double()
    c = x[:, :_LORA]
    c = c / torch.sqrt((c * c).mean(-1, keepdim=True) + _EPS)
    if s["w"] is not None:
        c = c * s["w"].double()
    rows = torch.cat([c, _exact_turn(x[:, _LORA:], _exact_positions(s), s["freq"], False)], -1)
    codes = s["pool"][:, 0, :_CODES].view(torch.float8_e4m3fn).double()
    scales = s["pool"][:, 0, _CODES: _CODES + 32].contiguous().view(torch.float32).double()
    table, byte = s["table"].tolist(), _block_bytes()
    for i, n in enumerate(s["lens0"]):
        first = n - (start[i + 1] - start[i])
        for b0 in range(first // _BLOCK * _BLOCK, n, _BLOCK):
            page, blk = table[i][b0 // _PAGE], b0 % _PAGE // _BLOCK
            a, z = max(first, b0) - b0, min(n, b0 + _BLOCK) - b0
            fresh = rows[start[i] + b0 + a - first: start[i] + b0 + z - first]
            for p, (lo, hi) in enumerate(((0, _LORA), (_LORA, _ROW))):
                # the least power of two that takes the largest within 448
                big = fresh[:, lo:hi].abs().amax() / _E4M3_MAX
                e = torch.frexp(big)
                scale = torch.where(e[0] == 0.5, big, torch.exp2(e[1].double()))
                if a:
                    scale = torch.maximum(scale, scales[page, 2 * blk + p])
                place = blk * _BLOCK * _ROW + byte[:, lo:hi]
                if a:
                    codes[page, place[:a]] *= scales[page, 2 * blk + p] / scale
                codes[page, place[a:z]] = fresh[:, lo:hi] / scale
                scales[page, 2 * blk + p] = scale
    return {"codes": codes[:, None], "scales": scales[:, None]}


def _shared_exact(s):
    """Every sequence by itself, over all its positions."""
    start = s["start"].tolist()
    byte = _block_bytes()
    value = torch.arange(256, device=_DEV)
    ex, man = value >> 3 & 15, (value & 7).double()
    value = torch.where(ex > 0, (8 + man) * torch.exp2(ex.double() - 10), man * 2.0**-9) \
        * torch.where(torch.arange(256, device=_DEV) >= 128, -1.0, 1.0)
    outs, lses = [], []
    for i, n in enumerate(s["lens0"]):
        pages = s["table"][i, : _pages(n)].long()
        held = s["pool"][pages, 0]
        codes = held[:, :_CODES].reshape(-1, _BLOCK * _ROW)[:, byte]            # [blocks][16][576]
        k = value[codes.long()]
        per = held[:, _CODES: _CODES + 32].contiguous().view(torch.float32).double().view(-1, 2)
        k[..., :_LORA] *= per[:, None, :1]
        k[..., _LORA:] *= per[:, None, 1:]
        k = k.view(-1, _ROW)[:n]
        q = s["q"][start[i]: start[i + 1]].double()
        m = q.shape[0]
        z = _SCALE * (q.view(-1, _ROW) @ k.T).view(m, _HEADS, n)
        late = torch.arange(n, device=_DEV)[None] > (n - m + torch.arange(m, device=_DEV))[:, None]
        z.masked_fill_(late[:, None], -math.inf)
        lse = torch.logsumexp(z, -1)
        w = torch.exp(z - lse[..., None])
        outs.append((w.view(-1, n) @ k[:, :_LORA]).view(m, _HEADS, _LORA))
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}

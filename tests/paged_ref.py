"""The paged 8-bit cache and the beams' choice, restated in NumPy from their
definitions (include/fleet_moe.h), one sequence, block and position at a time and
in 64 bits: what the GPU tests compare with."""
from __future__ import annotations

import numpy as np

ROW, C, PAGE, BLOCK, BYTES = 576, 512, 64, 16, 36992
CODES = PAGE * ROW
E_MIN = -110


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes (NaN for 0x7f and 0xff)."""
    b = np.arange(256)
    e, m = b >> 3 & 15, (b & 7).astype(np.float64)
    mag = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0**-9)
    mag[b & 127 == 127] = np.nan
    return np.where(b >= 128, -mag, mag)


VALUES = e4m3_values()


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """The codes nearest to x (|x| <= 448), ties to the even one; NaN is 0x7f."""
    mags = VALUES[:127]
    a = np.abs(x)
    hi = np.clip(np.searchsorted(mags, np.nan_to_num(a)), 1, 126)
    lo = hi - 1
    dl, dh = a - mags[lo], mags[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(x), 127, code)
    return (code + 128 * np.signbit(x)).astype(np.uint8)


def bf16(x) -> np.ndarray:
    """Values rounded to bf16, as fp32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + (u >> 16 & 1)) >> 16 << 16).astype(np.uint32)
    out = r.view(np.float32).copy()
    out[np.isnan(x)] = np.nan
    return out


def bits(x) -> np.ndarray:
    """bf16-valued fp32 as int16 bits."""
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(
        np.int16)


def values(b: np.ndarray) -> np.ndarray:
    """int16 bf16 bits as fp32."""
    return (b.astype(np.uint16).astype(np.uint32) << 16).view(np.float32)


def unpack(pool: np.ndarray):
    """Pool bytes [pages][layers][36992] as codes [pages][layers][64][576] and
    scales [pages][layers][4][2]."""
    n, layers = pool.shape[:2]
    codes = pool[..., :CODES].reshape(n, layers, 4, ROW // 16, BLOCK, 16)
    codes = codes.transpose(0, 1, 2, 4, 3, 5).reshape(n, layers, PAGE, ROW)
    scales = np.ascontiguousarray(pool[..., CODES: CODES + 32]).view(np.float32)
    return codes, scales.reshape(n, layers, 4, 2)


class Cache:
    def __init__(self, n_pages, n_seqs, max_pages, n_layers):
        self.n_pages, self.n_layers, self.max_pages = n_pages, n_layers, max_pages
        self.codes = np.zeros((n_pages, n_layers, PAGE, ROW), np.uint8)
        self.exps = np.zeros((n_pages, n_layers, PAGE // BLOCK, 2), np.int64)
        self.rows = [[] for _ in range(n_seqs)]          # pages
        self.lens = [0] * n_seqs

    def refs(self):
        r = np.zeros(self.n_pages, np.int32)
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def table(self):
        t = np.full((len(self.rows), self.max_pages), -1, np.int32)
        for i, row in enumerate(self.rows):
            t[i, : len(row)] = row
        return t

    def remap(self, parents):
        ok = [p if 0 <= p < len(self.rows) else -1 for p in parents]
        self.rows, self.lens = ([list(self.rows[p]) if p >= 0 else [] for p in ok],
                                [self.lens[p] if p >= 0 else 0 for p in ok])

    def grow(self, n_new) -> bool:
        """False, and nothing done, where the pages do not suffice."""
        if min(n_new) < 0:
            return False
        want = [-(-(n + a) // PAGE) for n, a in zip(self.lens, n_new)]
        if max(want) > self.max_pages:
            return False
        refs = self.refs()
        free = [p for p in range(self.n_pages) if refs[p] == 0]
        rows, copies = [list(r) for r in self.rows], []
        for s, a in enumerate(n_new):
            row, n = rows[s], self.lens[s]
            if a > 0 and n % PAGE and refs[row[-1]] > 1:
                if not free:
                    return False
                refs[row[-1]] -= 1
                copies.append((row[-1], free[0], -(-(n % PAGE) // BLOCK)))
                row[-1] = free.pop(0)
            while len(row) < want[s]:
                if not free:
                    return False
                row.append(free.pop(0))
        for src, dst, n in copies:
            self.codes[dst, :, : n * BLOCK] = self.codes[src, :, : n * BLOCK]
            self.exps[dst] = self.exps[src]
        self.rows, self.lens = rows, [n + a for n, a in zip(self.lens, n_new)]
        return True

    def compact(self) -> int:
        refs = self.refs()
        used = int((refs > 0).sum())
        movers = [p for p in range(used, self.n_pages) if refs[p]]
        holes = [p for p in range(used) if not refs[p]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.codes[b], self.exps[b] = self.codes[a], self.exps[a]
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return used

    def append(self, rows, start, layer=0):
        """rows fp32 (bf16-valued) [layers][n][576]."""
        for s in range(len(self.rows)):
            n, total = start[s + 1] - start[s], self.lens[s]
            first = total - n
            for b0 in range(max(first, 0) // BLOCK * BLOCK, total, BLOCK):
                page, blk = self.rows[s][b0 // PAGE], b0 % PAGE // BLOCK
                at = range(max(first, b0, 0), min(total, b0 + BLOCK))
                if not len(at):
                    continue
                for k in range(rows.shape[0]):
                    for part, (lo, hi) in enumerate(((0, C), (C, ROW))):
                        new = rows[k, [start[s] + p - first for p in at], lo:hi].astype(np.float64)
                        self._block(page, layer + k, blk, part, lo, hi, at, max(first, 0) - b0, new)

    def _block(self, page, layer, blk, part, lo, hi, at, aged, new):
        fin = np.abs(new[np.isfinite(new)])
        big = fin.max() if fin.size else 0.0
        e = E_MIN
        while big > 448.0 * 2.0**e:
            e += 1
        old = self.exps[page, layer, blk, part]
        if aged > 0:
            e = max(e, old)
            if e > old:
                sl = (page, layer, slice(blk * BLOCK, blk * BLOCK + aged), slice(lo, hi))
                self.codes[sl] = to_e4m3(VALUES[self.codes[sl]] * 2.0 ** float(old - e))
        self.exps[page, layer, blk, part] = e
        x = np.where(np.isinf(new), np.sign(new) * 448.0, new * 2.0 ** float(-e))
        where = [p % PAGE for p in at]
        self.codes[page, layer, where, lo:hi] = to_e4m3(x)

    def values(self, s, layer=0):
        """fp64 [lens[s]][576]."""
        n = self.lens[s]
        if n == 0:
            return np.zeros((0, ROW))
        v = VALUES[self.codes[self.rows[s], layer]].reshape(-1, ROW)[:n]
        e = np.repeat(self.exps[self.rows[s], layer].reshape(-1, 2), BLOCK, 0)[:n]
        return np.concatenate([v[:, :C] * 2.0 ** e[:, :1].astype(float),
                               v[:, C:] * 2.0 ** e[:, 1:].astype(float)], 1)


def attend(rows, q, positions, scale, window=0, sinks=0):
    """Attention of q [n][heads][576] at `positions` over rows [len][576], in 64
    bits: (out, lse, tolerance of out, tolerance of lse). The tolerances are
    what the stated arithmetic may be off by: half a bf16 step (2^-8) of out, and
    of each weight in numerator and denominator (2 * 2^-8 of A = sum w |c|);
    the fp32 sums of 576 products, 576 * 2^-24 of B = scale * sum |q row|, in every
    score, doubled for the weights; and 2^-20 for exponentials, logarithms and
    the additions of up to some thousand weights."""
    n, heads = q.shape[:2]
    out, lse = np.zeros((n, heads, C)), np.full((n, heads), -np.inf)
    t_out, t_lse = np.zeros((n, heads, C)), np.zeros((n, heads))
    at = np.arange(rows.shape[0])
    for i, p in enumerate(positions):
        see = at <= p
        if window > 0:
            see &= (at > p - window) | (at < sinks)
        k = rows[see]
        if not len(k):
            continue
        z = scale * q[i].astype(np.float64) @ k.T
        b = (scale * np.abs(q[i]).astype(np.float64) @ np.abs(k).T).max(1)
        m = z.max(1, keepdims=True)
        w = np.exp(z - m)
        lse[i] = m[:, 0] + np.log(w.sum(1))
        w /= w.sum(1, keepdims=True)
        out[i] = w @ k[:, :C]
        a = w @ np.abs(k[:, :C])
        err = 576 * 2.0**-24 * b
        t_out[i] = 2.0**-8 * np.abs(out[i]) + (2.0**-7 + 4 * err[:, None] + 2.0**-20) * a
        t_lse[i] = err + 2.0**-20 * (1 + np.abs(lse[i]))
    return out, lse, t_out, t_lse


def beam_select(logits, scores, finished, n_out, eos):
    """logits [groups][beams][vocab], scores [groups][beams]: lists of
    (score, parent row, token, finished) per group, best first."""
    groups, beams, vocab = logits.shape
    result = []
    for g in range(groups):
        cand = []
        for b in range(beams):
            s = float(scores[g, b])
            if np.isnan(s) or s == -np.inf:
                continue
            if finished[g, b]:
                cand.append((s, b, 0.0, eos if eos >= 0 else -1, 1))
                continue
            x = np.minimum(logits[g, b].astype(np.float64), np.float64(np.finfo(np.float32).max))
            ok = ~np.isnan(x) & (x != -np.inf)
            if not ok.any():
                continue
            m = x[ok].max()
            z = np.log(np.exp(x[ok] - m).sum())
            ids = np.flatnonzero(ok)
            best = ids[np.lexsort((ids, -x[ids]))][:n_out]
            cand += [(s + ((x[t] - m) - z), b, x[t], int(t), int(t == eos)) for t in best]
        cand.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        rows = [(c[0], g * beams + c[1], c[3], c[4]) for c in cand[:n_out]]
        result.append(rows + [(-np.inf, -1, -1, 0)] * (n_out - len(rows)))
    return result

"""GPU: projected rows into the pages (PagedCache.append_latent): the norm of c, the rotation
of k_pe and the rounding to a block's 8 bits, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, ops, paged, rope  # noqa: E402

FREQS = rope.frequencies().astype(np.float64)


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def say(msg):
    print(f"[gpu] {msg}", flush=True)


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def to_dev(x):
    return torch.from_numpy(ref.bits(x)).cuda()


def made(x, norm, pos, halves=False, eps=1e-6, freqs=FREQS, mag=1.0):
    """The cache's rows in 64 bits, of rows x [n][576] at positions pos."""
    c, pe = x[:, :512].astype(np.float64), x[:, 512:].astype(np.float64)
    with np.errstate(invalid="ignore"):
        c = c / np.sqrt((c * c).mean(1, keepdims=True) + eps)
        if norm is not None:
            c = c * norm
        a, b = (pe[:, :32], pe[:, 32:]) if halves else (pe[:, 0::2], pe[:, 1::2])
        ang = np.asarray(pos, np.float64)[:, None] * freqs
        co, si = mag * np.cos(ang), mag * np.sin(ang)
        return np.concatenate([c, a * co - b * si, b * co + a * si], 1)


class Cached:
    """The cache on the device, and what its positions should hold in 64 bits."""

    def __init__(self, n_seqs, n_pages=40, max_pages=20, n_layers=1, fill=0xFF):
        self.c = paged.PagedCache.empty(n_pages, n_seqs, max_pages, n_layers)
        self.c.pool.fill_(fill)
        self.rows = [np.zeros((0, ref.ROW)) for _ in range(n_seqs)]

    def append(self, counts, x, norm=None, halves=False, layer=0, mag=1.0, rows=None, eps=1e-6):
        r = ops.Rotary(FREQS, mag, halves_in=halves)
        self.c.grow(i32(counts))
        at = np.concatenate([[0], np.cumsum(counts)])
        self.c.append_latent(to_dev(x) if rows is None else rows, r,
                             None if norm is None else to_dev(norm), i32(at), layer, eps)
        for s, n in enumerate(counts):
            pos = len(self.rows[s]) + np.arange(n)
            new = made(x[at[s]: at[s + 1]], norm, pos, halves, eps, mag=mag)
            self.rows[s] = np.concatenate([self.rows[s], new])

    def check(self, layer=0, seqs=None):
        """The scale is the least that takes the block's largest value (and never falls: blocks
        here are appended to with values of one size, or the test looks itself). A value is
        off by half a step of 8 bits for every scale it was rounded under (2^-4 of it, or 2^-10
        of the scale below the least normal number), and 2^-18 for the norm and the angle in
        32 bits. Blocks that grew a row at a time were rounded up to 16 times."""
        assert self.c.status() == 0
        codes, scales = ref.unpack(self.c.pool.cpu().numpy())
        table = self.c.table.cpu().numpy()
        worst = 0.0
        for s, want in enumerate(self.rows):
            assert self.c.lens[s].item() == len(want)
            for b0 in range(0, len(want), 16):
                w = want[b0: b0 + 16]
                page, blk = table[s, b0 // 64], b0 % 64 // 16
                got = ref.VALUES[codes[page, layer, blk * 16: blk * 16 + len(w)]]
                for p, (lo, hi) in enumerate(((0, 512), (512, 576))):
                    scale = scales[page, layer, blk, p]
                    v = np.abs(w[:, lo:hi])
                    fin = v[np.isfinite(v)]
                    big = fin.max() if fin.size else 0.0
                    e = max(-110, int(np.ceil(np.log2(big / 448.0)))) if big > 0 else -110
                    assert scale == 2.0**e, (s, b0, p, scale, e)
                    ok = np.isfinite(w[:, lo:hi])
                    g = got[:, lo:hi] * scale
                    assert (np.isnan(g) == np.isnan(w[:, lo:hi])).all()
                    d = np.abs(g - np.where(ok, w[:, lo:hi], 0))[ok]
                    tol = np.maximum(2.0**-4 * v[ok], 2.0**-10 * scale)
                    worst = max(worst, (d / (tol + 2.0**-18 * big + 1e-300)).max(initial=0))
        return worst


def data(rng, n, big=3.0):
    x = rng.normal(size=(n, ref.ROW))
    x[:, 512:] *= big
    return ref.bf16(x)


@pytest.mark.parametrize("counts", [[1], [16], [17, 0, 1], [64, 65, 3], [300, 1, 128], [5] * 40])
@pytest.mark.parametrize("halves, normed", [(False, True), (True, False)])
def test_against_the_definition(counts, halves, normed):
    rng = np.random.default_rng(sum(counts))
    say(f"counts {counts[:4]} halves {halves}")
    t = Cached(len(counts))
    norm = ref.bf16(1 + 0.2 * rng.normal(size=512)) if normed else None
    t.append(counts, data(rng, sum(counts)), norm, halves, mag=1.25 if halves else 1.0)
    assert t.check() <= 1.0


def test_blocks_grow_a_row_at_a_time():
    """Rows of growing and falling size, one by one: the scale grows with them and never falls."""
    rng = np.random.default_rng(2)
    t = Cached(2, fill=0x7E)
    for i in range(40):
        norm = ref.bf16(np.full(512, 2.0 ** (i % 7 if i < 20 else -i)))
        x = data(rng, 2, 2.0 ** (i % 5))
        t.append([1, 1], x, norm)
    codes, scales = ref.unpack(t.c.pool.cpu().numpy())
    table = t.c.table.cpu().numpy()
    for s, want in enumerate(t.rows):
        for b0 in range(0, 40, 16):
            w, page, blk = want[b0: b0 + 16], table[s, 0], b0 // 16
            got = ref.VALUES[codes[page, 0, blk * 16: blk * 16 + len(w)]]
            for p, (lo, hi) in enumerate(((0, 512), (512, 576))):
                scale, v = scales[page, 0, blk, p], np.abs(w[:, lo:hi])
                assert scale == 2.0 ** np.ceil(np.log2(v.max() / 448.0))
                # rounded once for every scale since: at most 7 here
                tol = 8 * np.maximum(2.0**-4 * v, 2.0**-10 * scale) + 2.0**-18 * v.max()
                assert (np.abs(got[:, lo:hi] * scale - w[:, lo:hi]) <= tol).all()


def test_like_append_of_the_finished_rows():
    """What append() makes of the same rows, rounded to bf16 on the way: within that rounding
    and a step of 8 bits."""
    rng = np.random.default_rng(3)
    counts, x = [70, 3, 130], data(np.random.default_rng(4), 203)
    t = Cached(3)
    norm = ref.bf16(1 + 0.2 * rng.normal(size=512))
    t.append(counts, x, norm)
    other = paged.PagedCache.empty(40, 3, 20, 1)
    other.grow(i32(counts))
    start = i32(np.concatenate([[0], np.cumsum(counts)]))
    other.append(to_dev(ref.bf16(np.concatenate(t.rows).astype(np.float32))), start)
    out = [torch.zeros((203, ref.ROW), dtype=torch.int16, device="cuda") for _ in range(2)]
    for c, o in zip((t.c, other), out):
        c.read(o, start)
    a, b = (ref.values(o.cpu().numpy()).astype(np.float64) for o in out)
    assert (np.abs(a - b) <= (2.0**-3 + 2.0**-7) * np.maximum(np.abs(a), np.abs(b)) + 2.0**-9 * 2.0**-5).all()


def test_layers_strides_and_other_layers_untouched():
    """Rows that are the end of a fused projection's; one layer of three."""
    rng = np.random.default_rng(5)
    x = data(rng, 50)
    wide = torch.zeros((50, 16 * 192 + 576), dtype=torch.int16, device="cuda")
    rows = wide[:, 16 * 192:]
    rows.copy_(to_dev(x))
    t = Cached(2, n_layers=3)
    t.append([20, 30], x, layer=1, rows=rows)
    assert t.check(layer=1) <= 1.0
    assert (t.c.pool[:, 0] == 0xFF).all() and (t.c.pool[:, 2] == 0xFF).all()


def test_rows_of_every_kind_of_value():
    """Zeros, the largest and smallest numbers, infinities and NaN: they stay in their row and part,
    and the scale is of the finite ones."""
    rng = np.random.default_rng(6)
    x = data(rng, 12).astype(np.float64)
    x[0] = 0
    x[1, :512] *= 1e38 / 4
    x[2, :512] *= 1e-35
    x[3, :512] = 0
    x[3, 7] = 3e38
    x[4, 512:] = 0
    t = Cached(12)
    with np.errstate(over="ignore"):
        t.append([1] * 12, ref.bf16(x))
    assert t.check() <= 1.0
    x[5, 3], x[6, 4] = np.inf, np.nan
    x[7, 512 + 10], x[8, 512 + 11] = np.nan, -np.inf
    x[9, 512 + 20] = 3e38                       # rotated at position 0: alone in its pair
    t = Cached(12)
    t.append([1] * 12, ref.bf16(x))
    codes, scales = ref.unpack(t.c.pool.cpu().numpy())
    table = t.c.table.cpu().numpy()[:, 0]
    v = [ref.VALUES[codes[p, 0, 0]] * np.repeat(scales[p, 0, 0], [512, 64]) for p in table]
    # 1 / rms is 0: the infinity NaN, the others 0
    assert np.isnan(v[5][3]) and (np.delete(v[5][:512], 3) == 0).all()
    assert np.isnan(v[6][:512]).all()
    assert np.isnan(v[7][[5, 37]]).sum() == 0 and np.isnan(v[7][512:]).sum() == 2
    # an infinity times the sine 0 is NaN; times the cosine it is the largest code
    assert np.isnan(v[8][512:]).sum() + (np.abs(v[8][512:]) == 448 * scales[table[8], 0, 0, 1]).sum() == 2
    for i in (5, 6):
        w = t.rows[i][0, 512:]
        assert (np.abs(v[i][512:] - w) <= 2.0**-4 * np.abs(w) + 2.0**-9 * np.abs(w).max()).all()
    for i in (7, 8, 9):
        w = t.rows[i][0, :512]
        assert (np.abs(v[i][:512] - w) <= 2.0**-4 * np.abs(w) + 2.0**-9 * np.abs(w).max()).all()
    assert abs(v[9][512 + 10] - 3e38) <= 2.0**-4 * 3e38


def test_refused_growth_shared_and_bad_pages():
    """As append(): nothing is written where there is no room, a page is shared or outside
    the pool, or a row has no position."""
    rng = np.random.default_rng(7)
    r, x = ops.Rotary(FREQS), to_dev(data(rng, 2))
    c = paged.PagedCache.empty(2, 2, 2, 1)
    c.pool.fill_(0x11)
    c.grow(i32([64, 64]))
    before = c.pool.clone()
    c.grow(i32([1, 1]))
    c.append_latent(x, r)
    assert c.status() == _lib.ABORT_NO_PAGE and torch.equal(c.pool, before)
    c.clear_status()
    c.grow(i32([0, 0]))
    for page in (2, -1, 2**31 - 1):
        c.table[0, 0] = page
        c.append_latent(x[:1], r, start=i32([0, 1, 1]))
        assert c.status() == _lib.ABORT_BAD_PAGE and torch.equal(c.pool, before)
        c.clear_status()
    c.table[0, 0] = 0
    c.refs[0] = 2
    c.append_latent(x[:1], r, start=i32([0, 1, 1]))
    assert c.status() == _lib.ABORT_BAD_PAGE and torch.equal(c.pool, before)
    c.clear_status()
    c.refs[0] = 1
    c.lens.copy_(i32([129, 1]))
    c.append_latent(to_dev(data(rng, 5)), r, start=i32([0, 2, 5]))
    assert c.status() == _lib.ABORT_POSITION
    held = c.pool.view(2, 1, -1)
    assert torch.equal(held[int(c.table[0, 0])], before[0])


def test_rows_of_nobody_and_empty_calls():
    rng = np.random.default_rng(8)
    r = ops.Rotary(FREQS)
    x = data(rng, 9)
    t = Cached(2)
    t.c.grow(i32([3, 2]))
    t.c.append_latent(to_dev(x), r, start=i32([2, 5, 7]))
    for s, (a, z) in enumerate(((2, 5), (5, 7))):
        t.rows[s] = made(x[a:z], None, np.arange(z - a))
    assert t.check() <= 1.0
    before = t.c.pool.clone()
    t.c.append_latent(to_dev(x)[:0], r)
    t.c.append_latent(to_dev(x), r, start=i32([9, 9, 9]))
    assert torch.equal(t.c.pool, before) and t.c.status() == 0


def test_positions_far_out():
    """A row behind a million others: only its block is there, the angle is its own."""
    n = 1_000_003
    c = paged.PagedCache.empty(2, 1, n // 64 + 1, 1)
    c.lens.fill_(n)
    c.table[0, n // 64] = 1
    c.refs[1] = 1
    x = data(np.random.default_rng(9), 3)
    c.append_latent(to_dev(x), ops.Rotary(FREQS), start=i32([0, 3]))
    codes, scales = ref.unpack(c.pool.cpu().numpy())
    want = made(x, None, np.arange(n - 3, n))
    at = [p % 64 for p in range(n - 3, n)]
    assert at[0] // 16 == at[2] // 16 or c.status() == 0
    for i, p in enumerate(at):
        v = ref.VALUES[codes[1, 0, p]]
        for k, (lo, hi) in enumerate(((0, 512), (512, 576))):
            s = scales[1, 0, p // 16, k]
            tol = np.maximum(2.0**-4 * np.abs(want[i, lo:hi]), 2.0**-10 * s) + 2.0**-18 * 448 * s
            assert (np.abs(v[lo:hi] * s - want[i, lo:hi]) <= tol).all()


def test_refused_tensors():
    c = paged.PagedCache.empty(2, 2, 2, 1)
    r = ops.Rotary(FREQS)
    x = torch.zeros((2, ref.ROW), dtype=torch.int16, device="cuda")
    w = torch.zeros(512, dtype=torch.int16, device="cuda")
    for f in (lambda: c.append_latent(x.cpu(), r), lambda: c.append_latent(x.float(), r),
              lambda: c.append_latent(x[:, :-1], r), lambda: c.append_latent(x[None], r),
              lambda: c.append_latent(x[:1], r), lambda: c.append_latent(x.T, r),
              lambda: c.append_latent(x, r, norm=w[:-1]), lambda: c.append_latent(x, r, norm=w.float()),
              lambda: c.append_latent(x, r, start=i32([0, 2]))):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: c.append_latent(x, r, layer=1), lambda: c.append_latent(x, r, eps=0.0),
              lambda: c.append_latent(x, ops.Rotary(FREQS, halves_out=False)),
              lambda: c.append_latent(x, ops.Rotary(FREQS[:16])),
              lambda: c.append_latent(torch.zeros((2, 580), dtype=torch.int16, device="cuda")[:, 4:], r)):
        with pytest.raises(_lib.FleetMoeError):
            f()
    assert c.status() == 0

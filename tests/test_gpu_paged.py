"""GPU: the paged 8-bit cache (fleet_moe.paged) against its restatement in 64
bits (paged_ref.py): rows in and out, growing, forking and freeing, compaction,
and the attention over ragged, masked, strided and empty cases."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, paged  # noqa: E402

SCALE = paged.SOFTMAX_SCALE


def say(msg: str) -> None:
    print(f"[gpu] {msg}", flush=True)


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def starts(counts):
    return i32(np.concatenate([[0], np.cumsum(counts)]))


def to_dev(x):
    return torch.from_numpy(ref.bits(x)).cuda()


class Both:
    """The same cache on the device and restated."""

    def __init__(self, n_pages, n_seqs, max_pages, n_layers, fill=0xFF):
        self.dev = paged.PagedCache.empty(n_pages, n_seqs, max_pages, n_layers)
        self.dev.pool.fill_(fill)               # NaN codes where nothing was written
        self.ref = ref.Cache(n_pages, n_seqs, max_pages, n_layers)

    def grow(self, n_new):
        ok = self.ref.grow(list(n_new))
        self.dev.grow(i32(n_new))
        return ok

    def remap(self, parents):
        self.ref.remap(list(parents))
        self.dev.remap(i32(parents))

    def compact(self):
        used = self.ref.compact()
        assert int(self.dev.compact().item()) == used

    def append(self, counts, rows, layer=0):
        at = np.concatenate([[0], np.cumsum(counts)])
        self.ref.append(rows, at, layer)
        self.dev.append(to_dev(rows), i32(at), layer)

    def check(self, status=0, layers=slice(None)):
        """`layers`: those that were written."""
        torch.cuda.synchronize()
        d, r = self.dev, self.ref
        assert d.status() == status
        assert np.array_equal(d.lens.cpu().numpy(), r.lens)
        assert np.array_equal(d.table.cpu().numpy(), r.table())
        assert np.array_equal(d.refs.cpu().numpy(), r.refs())
        codes, scales = ref.unpack(d.pool.cpu().numpy())
        for s, n in enumerate(r.lens):
            for b0 in range(0, n, ref.BLOCK):
                p, blk, m = r.rows[s][b0 // ref.PAGE], b0 % ref.PAGE // ref.BLOCK, min(16, n - b0)
                sl = slice(blk * 16, blk * 16 + m)
                got, want = ref.VALUES[codes[p, layers, sl]], ref.VALUES[r.codes[p, layers, sl]]
                assert np.array_equal(got, want, equal_nan=True), (s, b0)
                want = 2.0 ** r.exps[p, layers, blk].astype(float)
                assert np.array_equal(scales[p, layers, blk], want)


def normal(rng, shape, k_pe=5.0):
    x = rng.normal(size=shape).astype(np.float32)
    x[..., ref.C:] *= k_pe
    return ref.bf16(x)


# ---------------------------------------------------------------- rows

@pytest.mark.parametrize("layers, counts", [
    (1, [1]), (1, [16, 1, 0, 17]), (3, [15, 64, 65, 0, 2]), (2, [130]), (1, [3] * 70)])
def test_rows_in_and_out(layers, counts):
    rng = np.random.default_rng(sum(counts))
    n = len(counts)
    b = Both(sum(-(-c // 64) for c in counts) + 5, n, 4, layers)
    assert b.grow(counts)
    rows = normal(rng, (layers, sum(counts), ref.ROW))
    b.append(counts, rows)
    b.check()
    back = torch.full((layers, sum(counts) + 2, ref.ROW), 0x55, dtype=torch.int16, device="cuda")
    b.dev.read(back, starts(counts))
    got = ref.values(back.cpu().numpy())
    at = 0
    for s, c in enumerate(counts):
        for k in range(layers):
            assert np.array_equal(got[k, at: at + c], b.ref.values(s, k).astype(np.float32))
        at += c
    assert (back[:, at:] == 0x55).all()         # rows behind the last sequence


def test_blocks_grow_a_row_at_a_time():
    """Rows of growing and shrinking size, one or a few at a time, in two layers
    out of four: scales grow, older codes are rounded again."""
    rng = np.random.default_rng(3)
    b = Both(8, 2, 4, 4)
    for step in range(40):
        counts = [1, int(rng.integers(0, 4))]
        assert b.grow(counts)
        rows = normal(rng, (2, sum(counts), ref.ROW)) * np.float32(2.0) ** rng.integers(-6, 7)
        b.append(counts, rows, layer=1)
        if step % 8 == 7:
            b.check(layers=slice(1, 3))


def test_rows_of_every_kind_of_value():
    special = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 448.0, -448.0, 464.0, 1e-40, 3.0e38,
                        -3.0e38, 2.0**-126, 7.0, 2.0**-119, 0.4375], np.float32)
    rng = np.random.default_rng(4)
    b = Both(12, 5, 2, 1)
    assert b.grow([20, 16, 16, 33, 16])
    rows = normal(rng, (1, 101, ref.ROW))
    rows[0, :20] = ref.bf16(rng.choice(special, size=(20, ref.ROW)))
    rows[0, 20:36] = 0.0
    rows[0, 36:52] = np.inf                     # no finite value at all
    rows[0, 60, 5] = np.nan
    rows[0, 70, 500] = -np.inf
    rows[0, 85:101] = ref.bf16(rows[0, 85:101] * np.float32(1e-36))
    b.append([20, 16, 16, 33, 16], rows)
    b.check()


def test_rows_with_strides():
    """The decoder's own cache as rows: a slice of [layers][positions][576]."""
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(ref.bits(normal(rng, (3, 100, 584)))).cuda()
    view = wide[:, 11: 11 + 70, : ref.ROW]
    b = Both(4, 1, 2, 3)
    assert b.grow([70])
    b.ref.append(ref.values(view.cpu().numpy()), [0, 70])
    b.dev.append(view, starts([70]))
    b.check()
    out = torch.zeros((3, 90, 640), dtype=torch.int16, device="cuda")
    b.dev.read(out[:, 3:73, : ref.ROW], starts([70]))
    got = ref.values(out.cpu().numpy())
    for k in range(3):
        assert np.array_equal(got[k, 3:73, : ref.ROW], b.ref.values(0, k).astype(np.float32))
    assert (got[:, :3] == 0).all() and (got[:, 73:] == 0).all() and (got[..., ref.ROW:] == 0).all()


def test_rows_of_all_layers_together():
    """The layers of a position behind each other: [positions][layers][576]."""
    rng = np.random.default_rng(8)
    wide = torch.from_numpy(ref.bits(normal(rng, (40, 3, ref.ROW)))).cuda()
    b = Both(4, 2, 2, 3)
    assert b.grow([33, 7])
    b.ref.append(ref.values(wide.transpose(0, 1).cpu().numpy()), [0, 33, 40])
    b.dev.append(wide.transpose(0, 1), starts([33, 7]))
    b.check()
    out = torch.zeros_like(wide)
    b.dev.read(out.transpose(0, 1), starts([33, 7]))
    got = ref.values(out.cpu().numpy())
    for k in range(3):
        for s, (a, n) in enumerate(((0, 33), (33, 7))):
            assert np.array_equal(got[a:a + n, k], b.ref.values(s, k).astype(np.float32))


@pytest.mark.parametrize("heads, counts", [(16, [1, 1, 1]), (5, [1, 2, 1]), (16, [0, 1, 0]),
                                           (16, [40, 0, 3]), (3, [70, 1, 30])])
def test_rows_before_the_first_start(heads, counts):
    """A batch whose first rows belong to no sequence, and so do its last."""
    lens = [900, 64, 130]
    b, rng = filled(heads + sum(counts), lens, max_pages=20)
    lead, n = 7, sum(counts)
    at = i32(lead + np.concatenate([[0], np.cumsum(counts)]))
    q = ref.bf16(rng.normal(size=(n, heads, ref.ROW)) * 0.5)
    wide = torch.full((lead + n + 2, heads, ref.ROW), 0x7fff, dtype=torch.int16, device="cuda")
    wide[lead:lead + n] = to_dev(q)
    out = torch.full((lead + n + 2, heads, 512), 0x55, dtype=torch.int16, device="cuda")
    lse = torch.full((lead + n + 2, heads), 3.0, device="cuda")
    say(f"heads {heads} counts {counts}")
    for bound in (900, 0):
        b.dev.attend(wide, at, max_len=bound, out=out, lse=lse)
        compare(b, q, counts, out[lead:lead + n], lse[lead:lead + n])
        for t, v in ((out, 0x55), (lse, 3.0)):
            assert (t[:lead] == v).all() and (t[lead + n:] == v).all()
    rows = torch.full((1, lead + n + 2, ref.ROW), 0x55, dtype=torch.int16, device="cuda")
    b.dev.read(rows, at)
    assert (rows[:, :lead] == 0x55).all() and (rows[:, lead + n:] == 0x55).all()
    got, k = ref.values(rows.cpu().numpy())[0, lead:], 0
    for s, c in enumerate(counts):
        assert np.array_equal(got[k:k + c], b.ref.values(s)[lens[s] - c:].astype(np.float32))
        k += c
    assert b.dev.status() == 0


def test_starts_that_decrease():
    """Not allowed, and on the device: reported by the attention of few rows, which then
    does nothing, and within bounds everywhere."""
    lens = [300, 64, 130]
    b, rng = filled(77, lens)
    q = to_dev(ref.bf16(rng.normal(size=(6, 16, ref.ROW))))
    out = torch.full((6, 16, 512), 0x55, dtype=torch.int16, device="cuda")
    b.dev.attend(q, i32([0, 4, 1, 6]), out=out)
    assert (out == 0x55).all() and b.dev.status() == _lib.ABORT_POSITION
    big = to_dev(ref.bf16(rng.normal(size=(60, 16, ref.ROW))))
    rows = torch.zeros((1, 60, ref.ROW), dtype=torch.int16, device="cuda")
    for at in ([0, 50, 10, 60], [60, 0, 60, 0], [5, 5, 60, 1], [60, 40, 20, 0]):
        say(f"starts {at}")
        b.dev.attend(big, i32(at))
        b.dev.attend(big[:6], i32(at))
        b.dev.read(rows, i32(at))
        torch.cuda.synchronize()
    q = ref.bf16(rng.normal(size=(3, 16, ref.ROW)) * 0.5)
    out, lse = b.dev.attend(to_dev(q))
    compare(b, q, [1, 1, 1], out, lse)


def test_one_row_each_without_start():
    rng = np.random.default_rng(6)
    b = Both(6, 5, 1, 1)
    for _ in range(3):
        assert b.grow([1] * 5)
        rows = normal(rng, (1, 5, ref.ROW))
        b.ref.append(rows, range(6))
        b.dev.append(to_dev(rows[0]))
    b.check()


def test_more_rows_than_positions_and_lengths_outside_the_table():
    rng = np.random.default_rng(7)
    b = Both(4, 2, 2, 1)
    assert b.grow([3, 20])
    rows = normal(rng, (1, 30, ref.ROW))
    b.ref.append(rows, [0, 10, 30])             # 10 rows, 3 positions: the last three count
    b.dev.append(to_dev(rows), i32([0, 10, 30]))
    b.check(status=_lib.ABORT_POSITION)
    back = torch.full((30, ref.ROW), 7, dtype=torch.int16, device="cuda")
    b.dev.read(back, i32([0, 10, 30]))
    assert (back[:7] == 7).all()
    assert np.array_equal(ref.values(back[7:10].cpu().numpy()), b.ref.values(0).astype(np.float32))
    for bad in (129, -1, 2**31 - 1):
        c = Both(4, 1, 2, 1)
        c.dev.lens.fill_(bad)
        c.dev.append(to_dev(rows), i32([0, 30]))
        assert c.dev.status() == _lib.ABORT_POSITION and (c.dev.pool == 0xFF).all()


def test_pages_outside_the_pool_and_shared_pages_are_not_written():
    rng = np.random.default_rng(8)
    rows = normal(rng, (1, 5, ref.ROW))
    for page in (4, -1, 2**31 - 1, -2**31):
        c = paged.PagedCache.empty(4, 1, 2, 1)
        c.pool.fill_(0xFF)
        c.lens.fill_(5)
        c.table[0, 0] = page
        c.append(to_dev(rows), starts([5]))
        back = torch.full((5, ref.ROW), 9, dtype=torch.int16, device="cuda")
        c.read(back, starts([5]))
        assert c.status() == _lib.ABORT_BAD_PAGE
        assert (c.pool == 0xFF).all() and (back == 9).all()
    b = Both(4, 2, 2, 1)
    assert b.grow([5, 0])
    b.append([5, 0], rows)
    b.remap([0, 0])
    before = b.dev.pool.clone()
    b.dev.append(to_dev(rows), starts([5, 0]))
    assert b.dev.status() == _lib.ABORT_BAD_PAGE and torch.equal(b.dev.pool, before)


# ---------------------------------------------------------------- pages

@pytest.mark.parametrize("seed, n_pages, n_seqs, max_pages", [
    (1, 40, 6, 5), (2, 9, 4, 3), (3, 300, 40, 20), (4, 5000, 3, 7), (5, 64, 130, 2)])
def test_pages_over_many_steps(seed, n_pages, n_seqs, max_pages):
    """Forks, frees, growth that fails and growth that copies, and compaction, at
    random; rows written in between."""
    rng = np.random.default_rng(seed)
    b = Both(n_pages, n_seqs, max_pages, 2)
    status = 0
    for step in range(30):
        kind = rng.integers(0, 5)
        if kind == 0:
            parents = rng.integers(-1, n_seqs, n_seqs)
            b.remap(parents)
        elif kind == 1:
            b.compact()
        else:
            top = int(rng.choice([2, 20, 100]))
            new = rng.integers(0, top, n_seqs) * (rng.random(n_seqs) < 0.6)
            say(f"step {step}: grow")
            if not b.grow(new):
                status |= _lib.ABORT_NO_PAGE
                b.check(status)
                continue
            refs = b.ref.refs()
            for s in range(n_seqs):                 # append needs pages of one holder
                if new[s] and max(refs[p] for p in b.ref.rows[s]) > 1:
                    first = (b.ref.lens[s] - new[s]) // 64
                    assert max(refs[p] for p in b.ref.rows[s][first:]) == 1
            b.append(new, normal(rng, (2, int(new.sum()), ref.ROW)))
        b.check(status)


NONE = slice(0, 0)                                  # no rows are written here


def test_remap_and_grow_edges():
    b = Both(8, 3, 2, 1)
    assert b.grow([128, 0, 1])                      # a full row
    b.check(layers=NONE)
    b.remap([0, 0, 0])
    b.check(layers=NONE)
    assert b.grow([0, 0, 0])
    assert not b.grow([0, 0, 1])                    # no place in the table
    b.check(_lib.ABORT_NO_PAGE, NONE)
    b.remap([7, -5, 1])                             # no such sequences
    assert b.dev.status() == _lib.ABORT_NO_PAGE | _lib.ABORT_BAD_ID
    b.check(_lib.ABORT_NO_PAGE | _lib.ABORT_BAD_ID, NONE)
    for lens, new, bit in (([0, 0, 0], [1, -1, 0], _lib.ABORT_POSITION),
                           ([0, 129, 0], [1, 0, 0], _lib.ABORT_POSITION),
                           ([0, 0, -3], [1, 0, 0], _lib.ABORT_POSITION),
                           ([0, 0, 0], [1, 2**31 - 1, 0], _lib.ABORT_NO_PAGE)):
        c = paged.PagedCache.empty(8, 3, 2, 1)
        c.lens.copy_(i32(lens))
        c.grow(i32(new))
        assert c.status() == bit and (c.table == -1).all() and (c.refs == 0).all()
        assert c.lens.tolist() == lens
    c = paged.PagedCache.empty(8, 3, 2, 1)
    c.lens[1] = 5
    c.table[1, 0] = 8                               # the last page is not one of the pool
    c.grow(i32([1, 1, 1]))
    assert c.status() == _lib.ABORT_BAD_PAGE and c.lens.tolist() == [0, 5, 0]


def test_pages_of_many_sequences():
    """The largest number of rows, all of one shared page."""
    n = 1024
    b = Both(n + 40, n, 2, 1)
    assert b.grow([5] + [0] * (n - 1))
    b.append([5] + [0] * (n - 1), normal(np.random.default_rng(9), (1, 5, ref.ROW)))
    b.remap([0] * n)
    assert b.grow([1] * n)                          # all but one copy it
    b.append([1] * n, normal(np.random.default_rng(10), (1, n, ref.ROW)))
    b.check()
    b.remap(list(range(1, n)) + [-1])
    b.check()
    b.remap([n - 1 - i if i % 3 else -1 for i in range(n)])
    b.compact()
    b.check()


# ---------------------------------------------------------------- attention

def filled(seed, lens, n_layers=1, max_pages=None, spare=3, fill=0xFF):
    rng = np.random.default_rng(seed)
    pages = [-(-n // 64) for n in lens]
    b = Both(sum(pages) + spare, len(lens), max_pages or max(max(pages), 1), n_layers, fill)
    # pages in a shuffled order
    perm = iter(rng.permutation(sum(pages) + spare))
    table = np.full((len(lens), b.ref.max_pages), -1, np.int32)
    for s, n in enumerate(pages):
        b.ref.rows[s] = [int(next(perm)) for _ in range(n)]
        table[s, :n] = b.ref.rows[s]
    b.ref.lens = list(lens)
    b.dev.table.copy_(torch.from_numpy(table))
    b.dev.lens.copy_(i32(lens))
    b.dev.refs.copy_(torch.from_numpy(b.ref.refs()))
    if sum(lens):
        b.append(lens, normal(rng, (n_layers, sum(lens), ref.ROW)))
    return b, rng


def compare(b, q, counts, out, lse, layer=0, window=0, sinks=0, scale=SCALE):
    got, lse = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    at = 0
    for s, n in enumerate(counts):
        total = b.ref.lens[s]
        want, wl, tol, tl = ref.attend(b.ref.values(s, layer), q[at: at + n],
                                       range(total - n, total), scale, window, sinks)
        d = np.abs(got[at: at + n] - want)
        assert (d <= tol).all(), (s, np.nanmax(d - tol), np.unravel_index(np.argmax(d - tol), d.shape))
        gl = lse[at: at + n]
        none = np.isneginf(wl)
        assert np.array_equal(none, np.isneginf(gl)), s
        assert (np.abs(gl[~none] - wl[~none]) <= tl[~none]).all(), s
        at += n


CASES = [
    # lens, new per sequence, heads, window, sinks
    ([1], [1], 16, 0, 0), ([0, 1, 2], [1, 1, 1], 16, 0, 0), ([31, 32, 33, 63, 64, 65], [1] * 6, 16, 0, 0),
    ([127, 128, 129, 1000], [1] * 4, 16, 0, 0), ([700, 5], [1, 1], 1, 0, 0),
    ([300, 17], [2, 3], 5, 0, 0), ([130, 400], [1, 1], 40, 0, 0), ([200], [1], 128, 0, 0),
    ([3000, 1, 700], [1, 1, 1], 16, 0, 0), ([100] * 70, [1] * 70, 16, 0, 0),
    # a window, first positions, both, neither reaching
    ([1000, 40, 3], [1, 1, 1], 16, 64, 0), ([1000, 40, 3], [1, 1, 1], 16, 64, 4),
    ([1000, 100], [1, 1], 16, 1, 0), ([1000, 33], [1, 1], 16, 1, 1), ([500], [1], 16, 37, 100),
    ([500], [1], 16, 100, 500), ([2000], [3], 16, 333, 65), ([500], [1], 16, 500, 7),
    # prompts: from the first token, behind others, ragged, more tokens than positions
    ([5], [5], 16, 0, 0), ([64], [64], 16, 0, 0), ([100], [100], 16, 0, 0),
    ([200, 33, 1, 0, 90], [50, 33, 1, 0, 7], 16, 0, 0), ([70, 10], [70, 10], 3, 0, 0),
    ([150], [60], 24, 0, 0), ([300], [120], 16, 50, 0), ([300], [120], 16, 50, 5),
    ([400, 80], [33, 80], 16, 100, 20), ([3, 9], [5, 12], 16, 0, 0), ([0], [4], 16, 0, 0),
    ([90], [40], 128, 0, 0), ([1100], [17], 16, 0, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case):
    lens, counts, heads, window, sinks = CASES[case]
    b, rng = filled(100 + case, lens)
    q = ref.bf16(rng.normal(size=(sum(counts), heads, ref.ROW)) * 0.5)
    say(f"lens {lens[:6]} new {counts[:6]} heads {heads} window {window} sinks {sinks}")
    out, lse = b.dev.attend(to_dev(q), starts(counts), window=window, sinks=sinks,
                            max_len=max(lens))
    compare(b, q, counts, out, lse, window=window, sinks=sinks)
    assert b.dev.status() == 0
    # without a bound on the lengths, or one that is wrong, and from call to call
    for bound in (0, 1):
        o, e = b.dev.attend(to_dev(q), starts(counts), window=window, sinks=sinks, max_len=bound)
        compare(b, q, counts, o, e, window=window, sinks=sinks)
    o, e = b.dev.attend(to_dev(q), starts(counts), window=window, sinks=sinks, max_len=max(lens))
    assert torch.equal(o, out) and torch.equal(e, lse)


@pytest.mark.parametrize("lens, counts, heads, window, sinks", [
    # many parts of few rows, few parts of more rows, a bound far above the lengths,
    # sequences of which only one is divided, a window and first positions
    ([5000], [3], 16, 0, 0), ([1500], [40], 16, 0, 0), ([700, 3], [9, 3], 16, 0, 0),
    ([2600, 40, 0], [20, 33, 2], 16, 0, 0), ([3000], [12], 5, 1500, 70), ([2049], [70], 1, 0, 0)])
def test_attention_of_many_rows_in_parts(lens, counts, heads, window, sinks):
    b, rng = filled(sum(lens) + heads, lens, max_pages=-(-max(lens) // 64) + 50)
    q = ref.bf16(rng.normal(size=(sum(counts), heads, ref.ROW)) * 0.5)
    say(f"lens {lens} new {counts} heads {heads} window {window} sinks {sinks}")
    for bound in (max(lens), 0):
        out, lse = b.dev.attend(to_dev(q), starts(counts), window=window, sinks=sinks,
                                max_len=bound)
        compare(b, q, counts, out, lse, window=window, sinks=sinks)
    assert b.dev.status() == 0


@pytest.mark.parametrize("lens, heads, window", [
    ([9000] + [20] * 24, 16, 0), ([20] * 24 + [9000, 7], 5, 0), ([6000, 3000] + [1] * 20, 16, 0),
    ([9000] * 2 + [20] * 24, 16, 7000)])
def test_attention_of_one_long_sequence_among_short_ones(lens, heads, window):
    """Few parts a sequence in the mean, and hundreds for one of them."""
    b, rng = filled(len(lens) + heads, lens)
    n = len(lens)
    q = ref.bf16(rng.normal(size=(n, heads, ref.ROW)) * 0.5)
    say(f"{n} sequences up to {max(lens)} heads {heads} window {window}")
    out, lse = b.dev.attend(to_dev(q), window=window)
    compare(b, q, [1] * n, out, lse, window=window)
    assert b.dev.status() == 0


def test_attention_layers_strides_and_given_outputs():
    b, rng = filled(1, [90, 200], n_layers=3)
    q = ref.bf16(rng.normal(size=(5, 16, ref.ROW)))
    wide = torch.zeros((5, 20, ref.ROW), dtype=torch.int16, device="cuda")
    wide[:, 2:18] = to_dev(q)
    out = torch.full((7, 16, 512), 77, dtype=torch.int16, device="cuda")
    lse = torch.full((7, 16), 77.0, device="cuda")
    for layer in range(3):
        # two tokens of the first sequence, three of the second, two rows behind them
        more = torch.cat([wide, wide[:2]])[:, 2:18]
        o, e = b.dev.attend(more, i32([0, 2, 5]), layer=layer, out=out, lse=lse, scale=0.05)
        assert o is out and e is lse
        compare(b, q, [2, 3], out[:5], lse[:5], layer=layer, scale=0.05)
        assert (out[5:] == 77).all() and (lse[5:] == 77).all()
    o, e = b.dev.attend(wide[3:5, 2:18])             # one token of each sequence
    compare(b, q[3:5], [1, 1], o, e)


def test_attention_meets_no_nan_that_it_does_not_see():
    """A NaN row, an infinite one, and unwritten bytes (all NaN codes here): tokens
    that do not see the NaN are as if it were not there; those that do are NaN."""
    b, rng = filled(2, [100, 70])
    rows = normal(rng, (1, 8, ref.ROW))
    rows[0, 0] = np.nan                              # position 100 of sequence 0
    rows[0, 3, 7] = np.nan                           # one value of position 103
    rows[0, 5, 3] = np.inf
    assert b.grow([8, 0])                            # (in the page's second half)
    b.append([8, 0], rows)
    q = ref.bf16(rng.normal(size=(12, 16, ref.ROW)) * 0.5)
    out, lse = b.dev.attend(to_dev(q), starts([9, 3]))
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    assert np.isnan(got[1:9]).all() and np.isnan(gl[1:9]).all()
    clean = b.ref.values(0)
    want, wl, tol, tl = ref.attend(clean[:100], q[:1], [99], SCALE)
    assert (np.abs(got[:1] - want) <= tol).all() and (np.abs(gl[:1] - wl) <= tl).all()
    # with a window the last token sees 104 .. 107 only
    out, lse = b.dev.attend(to_dev(q), starts([9, 3]), window=4)
    got = ref.values(out.cpu().numpy())
    want, wl, tol, tl = ref.attend(clean, q[8:9], [107], SCALE, 4)
    assert (np.abs(got[8:9] - want) <= tol).all()
    compare(b, q[9:], [0, 3], torch.cat([out[9:]]), lse[9:], window=4)
    # a NaN or an infinity in q stays in its row
    q[10, 5, 100] = np.nan
    q[11, 2, 3] = np.inf
    out, _ = b.dev.attend(to_dev(q), starts([9, 3]), window=4)
    bad = np.isnan(ref.values(out.cpu().numpy()))[9:].all(-1)
    want = np.zeros((3, 16), bool)
    want[1, 5] = True
    with np.errstate(invalid="ignore"):             # all scores -infinity: nothing is summed
        want[2, 2] = not np.isneginf(q[11, 2].astype(float) @ b.ref.values(1)[-4:].T).all()
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("fill", [0x7E, 0xFE, 0x7B, 0x7F, 0x78, 0x80, 0x00])
@pytest.mark.parametrize("lens, counts", [([5, 100, 17], [1, 1, 1]), ([700], [1]), ([90, 3], [70, 3]),
                                          ([1500], [5])])
def test_attention_over_a_pool_that_holds_anything(fill, lens, counts):
    """Blocks with no position yet, and positions behind the last, of any bytes: the largest
    codes with the largest scale are infinite, and have weight 0."""
    b, rng = filled(fill, lens, fill=fill)
    q = ref.bf16(rng.normal(size=(sum(counts), 16, ref.ROW)) * 0.5)
    say(f"fill {fill:x} lens {lens} new {counts}")
    out, lse = b.dev.attend(to_dev(q), starts(counts))
    compare(b, q, counts, out, lse)


@pytest.mark.parametrize("n, new", [(40, 40), (130, 3), (700, 90)])
def test_attention_meets_no_infinity_that_it_does_not_see(n, new):
    """Values that the cache holds as infinite (beyond the largest bf16 after rounding),
    in positions that only the last token sees."""
    b = Both(16, 1, 16, 1)
    assert b.grow([n])
    rng = np.random.default_rng(n)
    rows = normal(rng, (1, n, ref.ROW))
    rows[0, n - 1, 3] = -ref.values(np.array([0x7f7f], np.int16))[0]
    rows[0, n - 1, 200] = ref.values(np.array([0x7f7f], np.int16))[0]
    b.append([n], rows)
    assert np.abs(b.ref.values(0)).max() > np.finfo(np.float32).max
    q = ref.bf16(rng.normal(size=(new, 16, ref.ROW)) * 0.5)
    out, lse = b.dev.attend(to_dev(q), starts([new]))
    got = ref.values(out.cpu().numpy())
    # (the largest scale is the whole block's: its other values are zeros now)
    want, wl, tol, tl = ref.attend(b.ref.values(0), q[:-1], range(n - new, n - 1), SCALE)
    assert (np.abs(got[:-1] - want) <= tol).all()
    assert (np.abs(lse.cpu().numpy()[:-1] - wl) <= tl).all()


def test_attention_extreme_scores():
    """Scores far apart and equal ones: one position takes all, or all the same."""
    b, rng = filled(3, [300])
    q = ref.bf16(rng.normal(size=(2, 16, ref.ROW)) * 60)
    out, lse = b.dev.attend(to_dev(q), starts([2]))
    compare(b, q, [2], out, lse)
    q[:] = 0
    out, lse = b.dev.attend(to_dev(q), starts([2]))
    compare(b, q, [2], out, lse)


def test_attention_with_bad_tables():
    """Pages outside the pool are not seen, lengths outside the table see nothing."""
    b, rng = filled(4, [200, 90], max_pages=4)
    q = ref.bf16(rng.normal(size=(2, 16, ref.ROW)) * 0.5)
    good, lse = b.dev.attend(to_dev(q))
    for page in (b.ref.n_pages, -1, 2**31 - 1):
        b.dev.table[0, 1] = page
        out, l2 = b.dev.attend(to_dev(q))
        assert b.dev.status() == _lib.ABORT_BAD_PAGE
        assert torch.equal(out[1], good[1])
        rows = b.ref.values(0)
        want, wl, tol, tl = ref.attend(np.concatenate([rows[:64], rows[128:]]), q[:1], [135], SCALE)
        assert (np.abs(ref.values(out[:1].cpu().numpy()) - want) <= tol).all()
        assert (np.abs(l2[:1].cpu().numpy() - wl) <= tl).all()
    b.dev.lens[0] = 257
    out, l2 = b.dev.attend(to_dev(q))
    assert b.dev.status() == _lib.ABORT_BAD_PAGE | _lib.ABORT_POSITION
    assert (out[0] == 0).all() and torch.isneginf(l2[0]).all() and torch.equal(out[1], good[1])


@pytest.mark.parametrize("tokens", [1, 3])
def test_attention_with_a_bad_page_far_into_a_share(tokens):
    """One workgroup walks the whole sequence (the bound says it is short), looks its
    pages up 64 steps at a time, and sees every page that is none."""
    n = 4500
    b, rng = filled(21 + tokens, [n])
    q = ref.bf16(rng.normal(size=(tokens, 16, ref.ROW)) * 0.5)
    rows = b.ref.values(0)
    table = b.dev.table.clone()
    for bad in (0, 29, 30, 31, 32, 33, 61, 62, 63, 64, 65, 69):
        say(f"tokens {tokens} page {bad}")
        b.dev.table.copy_(table)
        b.dev.table[0, bad] = b.dev.n_pages + 3
        out, lse = b.dev.attend(to_dev(q), starts([tokens]), max_len=1)
        good = np.concatenate([rows[:bad * 64], rows[bad * 64 + 64:]])
        want, wl, tol, tl = ref.attend(good, q, range(len(good) - tokens, len(good)), SCALE)
        assert (np.abs(ref.values(out.cpu().numpy()) - want) <= tol).all(), bad
        assert (np.abs(lse.cpu().numpy() - wl) <= tl).all(), bad
        assert b.dev.status() == _lib.ABORT_BAD_PAGE
        b.dev.workspace[:256].zero_()


def test_offsets_beyond_32_bits():
    """A pool of 5 GB: rows and attention in its last pages and layer."""
    layers, pages = 27, 5100
    c = paged.PagedCache.empty(pages, 1, 3, layers)
    r = ref.Cache(3, 1, 3, 1)
    r.rows, r.lens = [[0, 1, 2]], [150]
    c.table[0] = i32([pages - 1, 17, pages - 2])
    c.refs[pages - 1] = c.refs[17] = c.refs[pages - 2] = 1
    c.lens[0] = 150
    rng = np.random.default_rng(11)
    rows = normal(rng, (1, 150, ref.ROW))
    r.append(rows, [0, 150])
    c.append(to_dev(rows), starts([150]), layer=layers - 1)
    back = torch.zeros((150, ref.ROW), dtype=torch.int16, device="cuda")
    c.read(back, starts([150]), layer=layers - 1)
    assert np.array_equal(ref.values(back.cpu().numpy()), r.values(0).astype(np.float32))
    q = ref.bf16(rng.normal(size=(1, 16, ref.ROW)) * 0.5)
    out, lse = c.attend(to_dev(q), layer=layers - 1)
    want, wl, tol, tl = ref.attend(r.values(0), q, [149], SCALE)
    assert (np.abs(ref.values(out.cpu().numpy()) - want) <= tol).all()
    # and a copy of the last page, every layer
    wide = paged.PagedCache(c.pool, i32([[pages - 1, -1], [pages - 1, -1]]), i32([20, 20]),
                            torch.where(torch.arange(pages, device="cuda") == pages - 1, 2, 0).to(
                                torch.int32))
    wide.refs[: pages - 2] = 1                      # the free page is the last but one
    wide.grow(i32([1, 0]))
    assert wide.table.tolist() == [[pages - 2, -1], [pages - 1, -1]] and wide.status() == 0
    n = 2 * 9216
    assert torch.equal(c.pool[pages - 2, :, :n], c.pool[pages - 1, :, :n])
    assert int(wide.compact().item()) == pages


def test_on_another_stream_and_in_a_graph():
    """A step (fork, grow, append, attend) captured and replayed between eager calls
    on the same cache, and a call on a stream of its own."""
    b, rng = filled(5, [70, 130, 10], max_pages=6, spare=40)
    c = b.dev
    saved = [t.clone() for t in (c.pool, c.table, c.lens, c.refs)]
    rows, q = to_dev(normal(rng, (3, ref.ROW))), to_dev(ref.bf16(rng.normal(size=(3, 16, ref.ROW))))
    parents, one = i32([1, 1, 0]), i32([1, 1, 1])
    out = torch.zeros((3, 16, 512), dtype=torch.int16, device="cuda")
    lse = torch.zeros((3, 16), device="cuda")

    def step():
        c.remap(parents)
        c.grow(one)
        c.append(rows)
        c.attend(q, max_len=300, out=out, lse=lse)

    def state():
        return [t.clone() for t in (c.table, c.lens, c.refs, out, lse)]

    def back():
        for t, s in zip((c.pool, c.table, c.lens, c.refs), saved):
            t.copy_(s)

    want = []
    for _ in range(2):
        step()
        want.append(state())
    back()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    for rep in range(4):
        back()
        for k in range(2):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(state(), want[k])), (rep, k)
        back()
        for k in range(2):                          # the same eagerly, in between
            step()
            assert all(torch.equal(x, y) for x, y in zip(state(), want[k])), (rep, k)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        o2, l2 = c.attend(q, max_len=300)
    o3, l3 = c.attend(q, max_len=300, stream=s)
    s.synchronize()
    assert torch.equal(o2, out) and torch.equal(o3, out) and torch.equal(l3, lse)


def test_refused_tensors():
    b, rng = filled(6, [20, 20])
    c = b.dev
    rows = torch.zeros((2, ref.ROW), dtype=torch.int16, device="cuda")
    q = torch.zeros((2, 16, ref.ROW), dtype=torch.int16, device="cuda")
    for f in (lambda: c.append(rows.float()), lambda: c.append(rows[:, :-1]),
              lambda: c.append(rows[:1]), lambda: c.append(rows.cpu()),
              lambda: c.append(rows, i32([0, 2])), lambda: c.append(rows, i32([0, 1, 2]).long()),
              lambda: c.append(rows.T), lambda: c.remap(i32([0])), lambda: c.grow(i32([1, 1, 1])),
              lambda: c.attend(q.float()), lambda: c.attend(q[:1]),
              lambda: c.attend(q, out=q), lambda: c.attend(q, lse=torch.zeros(2, 16)),
              lambda: c.attend(q[..., :512]), lambda: c.attend(q.transpose(0, 1)[:2]),
              lambda: paged.PagedCache(c.pool[..., :-1], c.table, c.lens, c.refs),
              lambda: paged.PagedCache(c.pool, c.table, c.lens[:1], c.refs),
              lambda: paged.PagedCache(c.pool.cpu(), c.table, c.lens, c.refs)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: c.append(rows, layer=1), lambda: c.read(rows, layer=-1),
              lambda: c.attend(q, layer=1), lambda: c.attend(q, window=-1),
              lambda: c.attend(q, scale=0.0),
              lambda: c.append(torch.zeros((2, 580), dtype=torch.int16, device="cuda")[:, 4:])):
        with pytest.raises(_lib.FleetMoeError):
            f()
    assert c.attend(q[:0], i32([0, 0, 0]))[0].shape == (0, 16, 512)
    c.append(rows[:0], i32([0, 0, 0]))
    assert c.status() == 0

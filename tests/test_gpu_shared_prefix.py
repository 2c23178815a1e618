"""GPU: attention of sequences that share their first pages (paged.SharedPrefix) against
every sequence's attention in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, paged  # noqa: E402
from test_gpu_paged import SCALE, Both, compare, filled, i32, normal, say, starts, to_dev  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


LONG = 9000
FEW = 16                # sequences behind LONG positions: pages for more than 2,048 units of 16 rows
both_heights = pytest.mark.parametrize("tall", [False, True])


def forked(seed, prefixes, own, layers=1, fill=0xFF, extra=(), room=0, tall=0):
    """Groups of sequences: group g has len(own[g]) of them behind prefixes[g] common positions,
    with own[g][i] positions of its own; then, with `tall`, that many behind LONG positions, so
    that units have 64 rows and not 16; then the sequences `extra` by themselves; `room` pages
    more for each."""
    if tall:
        prefixes, own = [*prefixes, LONG], [*own, [1] * tall]
    rng = np.random.default_rng(seed)
    n = sum(len(o) for o in own) + len(extra)
    top = max([p + max(o) for p, o in zip(prefixes, own)] + [*extra, 1])
    pages = sum(-(-p // 64) + sum(-(-x // 64) + 2 for x in o) for p, o in zip(prefixes, own))
    b = Both(pages + sum(-(-x // 64) for x in extra) + 3 + n * room, n, -(-top // 64) + 1 + room, layers,
             fill)
    counts, parents, first = [0] * n, list(range(n)), []
    at = 0
    for p, o in zip(prefixes, own):
        counts[at] = p
        first.append(at)
        for i in range(len(o)):
            parents[at + i] = at
        at += len(o)
    groups = first + [at]
    assert b.grow(counts)
    if sum(counts):
        b.append(counts, normal(rng, (layers, sum(counts), ref.ROW)))
    b.remap(parents)
    counts = [x for o in own for x in o] + list(extra)
    assert b.grow(counts)
    if sum(counts):
        b.append(counts, normal(rng, (layers, sum(counts), ref.ROW)))
    return b, rng, groups


def plan(b, groups, tokens, heads=16):
    p = paged.SharedPrefix(b.dev, i32(groups), max(tokens, 1), heads)
    p.update()
    return p


def query(rng, n, heads=16):
    return ref.bf16(rng.normal(size=(n, heads, ref.ROW)) * 0.5)


CASES = [
    # prefixes, own positions, new tokens a sequence, heads, extra sequences
    ([64], [[1, 1]], 1, 16, []), ([640], [[1, 40, 63, 64, 65, 100]], 1, 16, []),
    ([63], [[5, 9]], 1, 16, []), ([1], [[1, 1, 1]], 1, 16, []), ([200], [[1]], 1, 16, []),
    ([700, 64, 130], [[3, 9], [200], [1, 2, 3, 4, 5]], 1, 16, [5, 300]),
    ([1000], [[7] * 17], 1, 16, []), ([300], [[20, 30, 40]], 5, 16, [9]),
    ([2000], [[70, 3, 400]], 3, 5, []), ([500], [[4, 4]], 2, 128, []), ([500], [[1] * 9], 1, 1, []),
    ([130, 130], [[90, 90], [200, 70]], 70, 16, [80]), ([4500], [[3, 5]], 1, 16, []),
    ([64] * 30, [[2, 3]] * 30, 1, 16, []),
]


def compare_first(b, q, counts, out, lse, n, layer=0):
    """The first n sequences' rows."""
    r = sum(counts[:n])
    compare(b, q[:r], counts[:n] + [0] * (len(counts) - n), out[:r], lse[:r], layer)


@both_heights
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_every_sequence(case, tall):
    prefixes, own, new, heads, extra = CASES[case]
    say(f"case {CASES[case]} {tall}")
    b, rng, groups = forked(case, prefixes, own, extra=extra,
                            tall=-(-16 * 16 // (new * heads)) if tall else 0)
    if tall:
        prefixes = [*prefixes, LONG]
    n = len(b.ref.lens)
    counts = [min(new, x) for x in b.ref.lens]
    q = query(rng, sum(counts), heads)
    p = plan(b, groups, sum(counts), heads)
    want = [min(b.ref.lens[a: z]) // 64 if z - a > 1 else 0 for a, z in zip(groups, groups[1:])]
    want = [min(w, pre // 64) for w, pre in zip(want, prefixes)]
    assert p.pages.tolist() == want
    out, lse = p.attend(to_dev(q), starts(counts))
    compare_first(b, q, counts, out, lse, sum(map(len, own)) + 1 if tall else n)
    if new == 1 and all(c == 1 for c in counts):
        o2, l2 = p.attend(to_dev(q))
        assert torch.equal(o2, out) and torch.equal(l2, lse)
    assert b.dev.status() == 0


def test_many_sequences_and_few():
    """The largest cache: 1,024 sequences, all behind one page; then groups of many sizes, some of
    nothing, some without tokens."""
    n = 1024
    b, rng, groups = forked(50, [64], [[1] * n])
    q = query(rng, n, 2)
    out, lse = plan(b, groups, n, 2).attend(to_dev(q))
    compare(b, q, [1] * n, out, lse)
    b, rng, groups = forked(51, [300, 129], [[3, 4, 5, 6], [9, 8]], extra=[0, 50])
    b.remap([0, 1, -1, 3, 4, 5, 6, 7])
    p = plan(b, [0, 0, 4, 4, 6, 8], 30)
    assert p.pages.tolist() == [0, 4, 0, 2, 0]
    for counts in ([1, 0, 0, 1, 1, 1, 0, 1], [0, 2, 0, 0, 0, 3, 0, 0], [0] * 7 + [1],
                   [3, 1, 4, 1, 5, 2, 6, 5]):
        say(f"counts {counts}")
        q = query(rng, sum(counts))
        out, lse = p.attend(to_dev(q), starts(counts))
        compare(b, q, counts, out, lse)


@pytest.mark.parametrize("heads", [1, 16])
def test_more_sequences_than_threads(heads):
    """700 sequences in three groups and by themselves, units of 16 rows and of 64; a thread
    finds the work of two of them."""
    sizes, extra = [300, 200, 170], [500] * 30
    b, rng, groups = forked(62, [700, 129, 64], [[5 + i % 90 for i in range(n)] for n in sizes],
                            extra=extra)
    n = sum(sizes) + len(extra)
    counts = [1 + (i % 50 == 0) for i in range(n)]
    at = np.concatenate([[0], np.cumsum(counts)])
    q = query(rng, sum(counts), heads)
    p = plan(b, groups, sum(counts), heads)
    assert p.pages.tolist() == [10, 2, 1]
    out, lse = p.attend(to_dev(q), starts(counts))
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    for s in [0, 1, 50, 298, 299, 300, 301, 499, 500, 511, 512, 513, 669, 670, 671, 698, 699]:
        total, rows = b.ref.lens[s], slice(at[s], at[s + 1])
        want, wl, tol, tl = ref.attend(b.ref.values(s), q[rows], range(total - counts[s], total), SCALE)
        assert (np.abs(got[rows] - want) <= tol).all() and (np.abs(gl[rows] - wl) <= tl).all(), s
    assert b.dev.status() == 0


@both_heights
def test_tokens_inside_the_common_pages(tall):
    """Sequences that agree to the end: tokens stand in common pages and see them up to their own
    position; more tokens than positions see nothing."""
    more = [1] * FEW * tall
    b, rng, groups = forked(52, [256], [[0, 0, 0]], tall=len(more))
    p = plan(b, groups, 400)
    assert p.pages.tolist() == [4, LONG // 64][: 1 + tall]
    for counts in ([1, 1, 1], [1, 200, 70], [256, 10, 0], [3, 260, 1]):
        say(f"counts {counts}")
        counts = counts + more
        q = query(rng, sum(counts))
        out, lse = p.attend(to_dev(q), starts(counts))
        compare_first(b, q, counts, out, lse, 3)
    assert b.dev.status() == 0


@both_heights
@pytest.mark.parametrize("empty", [[0], [1], [3], [0, 1], [1, 2], [0, 1, 2, 3]])
def test_sequences_that_begin_after_the_update(empty, tall):
    """Sequences of a group that hold nothing at update() grow later, into pages of their own."""
    b, rng, groups = forked(61, [200], [[3, 9, 5, 70]], room=2, tall=FEW * tall)
    n = 4 + FEW * tall
    b.remap([-1 if s in empty else s for s in range(n)])
    p = plan(b, groups, 3 * n)
    assert p.pages[0] == (3 if len(empty) < 4 else 0)
    for new in (1, 2):
        counts = [new if s in empty else 1 for s in range(n)]
        assert b.grow(counts)
        b.append(counts, normal(rng, (1, sum(counts), ref.ROW)))
        q = query(rng, sum(counts))
        out, lse = p.attend(to_dev(q), starts(counts))
        compare_first(b, q, counts, out, lse, 4)
    assert b.dev.status() == 0


@both_heights
def test_steps_of_beams(tall):
    """remap, update, grow, append, attend over several steps; a plan that a remap has made stale
    is right too, and so is one that was never updated."""
    b, rng, groups = forked(53, [200, 70], [[3] * 4, [5] * 3], layers=2, room=4, tall=FEW * tall)
    n = 7 + FEW * tall
    more = list(range(7, n))
    p = plan(b, groups, n)
    old = plan(b, groups, n)
    new = paged.SharedPrefix(b.dev, i32(groups), n, 16)
    for step in range(6):
        parents = [*rng.integers(0, 4, 4), *(4 + rng.integers(0, 3, 3))]
        if step == 3:                           # the groups' sequences change places
            parents = [4, 5, 6, 0, 0, 1, 2]
        b.remap([int(x) for x in parents] + more)
        b.remap(list(range(n)))
        p.update()
        assert b.grow([1 + step * 9] * n)
        b.append([1 + step * 9] * n, normal(rng, (2, n * (1 + step * 9), ref.ROW)))
        q = query(rng, n)
        for layer in range(2):
            for x in (p, old, new):
                out, lse = x.attend(to_dev(q), layer=layer)
                compare_first(b, q, [1] * n, out, lse, 7, layer)
    if step:
        b.compact()                             # moves pages, for all rows alike
        out, lse = p.attend(to_dev(q))
        compare_first(b, q, [1] * n, out, lse, 7)
    assert b.dev.status() == 0


def test_groups_out_of_order_and_starts_that_decrease():
    b, rng, groups = forked(54, [200], [[3, 4, 5]])
    q = query(rng, 3)
    for bad in ([0, 4], [-1, 3], [2, 1, 3], [0, 3, 2]):
        p = plan(b, bad, 3)
        assert p.pages.tolist() == [0] * (len(bad) - 1)
        assert b.dev.status() == _lib.ABORT_POSITION
        b.dev.clear_status()
        out, lse = p.attend(to_dev(q))
        compare(b, q, [1] * 3, out, lse)
    p = plan(b, groups, 3)
    out = torch.full((3, 16, 512), 7, dtype=torch.int16, device="cuda")
    lse = torch.full((3, 16), 7.0, device="cuda")
    p.attend(to_dev(q), i32([0, 2, 1, 3]), out=out, lse=lse)
    assert b.dev.status() == _lib.ABORT_POSITION and (out == 7).all() and (lse == 7).all()
    b.dev.clear_status()
    # rows before the first start and behind the last are nobody's
    p.attend(to_dev(q), i32([1, 1, 2, 2]), out=out, lse=lse)
    assert (out[[0, 2]] == 7).all() and (lse[[0, 2]] == 7).all()
    compare(b, q[1:2], [0, 1, 0], out[1:2], lse[1:2])


@both_heights
def test_bad_tables(tall):
    """A page outside the pool ends what is shared, and is not seen; a length outside the table
    sees nothing."""
    b, rng, groups = forked(55, [400], [[3, 9, 5]], tall=FEW * tall)
    n = 3 + FEW * tall
    q = query(rng, n)
    good, gl = plan(b, groups, n).attend(to_dev(q))
    table = b.dev.table.clone()
    for page in (b.ref.n_pages, -1, 2**31 - 1):
        b.dev.table[:3, 2] = page
        p = plan(b, groups, n)
        assert p.pages[0] == 2
        out, lse = p.attend(to_dev(q))
        assert b.dev.status() == _lib.ABORT_BAD_PAGE
        b.dev.clear_status()
        for s in range(3):
            rows = b.ref.values(s)
            rows = np.concatenate([rows[:128], rows[192:]])
            want, wl, tol, tl = ref.attend(rows, q[s: s + 1], [len(rows) - 1], SCALE)
            assert (np.abs(ref.values(out[s: s + 1].cpu().numpy()) - want) <= tol).all()
            assert (np.abs(lse[s: s + 1].cpu().numpy() - wl) <= tl).all()
    b.dev.table.copy_(table)
    b.dev.table[1, 1] = b.dev.table[1, 0]       # one differs in the second page
    p = plan(b, groups, n)
    assert p.pages[0] == 1
    b.dev.table.copy_(table)
    p = plan(b, groups, n)
    b.dev.lens[1] = 64 * b.dev.max_pages + 1
    out, lse = p.attend(to_dev(q))
    assert b.dev.status() == _lib.ABORT_POSITION
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()
    # (the parts are other ones now, so are the sums' last bits)
    compare_first(b, q, [1] * n, out, lse, 1)
    b.dev.clear_status()
    b.dev.lens[1] = -1
    p.update()
    assert p.pages[0] == 6                      # of those that hold anything


@pytest.mark.parametrize("fill", [0x7E, 0x7F, 0xFF, 0x78])
@both_heights
def test_a_pool_that_holds_anything(fill, tall):
    b, rng, groups = forked(56, [130, 700], [[1, 40, 64], [9, 9]], fill=fill, tall=FEW * tall)
    n = 5 + FEW * tall
    q = query(rng, n)
    out, lse = plan(b, groups, n).attend(to_dev(q))
    compare_first(b, q, [1] * n, out, lse, 5)


@both_heights
def test_what_is_not_finite_and_extreme_scores(tall):
    """A NaN in the common pages reaches all, one in a sequence's own that alone; scores far apart
    and equal ones."""
    b, rng, groups = forked(57, [200], [[30, 40, 50]], tall=FEW * tall)
    n = 3 + FEW * tall
    q = query(rng, n)
    p = plan(b, groups, n)
    for mag in (60.0, 0.0):
        out, lse = p.attend(to_dev(ref.bf16(q * mag)))
        compare_first(b, ref.bf16(q * mag), [1] * n, out, lse, 3)
    good, gl = p.attend(to_dev(q))
    last = int(b.dev.table[1, 3])
    b.dev.pool[last, 0, 9216 + 5 * 16] = 0x7F               # sequence 1, positions 208 on
    out, lse = p.attend(to_dev(q))
    assert torch.equal(out[0], good[0]) and torch.equal(lse[0], gl[0])
    assert torch.equal(out[2:], good[2:]) and torch.equal(lse[2:], gl[2:])
    assert np.isnan(ref.values(out[1].cpu().numpy())).all()
    bad = query(rng, n)
    bad[2, 5, 100] = np.nan
    out, _ = p.attend(to_dev(bad))
    nan = np.isnan(ref.values(out.cpu().numpy()))
    assert nan[1].all() and nan[2, 5].all() and not nan[0].any() and not np.delete(nan[2], 5, 0).any()
    assert not nan[3:].any()
    b.dev.pool[int(b.dev.table[0, 1]), 0, 3] = 0xFF          # common
    out, _ = p.attend(to_dev(q))
    nan = np.isnan(ref.values(out.cpu().numpy()))
    assert nan[:3].all() and not nan[3:].any()


def test_strides_and_given_outputs():
    b, rng, groups = forked(58, [300], [[3, 4]], layers=3)
    q = query(rng, 4)
    wide = torch.zeros((4, 16 * 576 + 64), dtype=torch.int16, device="cuda")
    v = wide[:, 8: 8 + 16 * 576].view(4, 16, 576)
    v.copy_(to_dev(q))
    p = plan(b, groups, 9)
    out = torch.zeros((4, 16, 512), dtype=torch.int16, device="cuda")
    lse = torch.zeros((4, 16), device="cuda")
    got = p.attend(v, starts([1, 3]), layer=2, scale=0.05, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    compare(b, q, [1, 3], out, lse, 2, scale=0.05)
    # a plan for more tokens and heads serves fewer, of any heads
    h = query(rng, 18, 7)
    o, l = p.attend(to_dev(h), starts([9, 9]))
    compare(b, h, [9, 9], o, l)
    with pytest.raises(ValueError):
        p.attend(to_dev(query(rng, 10)), starts([9, 1]))


def test_on_another_stream_and_in_a_graph():
    """Two plans on one cache, captured steps replayed between eager calls."""
    b, rng, groups = forked(59, [500, 100], [[70, 10, 30], [5, 6]])
    c, q = b.dev, to_dev(query(rng, 5))
    p, other = plan(b, groups, 5), plan(b, [0, 2], 5)
    saved = [t.clone() for t in (c.pool, c.table, c.lens, c.refs)]
    rows, parents = to_dev(normal(rng, (5, ref.ROW))), i32([1, 1, 0, 4, 4])
    out = torch.zeros((5, 16, 512), dtype=torch.int16, device="cuda")
    lse = torch.zeros((5, 16), device="cuda")

    def step():
        c.remap(parents)
        p.update()
        c.grow(i32_one)
        c.append(rows)
        p.attend(q, out=out, lse=lse)

    def back():
        for t, s in zip((c.pool, c.table, c.lens, c.refs), saved):
            t.copy_(s)

    i32_one = i32([1] * 5)
    step()
    want = [out.clone(), lse.clone(), p.pages.clone()]
    back()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    for rep in range(3):
        back()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((out, lse, p.pages), want)), rep
        back()
        other.update()
        other.attend(q)
        step()
        assert all(torch.equal(x, y) for x, y in zip((out, lse, p.pages), want)), rep
    torch.cuda.synchronize()
    o2, l2 = p.attend(q, stream=s)
    s.synchronize()
    assert torch.equal(o2, out) and torch.equal(l2, lse)


def test_refused():
    b, rng = filled(60, [20, 20])
    c, g = b.dev, i32([0, 2])
    q = torch.zeros((2, 16, ref.ROW), dtype=torch.int16, device="cuda")
    p = paged.SharedPrefix(c, g, 2, 16)
    for f in (lambda: paged.SharedPrefix(c, g.cpu(), 2, 16), lambda: paged.SharedPrefix(c, g[:1], 2, 16),
              lambda: paged.SharedPrefix(c, g.long(), 2, 16),
              lambda: paged.SharedPrefix(c, i32([0, 1, 1, 2]), 2, 16),
              lambda: paged.SharedPrefix(c, g, 0, 16), lambda: paged.SharedPrefix(c, g, 2, 129),
              lambda: paged.SharedPrefix(c, g, 1 << 20, 16), lambda: p.attend(q.float()),
              lambda: p.attend(q[:1]), lambda: p.attend(q.cpu()), lambda: p.attend(q, i32([0, 2])),
              lambda: p.attend(q, out=q), lambda: p.attend(q[..., :512])):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: p.attend(q, layer=1), lambda: p.attend(q, layer=-1), lambda: p.attend(q, scale=0.0)):
        with pytest.raises(_lib.FleetMoeError):
            f()
    assert p.attend(q[:0], i32([0, 0, 0]))[0].shape == (0, 16, 512)
    assert c.status() == 0

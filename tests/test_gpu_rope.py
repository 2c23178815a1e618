"""GPU: the rotation of heads by their positions (ops.Rotary, PagedCache.rotate) against
the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, ops, paged, rope  # noqa: E402

BITS, F32 = torch.int16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def dev(x, dtype):
    x = np.ascontiguousarray(x, np.float32)
    return torch.from_numpy(x if dtype == F32 else ref.bits(ref.bf16(x))).cuda()


def host(t):
    a = t.cpu().contiguous()
    return a.numpy().astype(np.float64) if a.dtype == F32 else ref.values(a.numpy()).astype(np.float64)


def turned(x, pos, freqs, at, halves_in, halves_out, mag=1.0):
    """(want, |a| + |b| of every value's pair): x [tokens][heads][width] in 64 bits."""
    d = 2 * len(freqs)
    ang = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs, np.float64)
    c, s = mag * np.cos(ang)[:, None], mag * np.sin(ang)[:, None]
    v = x[..., at: at + d]
    a, b = (v[..., : d // 2], v[..., d // 2:]) if halves_in else (v[..., 0::2], v[..., 1::2])
    first, second, size = a * c - b * s, b * c + a * s, np.abs(a) + np.abs(b)
    want, both = x.copy(), np.zeros_like(x)
    for to, f, g in ((want, first, second), (both, size, size)):
        if halves_out:
            to[..., at: at + d] = np.concatenate([f, g], -1)
        else:
            to[..., at: at + d: 2], to[..., at + 1: at + d: 2] = f, g
    return want, abs(mag) * both


def check(got, want, both, f32):
    """The angle is off by pi * 2^-25 where it is rounded to fp32 and by 2^-24 before that
    (positions up to 2^27 radians), cos and sin by 2^-23 more: 2^-21.5 of |a| + |b|, with the
    products' roundings 2^-21; the result by half a step."""
    half = 2.0**-24 if f32 else 2.0**-8
    d = np.abs(host(got) - want)
    tol = half * np.abs(want) + 2.0**-21 * both
    assert (d <= tol).all(), (np.nanmax(d - tol), np.unravel_index(np.argmax(d - tol), d.shape))


CASES = [
    # tokens, heads, width, at, dim
    (1, 16, 64, 0, 64), (1, 1, 2, 0, 2), (5, 16, 192, 128, 64), (3, 7, 40, 4, 34),
    (9, 3, 31, 5, 6), (2, 128, 64, 0, 64), (700, 16, 192, 128, 64), (1300, 5, 27, 1, 22),
    (40, 2, 1200, 100, 1024), (1, 4000, 8, 0, 8),
]


@pytest.mark.parametrize("tokens, heads, width, at, dim", CASES)
@pytest.mark.parametrize("dtype", [BITS, F32])
@pytest.mark.parametrize("hin, hout", [(False, True), (False, False), (True, True), (True, False)])
def test_against_the_formula(tokens, heads, width, at, dim, dtype, hin, hout):
    rng = np.random.default_rng(tokens + heads + width)
    freqs = 10000.0 ** (-np.arange(dim // 2) / max(dim // 2, 1))
    pos = rng.integers(0, 5000, tokens)
    x = dev(rng.normal(size=(tokens, heads, width)), dtype)
    r = ops.Rotary(freqs, 1.25, hin, hout)
    got = r.rotate(x, i32(pos), at=at)
    want, both = turned(host(x), pos, freqs, at, hin, hout, 1.25)
    check(got, want, both, dtype == F32)
    if hin == hout:                                       # in place
        r.rotate(x, i32(pos), out=x, at=at)
        assert torch.equal(x, got)


def test_positions_far_out_and_below_zero():
    f = rope.frequencies().astype(np.float64)
    pos = np.array([0, 1, -1, -4096, 1 << 20, (1 << 27) - 1, -(1 << 27)])
    x = dev(np.random.default_rng(1).normal(size=(7, 2, 64)), F32)
    r = ops.Rotary(f, rope.magnitude())
    want, both = turned(host(x), pos, f, 0, False, True)
    check(r.rotate(x, i32(pos)), want, both, True)
    # there and back again: the rotation by -p of what p left
    back = ops.Rotary(f, halves_in=True, halves_out=False)
    y = back.rotate(r.rotate(x, i32(pos)), i32(-pos))
    assert (np.abs(host(y) - host(x)) <= 2 * 2.0**-21 * 2 * np.abs(host(x)).max()).all()
    # far beyond: finite, and the length of every pair is kept
    far = r.rotate(x, i32([2**31 - 1] * 6 + [-2**31]))
    n = lambda v, a, b: v[..., a] ** 2 + v[..., b] ** 2  # noqa: E731
    assert np.allclose(n(host(far), slice(0, 32), slice(32, 64)),
                       n(host(x), slice(0, 64, 2), slice(1, 64, 2)), rtol=1e-5)


def test_like_the_decoders_tables():
    """The frequencies are the tables': equal up to what fp32 angles lose, half a step of 2^-24
    of the angle."""
    cos, sin = rope.yarn_tables(4096)
    pos = np.array([0, 1, 17, 1000, 4095])
    x = dev(np.random.default_rng(2).normal(size=(5, 3, 64)), F32)
    v = host(x)
    v = np.concatenate([v[..., 0::2], v[..., 1::2]], -1)
    rot = np.concatenate([-v[..., 32:], v[..., :32]], -1)
    want = v * cos[pos][:, None] + rot * sin[pos][:, None]
    got = host(ops.Rotary(rope.frequencies(), rope.magnitude()).rotate(x, i32(pos)))
    assert (np.abs(got - want) <= (4095 * 2.0**-24 + 2.0**-20) * (np.abs(v) + np.abs(rot))).all()


def test_parts_of_wider_rows():
    """Queries out of the projection's rows and into the absorbed ones; any strides; heads before
    tokens; one row for all."""
    rng = np.random.default_rng(3)
    f = rope.frequencies().astype(np.float64)
    r, pos = ops.Rotary(f), np.array([5, 900, 3])
    row = dev(rng.normal(size=(3, 16 * 192 + 576)), BITS)
    q = torch.full((3, 16, 576), 7, dtype=BITS, device="cuda")
    x = row[:, : 16 * 192].view(3, 16, 192)[..., 128:]
    r.rotate(x, i32(pos), out=q[..., 512:])
    want, both = turned(host(x), pos, f, 0, False, True)
    check(q[..., 512:], want, both, False)
    assert (q[..., :512] == 7).all()
    for lo in (1, 3):                                     # not in fours
        x = row[:, lo: lo + 16 * 192].view(3, 16, 192)[..., 100:170]
        out = torch.zeros((16, 3, 71), dtype=BITS, device="cuda").transpose(0, 1)[..., 1:]
        r.rotate(x, i32(pos), out=out, at=4)
        want, both = turned(host(x), pos, f, 4, False, True)
        check(out, want, both, False)
    one = row[:1, :64].view(1, 1, 64).expand(3, 4, 64)
    want, both = turned(host(one), pos, f, 0, False, True)
    check(r.rotate(one, i32(pos)), want, both, False)


@pytest.mark.parametrize("dtype", [BITS, F32])
@pytest.mark.parametrize("tokens", [2, 3000])
@pytest.mark.parametrize("width, at", [(192, 128), (83, 7), (100, 31), (64 + 12, 0)])
def test_other_values_keep_their_bits(dtype, tokens, width, at):
    """What is not rotated is copied, whatever its bits are."""
    ints = torch.int16 if dtype == BITS else torch.int32
    info = torch.iinfo(ints)
    x = torch.randint(info.min, info.max + 1, (tokens, 5, width), device="cuda", dtype=ints)
    rest = torch.ones(width, dtype=torch.bool, device="cuda")
    rest[at: at + 64] = False
    r, p = ops.Rotary(rope.frequencies()), i32(np.arange(tokens))
    got = r.rotate(x.view(dtype), p, at=at).view(ints)
    assert torch.equal(got[..., rest], x[..., rest])


@pytest.mark.parametrize("dtype, tokens, width, at", [(F32, 5500, 192, 128), (BITS, 11_000, 193, 3)])
def test_more_than_the_caches_hold(dtype, tokens, width, at):
    """Results of 64 MB and more, of 16 heads, and in place."""
    rng = np.random.default_rng(9)
    f = rope.frequencies().astype(np.float64)
    x = dev(rng.normal(size=(tokens, 16, width)).astype(np.float32), dtype)
    pos = rng.integers(0, 1 << 20, tokens)
    want, both = turned(host(x), pos, f, at, False, False)
    r = ops.Rotary(f, halves_out=False)
    got = r.rotate(x, i32(pos), at=at)
    check(got, want, both, dtype == F32)
    assert torch.equal(got[..., :at], x[..., :at]) and torch.equal(got[..., at + 64:], x[..., at + 64:])
    assert r.rotate(x, i32(pos), out=x, at=at) is x and torch.equal(x, got)


@pytest.mark.parametrize("tokens", [3, 900])
def test_positions_of_the_cache(tokens):
    rng = np.random.default_rng(tokens)
    f = rope.frequencies().astype(np.float64)
    r = ops.Rotary(f)
    counts = [0, tokens - 1, 0, 1, 0]
    lens = [7, tokens + 40, 0, 64, 3]
    c = paged.PagedCache.empty(4, 5, 20, 1)
    c.lens.copy_(i32(lens))
    x = dev(rng.normal(size=(tokens + 2, 4, 64)), BITS)
    start = i32(1 + np.concatenate([[0], np.cumsum(counts)]))       # the first and last are nobody's
    out = torch.full((tokens + 2, 4, 64), 9, dtype=BITS, device="cuda")
    c.rotate(r, x, start, out=out)
    pos = np.concatenate([np.arange(lens[1] - counts[1], lens[1]), [63]])
    want, both = turned(host(x)[1:-1], pos, f, 0, False, True)
    check(out[1:-1], want, both, False)
    assert (out[0] == 9).all() and (out[-1] == 9).all() and c.status() == 0
    # one token each, and a length outside the table, or none
    c.lens.copy_(i32([5, 64 * 20 + 1, 0, 64, -3]))
    out.fill_(9)
    c.rotate(r, x[:5], out=out[:5])
    assert c.status() == _lib.ABORT_POSITION
    want, both = turned(host(x)[[0, 3]], [4, 63], f, 0, False, True)
    check(out[[0, 3]], want, both, False)
    assert (out[[1, 2, 4]] == 9).all()


def test_many_sequences():
    n = 1024
    rng = np.random.default_rng(8)
    f = rope.frequencies().astype(np.float64)
    lens = rng.integers(3, 60, n)
    counts = rng.integers(0, 3, n)
    c = paged.PagedCache.empty(1, n, 1, 1)
    c.lens.copy_(i32(lens))
    total = int(counts.sum())
    x = dev(rng.normal(size=(total, 2, 64)), BITS)
    out = c.rotate(ops.Rotary(f), x, i32(np.concatenate([[0], np.cumsum(counts)])))
    pos = np.concatenate([np.arange(l - k, l) for l, k in zip(lens, counts)])
    want, both = turned(host(x), pos, f, 0, False, True)
    check(out, want, both, False)


def test_refused_and_empty():
    r = ops.Rotary(rope.frequencies())
    x = torch.zeros((4, 2, 64), dtype=BITS, device="cuda")
    p = i32([1, 2, 3, 4])
    c = paged.PagedCache.empty(1, 4, 1, 1)
    for f in (lambda: r.rotate(x.cpu(), p), lambda: r.rotate(x.half(), p),
              lambda: r.rotate(x[0], p), lambda: r.rotate(x.transpose(1, 2), p),
              lambda: r.rotate(x, p[:3]), lambda: r.rotate(x, p.long()),
              lambda: r.rotate(x, p, out=x.float()), lambda: r.rotate(x, p, out=x[:, :1]),
              lambda: c.rotate(r, x[:3]), lambda: c.rotate(r, x, p),
              lambda: ops.Rotary([]), lambda: ops.Rotary([[1.0]])):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: r.rotate(x, p, out=x), lambda: r.rotate(x, p, at=2),
              lambda: r.rotate(x[..., :62], p), lambda: r.rotate(x, p, at=-1),
              lambda: r.rotate(x, p, out=x[:1].expand(4, 2, 64))):
        with pytest.raises(_lib.FleetMoeError):
            f()
    assert r.rotate(x[:0], p[:0]).shape == (0, 2, 64)
    assert c.rotate(r, x[:0], i32([0] * 5)).shape == (0, 2, 64)


def test_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(9)
    r, pos = ops.Rotary(rope.frequencies()), i32([3, 77, 1000])
    x = dev(rng.normal(size=(3, 16, 64)), BITS)
    want = r.rotate(x, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = r.rotate(x, pos, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        r.rotate(x, pos, out=out)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        out.zero_()
        pos.add_(i)                                       # the graph reads the positions of now
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r.rotate(x, pos))

"""GPU: the paged cache's calls at the ends of the ranges they accept."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, ops, paged  # noqa: E402


def say(msg: str) -> None:
    print(f"[gpu] {msg}", flush=True)


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def cache_of(seed, n, k_pe=5.0):
    """One sequence of n positions on the device, and its values in 64 bits."""
    rng = np.random.default_rng(seed)
    pages = -(-n // 64)
    dev, want = paged.PagedCache.empty(pages, 1, pages, 1), ref.Cache(pages, 1, pages, 1)
    dev.pool.fill_(0xFF)
    rows = rng.normal(size=(1, n, ref.ROW)).astype(np.float32)
    rows[..., ref.C:] *= k_pe
    rows = ref.bf16(rows)
    assert want.grow([n])
    want.append(rows, [0, n])
    dev.grow(i32([n]))
    dev.append(torch.from_numpy(ref.bits(rows)).cuda(), i32([0, n]))
    return dev, want.values(0), rng


def test_attention_of_more_than_2_24_rows():
    """One head and 2^24 + 200 tokens, of which the last 130 stand at positions: the row
    of a token there is beyond 2^24."""
    n, tokens = 130, (1 << 24) + 200
    dev, rows, rng = cache_of(1, n)
    q = torch.zeros((tokens, 1, ref.ROW), dtype=torch.int16, device="cuda")
    last = ref.bf16(rng.normal(size=(n, 1, ref.ROW)) * 0.5)
    q[-n:] = torch.from_numpy(ref.bits(last)).cuda()
    say(f"{tokens} tokens")
    out, lse = dev.attend(q, i32([0, tokens]))
    assert dev.status() == 0
    assert not out[:-n].any() and torch.isneginf(lse[:-n]).all()
    want, wl, tol, tl = ref.attend(rows, last, range(n), paged.SOFTMAX_SCALE)
    assert (np.abs(ref.values(out[-n:].cpu().numpy()) - want) <= tol).all()
    assert (np.abs(lse[-n:].cpu().numpy() - wl) <= tl).all()


@pytest.mark.parametrize("scale", [1e-45, 1e-39, 1e-38, 1.6e-38, 1e-37, 1e30])
@pytest.mark.parametrize("n, new", [(100, 1), (5000, 1), (100, 40), (1500, 40)])
def test_attention_with_scales_at_both_ends(scale, n, new):
    """Few and many rows, whole and in parts. Small scales weigh all positions alike; with
    the largest the queries are as small."""
    dev, rows, rng = cache_of(n + new, n)
    q = ref.bf16(rng.normal(size=(new, 16, ref.ROW)) * (0.5 if scale < 1 else 0.05 / scale))
    say(f"scale {scale} {n} positions {new} tokens")
    out, lse = dev.attend(torch.from_numpy(ref.bits(q)).cuda(), i32([0, new]), scale=scale)
    want, wl, tol, tl = ref.attend(rows, q, range(n - new, n), float(np.float32(scale)))
    assert (np.abs(ref.values(out.cpu().numpy()) - want) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - wl) <= tl).all()
    assert dev.status() == 0


def test_attention_with_the_largest_scale():
    dev, rows, rng = cache_of(5, 70)
    q = torch.zeros((1, 16, ref.ROW), dtype=torch.int16, device="cuda")
    out, lse = dev.attend(q, scale=2.35e38)
    want, wl, tol, tl = ref.attend(rows, np.zeros((1, 16, ref.ROW)), [69], 1.0)
    assert (np.abs(ref.values(out.cpu().numpy()) - want) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - wl) <= tl).all()


@pytest.mark.parametrize("n, new", [(100, 2), (5000, 2), (100, 40), (1500, 40)])
def test_attention_with_scores_beyond_fp32(n, new):
    """Finite products q . row that are infinite times the scale: +infinity makes its token
    and head NaN, and no other."""
    dev, rows, rng = cache_of(n * new, n)
    scale = 1e20
    q = ref.bf16(rng.normal(size=(new, 16, ref.ROW)) * 0.05 / scale)
    q[0, ::2] = ref.bf16(rng.normal(size=(8, ref.ROW)) * 1e19)
    say(f"{n} positions {new} tokens")
    z = q[0, ::2].astype(float) @ rows[:n - new + 1].T
    top = float(np.finfo(np.float32).max)
    assert (np.abs(z) < top).all() and (scale * z.max(1) > 2 * top).all()
    out, lse = dev.attend(torch.from_numpy(ref.bits(q)).cuda(), i32([0, new]), scale=scale)
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    assert np.isnan(got[0, ::2]).all() and np.isnan(gl[0, ::2]).all()
    with np.errstate(invalid="ignore", over="ignore"):
        want, wl, tol, tl = ref.attend(rows, q, range(n - new, n), scale)
    for at in (np.s_[0, 1::2], np.s_[1:]):
        assert (np.abs(got[at] - want[at]) <= tol[at]).all()
        assert (np.abs(gl[at] - wl[at]) <= tl[at]).all()


@pytest.mark.parametrize("n, new", [(1, 1), (64, 1), (200, 1), (5000, 1), (64, 40), (1500, 40)])
def test_attention_with_scores_of_minus_infinity(n, new):
    """The first 64 positions have finite products that are -infinity times the scale, the
    others 0: the first have no weight, and where there is nothing else the output is 0."""
    rng = np.random.default_rng(n)
    rows = np.zeros((1, n, ref.ROW), np.float32)
    rows[0, :64, :256] = ref.bf16(np.abs(rng.normal(size=(min(n, 64), 256))) + 1)
    rows[0, 64:, 256:512] = ref.bf16(rng.normal(size=(max(n - 64, 0), 256)))
    pages = -(-n // 64)
    dev, want = paged.PagedCache.empty(pages, 1, pages, 1), ref.Cache(pages, 1, pages, 1)
    assert want.grow([n])
    want.append(rows, [0, n])
    dev.grow(i32([n]))
    dev.append(torch.from_numpy(ref.bits(rows)).cuda(), i32([0, n]))
    q = np.zeros((new, 16, ref.ROW), np.float32)
    q[..., :256] = -1e19
    say(f"{n} positions {new} tokens")
    out, lse = dev.attend(torch.from_numpy(ref.bits(ref.bf16(q))).cuda(), i32([0, new]), scale=1e20)
    if n <= 64:
        assert not out.any() and torch.isneginf(lse).all()
        return
    o, e, tol, tl = ref.attend(want.values(0)[64:], q, range(n - 64 - new, n - 64), 1.0)
    assert (np.abs(ref.values(out.cpu().numpy()) - o) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - e) <= tl).all()


BIG = 2**32                         # whose low 32 bits are zero


def test_arguments_beyond_32_bits():
    """A window, first positions or a bound beyond any length are as good as that; a layer
    is none."""
    dev, rows, rng = cache_of(7, 150)
    q = ref.bf16(rng.normal(size=(1, 16, ref.ROW)) * 0.5)
    dq = torch.from_numpy(ref.bits(q)).cuda()
    want, wl, tol, tl = ref.attend(rows, q, [149], paged.SOFTMAX_SCALE)
    for kw in (dict(window=BIG + 5), dict(window=5, sinks=BIG), dict(max_len=BIG + 1)):
        out, lse = dev.attend(dq, **kw)
        assert (np.abs(ref.values(out.cpu().numpy()) - want) <= tol).all(), kw
        assert (np.abs(lse.cpu().numpy() - wl) <= tl).all(), kw
    row = torch.zeros((1, ref.ROW), dtype=torch.int16, device="cuda")
    for f in (lambda: dev.attend(dq, layer=BIG), lambda: dev.attend(dq, layer=-BIG),
              lambda: dev.attend(dq, window=-BIG), lambda: dev.attend(dq, sinks=-BIG),
              lambda: dev.attend(dq, max_len=-BIG), lambda: dev.append(row, layer=BIG),
              lambda: dev.append(row, layer=-BIG), lambda: dev.read(row, layer=BIG)):
        with pytest.raises(_lib.FleetMoeError):
            f()


def test_beam_arguments_beyond_32_bits():
    for bad in ((BIG + 1, 2, 2, 100), (1, BIG + 2, 2, 100), (1, 2, BIG + 2, 100), (1, 2, 2, BIG + 100)):
        with pytest.raises(ValueError):
            ops.BeamSelector(*bad)
    with pytest.raises(ValueError):
        ops.BeamSelector(1, 2, 2, 100, eos=BIG)
    select = ops.BeamSelector(1, 2, 2, 100, eos=3 - BIG)            # no such token
    logits = torch.zeros((2, 100), device="cuda")
    logits[1, 3] = 20.0
    got = select.select(logits, torch.tensor([[-1.0, -2.0]], device="cuda"),
                        torch.tensor([[1, 0]], dtype=torch.uint8, device="cuda"))
    assert got["tokens"].tolist() == [[-1, 3]] and got["finished"].tolist() == [[1, 0]]

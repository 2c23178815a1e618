"""GPU: the paged cache's calls at the ends of the ranges they accept."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import paged  # noqa: E402


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

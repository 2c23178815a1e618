"""GPU: the paged cache with as many sequences as it takes, 1,024: attention over ragged
ones, rows out, and a reordering in a graph."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import paged  # noqa: E402

N = 1024


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def cache(gpu):
    """Lengths from 0 to 300, three in four of them short."""
    rng = np.random.default_rng(1)
    lens = np.where(rng.random(N) < 0.75, rng.integers(0, 40, N), rng.integers(0, 301, N))
    lens[[0, 63, 64, 500, 1023]] = [0, 1, 300, 65, 64]
    pages = int((-(-lens // 64)).sum())
    dev, want = paged.PagedCache.empty(pages + 3, N, 6, 1), ref.Cache(pages + 3, N, 6, 1)
    dev.pool.fill_(0xFF)
    rows = ref.bf16(rng.normal(size=(1, lens.sum(), ref.ROW)))
    at = np.concatenate([[0], np.cumsum(lens)])
    assert want.grow(lens.tolist())
    want.append(rows, at)
    dev.grow(i32(lens))
    dev.append(torch.from_numpy(ref.bits(rows)).cuda(), i32(at))
    return dev, want, lens


@pytest.mark.parametrize("kind, heads, window, sinks", [
    ("one", 16, 0, 0), ("one", 5, 30, 2), ("some", 16, 0, 0), ("prompts", 16, 0, 0),
    ("prompts", 3, 50, 4)])
def test_attention(cache, kind, heads, window, sinks):
    """A token each; none, one or three; and prompts among single tokens."""
    dev, want, lens = cache
    rng = np.random.default_rng(heads + window)
    counts = np.ones(N, int)
    if kind == "some":
        counts = rng.choice([0, 1, 3], N)
    elif kind == "prompts":
        counts = np.where(rng.random(N) < 0.05, lens, counts)
    at = np.concatenate([[0], np.cumsum(counts)])
    q = ref.bf16(rng.normal(size=(at[-1], heads, ref.ROW)) * 0.5)
    print(f"[gpu] {at[-1]} tokens, {heads} heads", flush=True)
    out, lse = dev.attend(torch.from_numpy(ref.bits(q)).cuda(), i32(at), window=window, sinks=sinks)
    assert dev.status() == 0
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    for s in range(N):
        a, z = at[s], at[s + 1]
        w, wl, tol, tl = ref.attend(want.values(s), q[a:z], range(lens[s] - (z - a), lens[s]),
                                    paged.SOFTMAX_SCALE, window, sinks)
        assert (np.abs(got[a:z] - w) <= tol).all(), s
        none = np.isneginf(wl)
        assert np.array_equal(none, np.isneginf(gl[a:z])), s
        assert (np.abs(gl[a:z][~none] - wl[~none]) <= tl[~none]).all(), s


def test_rows(cache):
    dev, want, lens = cache
    at = np.concatenate([[0], np.cumsum(lens)])
    back = torch.zeros((1, at[-1], ref.ROW), dtype=torch.int16, device="cuda")
    dev.read(back, i32(at))
    got = ref.values(back.cpu().numpy())[0]
    for s in range(N):
        assert np.array_equal(got[at[s]:at[s + 1]], want.values(s).astype(np.float32)), s


def test_a_reordering_in_a_graph(cache):
    """The table of 1,024 rows takes more LDS than a launch has by itself, which has to be
    asked for while a graph is captured too."""
    dev, want, lens = cache
    saved = [t.clone() for t in (dev.table, dev.lens, dev.refs)]
    parents = i32(np.roll(np.arange(N), 7))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        dev.remap(parents)
    torch.cuda.current_stream().wait_stream(s)
    for k in range(1, 4):
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(dev.lens.cpu().numpy(), np.roll(lens, 7 * k))
        assert np.array_equal(dev.table.cpu().numpy(), np.roll(want.table(), 7 * k, 0))
        assert torch.equal(dev.refs, saved[2])
    for t, x in zip((dev.table, dev.lens, dev.refs), saved):
        t.copy_(x)
    assert dev.status() == 0

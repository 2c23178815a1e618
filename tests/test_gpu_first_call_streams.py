"""GPU: the first call on an object may be on another stream than the one it was made on, with
work of that one still to come."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import ops, paged, rope  # noqa: E402
from test_gpu_paged import compare, i32, normal, starts, to_dev  # noqa: E402
from test_gpu_shared_prefix import forked, query  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def other():
    """Another stream, where what the tests made so far is ready."""
    torch.cuda.synchronize()
    return torch.cuda.Stream()


def busy():
    """Some 50 ms of work on the current stream."""
    torch.cuda._sleep(100_000_000)


@pytest.mark.parametrize("where", ["host", "device"])
def test_rotary(where):
    f = rope.frequencies().astype(np.float64)
    x, pos = torch.randn((5, 2, 64), device="cuda"), i32([0, 1, 70, 4000, -3])
    want = ops.Rotary(f).rotate(x, pos)
    given = f if where == "host" else torch.from_numpy(f).cuda()
    s = other()
    busy()
    got = ops.Rotary(given).rotate(x, pos, stream=s)
    s.synchronize()
    assert torch.equal(got, want)


def test_shared_prefix():
    b, rng, groups = forked(90, [640], [[30, 7, 100]])
    q, at = query(rng, 3), i32(groups)
    dev = to_dev(q)
    s = other()
    busy()
    p = paged.SharedPrefix(b.dev, at, 3, 16)
    out, lse = p.attend(dev, stream=s)                    # (without a plan)
    pages = p.update(stream=s)
    out2, lse2 = p.attend(dev, stream=s)
    s.synchronize()
    torch.cuda.synchronize()
    assert pages.tolist() == [10]
    compare(b, q, [1] * 3, out, lse)
    compare(b, q, [1] * 3, out2, lse2)


def test_paged_cache():
    rng = np.random.default_rng(91)
    rows = normal(rng, (1, 70, ref.ROW))
    dev, n = to_dev(rows), i32([70])
    want = paged.PagedCache.empty(3, 1, 3, 1)
    want.grow(n)
    want.append(dev, starts([70]))
    back, start = torch.zeros((70, ref.ROW), dtype=torch.int16, device="cuda"), starts([70])
    want.read(back, start)
    got = torch.zeros_like(back)
    s = other()
    busy()
    c = paged.PagedCache.empty(3, 1, 3, 1)
    c.grow(n, stream=s)
    c.append(dev, start, stream=s)
    c.read(got, start, stream=s)
    s.synchronize()
    torch.cuda.synchronize()
    assert c.status() == 0 and torch.equal(got, back)

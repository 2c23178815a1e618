"""GPU: the attention's weights with few rows keep 16 bits: sums in which they nearly
cancel, that weights rounded to bf16 would lose."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import paged  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n, new, heads, window, sinks", [
    (2, 1, 16, 0, 0), (64, 1, 16, 0, 0), (6000, 1, 16, 0, 0), (300, 2, 16, 0, 0), (500, 1, 32, 0, 0),
    (900, 1, 5, 200, 4)])
def test_weights_that_nearly_cancel(n, new, heads, window, sinks):
    """c is 1 at even positions and -1 at odd ones, whose scores are lower by 11/8192: the
    weights are 1 and 0.99866, which is nearest to 1 in bf16, and the output 0.00067."""
    rows = np.zeros((1, n, ref.ROW), np.float32)
    rows[0, 0::2, :ref.C], rows[0, 1::2, :ref.C] = 1.0, -1.0
    rows[0, 1::2, ref.C] = -11 / 8192
    pages = -(-n // 64)
    dev, want = paged.PagedCache.empty(pages, 1, pages, 1), ref.Cache(pages, 1, pages, 1)
    assert want.grow([n])
    want.append(rows, [0, n])
    dev.grow(i32([n]))
    dev.append(torch.from_numpy(ref.bits(rows)).cuda(), i32([0, n]))
    assert np.array_equal(want.values(0), rows[0])
    q = np.zeros((new, heads, ref.ROW), np.float32)
    q[..., ref.C] = 1.0
    print(f"[gpu] {n} positions, {new} tokens of {heads} heads", flush=True)
    out, lse = dev.attend(torch.from_numpy(ref.bits(q)).cuda(), i32([0, new]), scale=1.0,
                          window=window, sinks=sinks)
    o, e, _, tl = ref.attend(want.values(0), q, range(n - new, n), 1.0, window, sinks)
    # half a bf16 step of the output; half a step of 16 bits of each weight, in numerator and
    # denominator, and 2^-20 for exponentials and sums, of sum w |c| = 1
    tol = 2.0**-8 * np.abs(o) + 2 * 2.0**-16 + 2.0**-20
    assert (np.abs(ref.values(out.cpu().numpy()) - o) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - e) <= tl).all()

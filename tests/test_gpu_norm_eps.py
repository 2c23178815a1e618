"""GPU: ops.residual_norm at both ends of the eps that it accepts, with rows on both sides of
where the squares are taken again of smaller values."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from fleet_moe import ops  # noqa: E402
from test_gpu_residual_norm import BITS, F32, check, dev  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("eps", [1e-30, 1e-6, 1.0, 1e28, 1e29, 1e30])
@pytest.mark.parametrize("width", [64, 2048, 8193, 32768])
@pytest.mark.parametrize("dtype", [BITS, F32])
def test_eps_at_both_ends(dtype, width, eps):
    """Row i has a sum of squares of about 2^(119 + i / 2), from below 2^120, where one pass
    ends, to above, and then of the size of eps and far from it."""
    rng = np.random.default_rng(width)
    size = [2.0 ** ((119 + i / 2) / 2) / width ** 0.5 for i in range(6)]
    size += [eps**0.5, 1e-3 * eps**0.5, 1e3 * eps**0.5, 1e-18, 1e18]
    v = rng.normal(size=(len(size), width))
    v *= np.array(size)[:, None] / np.sqrt((v * v).mean(-1, keepdims=True))
    x, norm = dev(v, dtype), dev(1 + 0.1 * rng.normal(size=width), BITS)
    print(f"[gpu] width {width}, eps {eps}", flush=True)
    check(x, None, norm, eps=eps, got=ops.residual_norm(x, None, norm, eps=eps))
    # and the norm of y, beside a residual of its own
    post = dev(0.5 + 0.1 * rng.normal(size=width), BITS)
    r = dev(rng.normal(size=v.shape), F32)
    check(r, x, norm, post, eps=eps, got=ops.residual_norm(r, x, norm, post_norm=post, eps=eps))


def test_a_large_row_with_a_large_eps():
    """32,768 equal values of 2^52.5 and a little with eps = 1e30: h is 0.988, not 1."""
    for v in (0.999 * 2.0**52.5, 1.001 * 2.0**52.5):
        x = torch.full((1, 32768), v, device="cuda")
        _, h = ops.residual_norm(x, eps=1e30)
        want = v / np.sqrt(v * v + 1e30)
        got = h.cpu().view(torch.bfloat16).double()
        # half a step of bf16, and 2^-18 for sum, root and product in 32 bits
        assert ((got - want).abs() <= (2.0**-8 + 2.0**-18) * want).all(), v
        assert want < 0.99

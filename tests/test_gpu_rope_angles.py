"""GPU: how good the angles of a rotation are: cosine and sine themselves, of fp32 pairs
(1, 0)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from fleet_moe import ops  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("far", [1 << 10, 1 << 20, 1 << 27])
def test_angles_to_a_24th_bit(far):
    """An angle is good to 2^-24 up to 2^27 radians, in every direction: the turns of a position
    and their product with it are off by 2^-51.7 of the angle, 2^-24.7, and what is left of a quarter
    turn, in half turns at most 1/4, by pi * 2^-27 where it is rounded to fp32. Cosine and sine of
    it may be off by two units of their last place, 2^-22 of them. (Frequencies are powers of two:
    a position times one is exact here, too.)"""
    rng = np.random.default_rng(far)
    freqs = 2.0 ** -np.arange(32)
    pos = np.concatenate([rng.integers(-far, far + 1, 20000), [0, 1, -1, far, -far]])
    x = torch.zeros((len(pos), 1, 64), device="cuda")
    x[..., :32] = 1.0
    print(f"[gpu] positions up to {far}", flush=True)
    got = ops.Rotary(freqs, halves_in=True).rotate(x, torch.from_numpy(pos.astype(np.int32)).cuda())
    got = got.cpu().numpy().astype(np.float64)[:, 0]
    ang = pos[:, None] * freqs
    c, s = np.cos(ang), np.sin(ang)
    for name, g, want, other in (("cos", got[:, :32], c, s), ("sin", got[:, 32:], s, c)):
        d = np.abs(g - want) - (2.0**-24 * np.abs(other) + 2.0**-22 * np.abs(want) + 2.0**-48)
        i = np.unravel_index(np.argmax(d), d.shape)
        assert d[i] <= 0, (name, pos[i[0]], i[1], d[i], want[i])

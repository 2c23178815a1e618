"""GPU: the weights of shared attention (paged.SharedPrefix) have 16 bits whatever the units'
height, so a sequence's result does not lose bits as other requests join a call."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from test_gpu_paged import SCALE, say, starts, to_dev  # noqa: E402
from test_gpu_shared_limits import of_rows  # noqa: E402
from test_gpu_shared_prefix import FEW, forked, plan, query  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# (units of 64 rows where those of 16 would be more than 2,048 pages: the first four)
@pytest.mark.parametrize("n, common, own, new, heads", [
    (40, 9000, 64, 1, 16), (20, 9000, 200, 2, 16), (6, 9000, 100, 5, 32), (20, 64 * 180, 5, 1, 25),
    (3, 640, 100, 4, 16)])
def test_weights_that_nearly_cancel(n, common, own, new, heads):
    """c is 1 at even positions and -1 at odd ones, whose scores are lower by 11/8192: the
    weights are 1 and 0.99866, which is nearest to 1 in bf16, and the output 0.00067."""
    rows = np.zeros((common + own, ref.ROW), np.float32)
    rows[0::2, :ref.C], rows[1::2, :ref.C] = 1.0, -1.0
    rows[1::2, ref.C] = -11 / 8192
    b, p = of_rows(n, rows[:common], rows[common:], new, heads)
    assert p.update()[0] == common // 64
    q = np.zeros((n * new, heads, ref.ROW), np.float32)
    q[..., ref.C] = 1.0
    say(f"{n} sequences, {common} + {own}, {new} tokens of {heads} heads")
    out, lse = p.attend(to_dev(ref.bf16(q)), starts([new] * n), scale=1.0)
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    o, e, _, tl = ref.attend(rows.astype(float), q[:new], range(len(rows) - new, len(rows)), 1.0)
    # half a bf16 step of the output; half a step of 16 bits of each weight, in numerator and
    # denominator, and 2^-20 for exponentials and sums, of sum w |c| = 1
    tol = 2.0**-8 * np.abs(o) + 2 * 2.0**-16 + 2.0**-20
    for s in range(n):
        assert (np.abs(got[s * new: (s + 1) * new] - o) <= tol).all(), s
        assert (np.abs(gl[s * new: (s + 1) * new] - e) <= tl).all(), s


@pytest.mark.parametrize("new, own", [(1, [30, 64, 200]), (5, [20, 7, 300])])
@pytest.mark.parametrize("tall", [False, True])
def test_the_same_bits_beside_other_requests(tall, new, own):
    """Scores that move the reference, in common pages and own ones: within what weights of 16
    bits leave, alone and with requests beside them that make the units 64 rows high."""
    b, rng, groups = forked(80 + new, [700], [own], tall=FEW * tall)
    counts = [new] * 3 + [1] * FEW * tall
    q = ref.bf16(3 * query(rng, sum(counts)))
    out, lse = plan(b, groups, sum(counts)).attend(to_dev(q), starts(counts))
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    for s in range(3):
        total, at = b.ref.lens[s], slice(s * new, (s + 1) * new)
        rows = b.ref.values(s)
        o, e, tol, tl = ref.attend(rows, q[at], range(total - new, total), SCALE)
        # ref.attend's tolerance with 2^-16 for each weight in numerator and denominator
        # where it has 2^-8: less (2^-7 - 2^-15) of sum w |c|
        a = np.zeros_like(o)
        for i in range(new):
            k = rows[: total - new + 1 + i].astype(np.float64)
            z = SCALE * q[at][i].astype(np.float64) @ k.T
            w = np.exp(z - z.max(1, keepdims=True))
            a[i] = (w / w.sum(1, keepdims=True)) @ np.abs(k[:, :ref.C])
        tol = tol - (2.0**-7 - 2.0**-15) * a
        d = np.abs(got[at] - o)
        assert (d <= tol).all(), (s, (d - tol).max())
        assert (np.abs(gl[at] - e) <= tl).all(), s
    assert b.dev.status() == 0

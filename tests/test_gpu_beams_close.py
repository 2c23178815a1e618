"""GPU: beam selection where candidates of different beams are nearer to each other than
sums in 32 bits tell apart: the order is that of 64 bits (paged_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import ops  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def log_p(x):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def compare(logits, scores, finished, n_out, eos=-1):
    """No two candidates of different beams may be closer than what 64-bit sums in another
    order can change, so that the order is one. A log sum: 100 additions of a thread, 6 of
    a wave, 16 of the waves and an exponential on one side, numpy's 16 + 10 and an
    exponential on the other, half a step each: 150 * 2^-53. A score: three roundings of
    half a step of the largest term on either side. For both candidates twice that:
    300 * 2^-53 + 12 * 2^-53 * |score|."""
    groups, beams, vocab = logits.shape
    assert vocab <= 102400
    gap = 300 * 2.0**-53 + 12 * 2.0**-53 * max(float(np.abs(scores[np.isfinite(scores)]).max()), 30)
    best = ref.beam_select(logits, scores, finished, n_out, eos)
    for rows in ref.beam_select(logits, scores, finished, n_out + 1, eos):
        for a, b in zip(rows, rows[1:]):
            assert a[1] == b[1] or a[0] - b[0] > gap or a[0] == b[0] == -np.inf
    select = ops.BeamSelector(groups, beams, n_out, vocab, eos=eos)
    got = select.select(torch.from_numpy(logits).cuda().view(groups * beams, vocab),
                        torch.from_numpy(scores).cuda(),
                        torch.from_numpy(finished.astype(np.uint8)).cuda())
    for g in range(groups):
        assert got["parents"][g].tolist() == [r[1] for r in best[g]], g
        assert got["tokens"][g].tolist() == [r[2] for r in best[g]], g
        assert got["finished"][g].tolist() == [r[3] for r in best[g]], g
        # half a step of fp32 and 2^-18, the log sum's
        want = np.array([r[0] for r in best[g]])
        assert (np.abs(got["scores"][g].cpu().numpy() - want)
                <= 2.0**-24 * np.abs(want) + 2.0**-18).all()


@pytest.mark.parametrize("beams, n_out, vocab", [(2, 2, 700), (4, 4, 5000), (8, 16, 9000),
                                                 (64, 64, 300), (3, 1, 40000)])
def test_best_tokens_of_beams_that_nearly_agree(beams, n_out, vocab):
    """Every beam's best token has the same score up to the rounding of `scores` to fp32."""
    rng = np.random.default_rng(beams + vocab)
    groups = 32
    logits = (3 * rng.normal(size=(groups, beams, vocab))).astype(np.float32)
    top = log_p(logits).max(-1)
    scores = (-9.0 - rng.random((groups, 1)) - top).astype(np.float32)
    compare(logits, scores, np.zeros((groups, beams), bool), n_out)


def test_the_last_place_between_two_beams():
    """The n_out best of one beam are ahead of the other's but for the last, which nearly
    ties with the other's first: the choice is who comes in, not the order."""
    rng = np.random.default_rng(2)
    groups, vocab, n_out = 64, 3000, 5
    logits = (2 * rng.normal(size=(groups, 2, vocab))).astype(np.float32)
    lp = -np.sort(-log_p(logits), -1)
    scores = np.zeros((groups, 2), np.float32)
    scores[:, 1] = lp[:, 0, n_out - 1] - lp[:, 1, 0]
    compare(logits, scores, np.zeros((groups, 2), bool), n_out)


def test_a_finished_beam_and_one_that_goes_on():
    """A finished beam's score is exact; the other's best comes near it."""
    rng = np.random.default_rng(3)
    groups, vocab = 64, 3000
    logits = (2 * rng.normal(size=(groups, 2, vocab))).astype(np.float32)
    top = log_p(logits).max(-1)
    scores = np.full((groups, 2), -4.0, np.float32)
    scores[:, 1] = (-4.0 - top[:, 1]).astype(np.float32)
    finished = np.zeros((groups, 2), bool)
    finished[:, 0] = True
    compare(logits, scores, finished, 3, eos=2)


@pytest.mark.parametrize("score", [-3.0, -1e4])
def test_more_ties_than_are_ranked_at_once(score):
    """Most tokens of a beam have one logit, so that over a thousand candidates tie within
    their beam, and the beams nearly."""
    rng = np.random.default_rng(4)
    beams, vocab, n_out = 4, 102400, 64
    logits = np.zeros((1, beams, vocab), np.float32)
    for b in range(beams):
        low = rng.integers(0, vocab, 5000)
        logits[0, b, low] = -rng.random(5000).astype(np.float32) * 9
    top = log_p(logits).max(-1)
    scores = (score - top).astype(np.float32)
    compare(logits, scores, np.zeros((1, beams), bool), n_out)


def test_logits_of_every_kind_beside_near_ties():
    """NaN, infinities and the largest numbers in rows whose sums are taken anew."""
    rng = np.random.default_rng(5)
    groups, beams, vocab = 16, 3, 2000
    logits = rng.normal(size=(groups, beams, vocab)).astype(np.float32)
    logits[:, :, 5::7] = -np.inf
    logits[:, :, 6::7] = np.nan
    clean = np.where(np.isfinite(logits), logits, -1e4)
    top = log_p(clean).max(-1)
    scores = (-5.0 - top).astype(np.float32)
    scores[::4, 1] = -np.inf
    scores[1::4, 2] = np.nan
    logits[2::4, 0, 9] = np.inf
    compare(logits, scores, np.zeros((groups, beams), bool), 4)


def test_the_same_beam_twice():
    """Equal rows and scores: the lower beam first, as before."""
    rng = np.random.default_rng(6)
    row = rng.normal(size=(8, 1, 4000)).astype(np.float32)
    logits = np.repeat(row, 3, 1)
    scores = np.zeros((8, 3), np.float32)
    select = ops.BeamSelector(8, 3, 6, 4000)
    got = select.select(torch.from_numpy(logits).cuda().view(24, 4000), torch.from_numpy(scores).cuda())
    order = np.argsort(-row[:, 0], 1, kind="stable")[:, :2]
    for g in range(8):
        assert got["parents"][g].tolist() == [3 * g, 3 * g + 1, 3 * g + 2] * 2
        assert got["tokens"][g].tolist() == [order[g, 0]] * 3 + [order[g, 1]] * 3

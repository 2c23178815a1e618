"""GPU: the choice of beams (ops.BeamSelector) against its restatement in 64 bits
(paged_ref.beam_select): parents, tokens and finished flags exactly, scores to the
rounding of the exponentials' sum."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, ops  # noqa: E402


def say(msg: str) -> None:
    print(f"[gpu] {msg}", flush=True)


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def run(logits, scores, finished, n_out, eos, pad=0):
    g, b, v = logits.shape
    x = torch.zeros((g * b, v + pad), device="cuda")
    x[:, :v] = torch.from_numpy(logits.reshape(g * b, v))
    sel = ops.BeamSelector(g, b, n_out, v, eos=eos)
    f = None if finished is None else torch.from_numpy(finished.astype(np.uint8)).cuda()
    r = sel.select(x[:, :v], torch.from_numpy(scores.astype(np.float32)).cuda(), f)
    again = sel.select(x[:, :v], torch.from_numpy(scores.astype(np.float32)).cuda(), f)
    assert all(torch.equal(r[k], again[k]) for k in r)
    return {k: t.cpu().numpy() for k, t in r.items()}


def check(logits, scores, finished=None, n_out=4, eos=-1, pad=0):
    say(f"groups, beams, vocab {logits.shape} out {n_out}")
    got = run(logits, scores, finished, n_out, eos, pad)
    done = np.zeros(scores.shape, bool) if finished is None else finished
    want = ref.beam_select(logits, scores, done, n_out, eos)
    for g, rows in enumerate(want):
        for k, (score, parent, token, end) in enumerate(rows):
            at = (got["parents"][g, k], got["tokens"][g, k], got["finished"][g, k])
            assert at == (parent, token, end), (g, k, at, rows[k])
            s = got["scores"][g, k]
            # half a step of fp32, and of the sum: exponentials within 2^-20 of each
            # (the argument's rounding times up to 16 where they matter)
            ok = s == score if np.isinf(score) else abs(s - score) <= 2.0**-24 * abs(score) + 2.0**-20
            assert ok, (g, k, s, score)


@pytest.mark.parametrize("groups, beams, vocab, n_out", [
    (1, 1, 1, 1), (1, 1, 5, 4), (2, 3, 2, 8), (1, 4, 102400, 4), (3, 8, 4097, 16), (2, 5, 4096, 64),
    (1, 64, 1000, 64), (4, 2, 8191, 3), (1, 2, 50001, 64), (9, 1, 300, 1)])
def test_choice(groups, beams, vocab, n_out):
    rng = np.random.default_rng(vocab + beams)
    logits = ref.bf16(rng.normal(size=(groups, beams, vocab)) * 3)
    scores = -10 * rng.random((groups, beams)).astype(np.float32)
    check(logits, scores, n_out=n_out)
    finished = rng.random((groups, beams)) < 0.3
    check(logits, scores, finished, n_out, eos=int(rng.integers(vocab)), pad=3)
    check(logits, scores, finished, n_out, eos=-1, pad=8)


def test_first_step():
    """One beam alive, the others at -infinity: all continuations are its own."""
    rng = np.random.default_rng(1)
    logits = ref.bf16(rng.normal(size=(2, 4, 6000)))
    scores = np.full((2, 4), -np.inf, np.float32)
    scores[0, 0], scores[1, 2] = 0, -3
    check(logits, scores, n_out=4, eos=7)
    scores[1, 2] = np.nan
    check(logits, scores, n_out=4, eos=7)           # the second group offers nothing


@pytest.mark.parametrize("vocab", [100, 4096, 9000])
def test_ties_go_to_the_lowest(vocab):
    """Equal logits everywhere, in long runs, and equal beams."""
    x = np.zeros((1, 3, vocab), np.float32)
    check(x, np.zeros((1, 3), np.float32), n_out=40)
    rng = np.random.default_rng(2)
    x = np.round(rng.normal(size=(2, 3, vocab))).astype(np.float32)
    x[1, 2] = x[1, 0]
    scores = np.array([[0, 0, -1], [-2, -2, -2]], np.float32)
    check(x, scores, n_out=64)
    x[0, 1] = -0.0
    x[0, 1, ::2] = 0.0                              # zeros of either sign are equal
    check(x, scores, n_out=64)
    x = np.sort(rng.normal(size=(1, 1, vocab)).astype(np.float32), -1)   # the best side by side
    check(x, np.zeros((1, 1), np.float32), n_out=64)


def test_masked_logits():
    rng = np.random.default_rng(3)
    x = rng.normal(size=(3, 2, 5000)).astype(np.float32)
    x[0, 0, 10:] = -np.inf                          # ten tokens left
    x[0, 1] = -np.inf                               # none
    x[1, 0, ::3] = np.nan
    x[1, 0, 1::3] = np.finfo(np.float32).min
    x[1, 1, 4999] = np.inf
    x[2, 0, 100:200] = np.inf
    x[2, 1] = np.finfo(np.float32).min              # the type's lowest value, all the same
    scores = np.array([[-1, -2], [-3, -1], [0, -5]], np.float32)
    check(x, scores, n_out=16, eos=3)
    check(x, scores, np.array([[0, 1], [0, 0], [1, 1]], bool), n_out=64, eos=3)


def test_scores_far_apart_and_infinite():
    rng = np.random.default_rng(4)
    x = rng.normal(size=(2, 3, 700)).astype(np.float32)
    check(x, np.array([[0, -1e30, -20], [3e38, -3e38, 0]], np.float32), n_out=5)
    x *= 80
    check(x, np.array([[0, -50, -20], [-1, -2, 0]], np.float32), n_out=9)


def test_refusals():
    for bad in (dict(n_groups=0, n_beams=1), dict(n_groups=1, n_beams=65),
                dict(n_groups=1, n_beams=1, n_out=65), dict(n_groups=1, n_beams=1, vocab=0),
                dict(n_groups=1, n_beams=1, vocab=10, eos=10)):
        with pytest.raises(ValueError):
            ops.BeamSelector(**bad)
    sel = ops.BeamSelector(2, 2, 2, 100)
    x, s = torch.zeros((4, 100), device="cuda"), torch.zeros((2, 2), device="cuda")
    for args in ((x[:3], s), (x[:, :99], s), (x.half(), s), (x.cpu(), s), (x.T[:4], s),
                 (x[:1].expand(4, 100), s), (x, s[0]), (x, s, s), (x, s.cpu())):
        with pytest.raises(ValueError):
            sel.select(*args)


def test_in_a_graph():
    rng = np.random.default_rng(5)
    sel = ops.BeamSelector(2, 4, 4, 3000, eos=1)
    x = torch.zeros((8, 3000), device="cuda")
    s = torch.zeros((2, 4), device="cuda")
    f = torch.zeros((2, 4), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        out = sel.select(x, s, f)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        x.copy_(torch.from_numpy(rng.normal(size=(8, 3000)).astype(np.float32)))
        s.copy_(torch.from_numpy(-rng.random((2, 4)).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        got = {k: t.clone() for k, t in out.items()}
        eager = sel.select(x, s, f)
        assert all(torch.equal(got[k], eager[k]) for k in got)


def test_library_error_names_the_call():
    with pytest.raises(_lib.FleetMoeError, match="fleet_beam_select"):
        _lib.check(_lib.ERR_ARG, "fleet_beam_select")

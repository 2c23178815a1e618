"""GPU: shared attention of a cache of which few sequences have tokens in a call: what is
between them takes no time of its own."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import paged  # noqa: E402
from test_gpu_paged import Both, compare, i32, normal, say, starts, to_dev  # noqa: E402
from test_gpu_shared_prefix import query  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def holding(seed, n, lens):
    """A cache of n sequences of which lens[s] positions are held by sequence s."""
    counts = [lens.get(s, 0) for s in range(n)]
    b = Both(sum(-(-x // 64) for x in counts) + 1, n, -(-max(counts) // 64), 1)
    rng = np.random.default_rng(seed)
    assert b.grow(counts)
    b.append(counts, normal(rng, (1, sum(counts), ref.ROW)))
    return b, rng


def alone(b, tokens, heads):
    p = paged.SharedPrefix(b.dev, i32([0, 1]), tokens, heads)
    p.update()
    return p


# (units of 16 rows, and of 64 where those would be more than 2,048 pages)
HEIGHTS = pytest.mark.parametrize("heads, length", [(16, 700), (128, 9000)])


@HEIGHTS
@pytest.mark.parametrize("n, held", [(1024, [0, 1023]), (1024, [0, 1, 511, 512, 1022]), (1024, [1023]),
                                     (1023, [0, 63, 64, 127, 128, 1022]), (513, [1, 512]),
                                     (512, [0, 63, 64, 511]), (300, [7, 299])])
def test_far_apart(n, held, heads, length):
    say(f"{n} sequences, {held}, {heads} heads of {length}")
    lens = {s: length - 17 * i for i, s in enumerate(held)}
    b, rng = holding(n + len(held), n, lens)
    counts = [1 + (s % 2) if s in lens else 0 for s in range(n)]
    q = query(rng, sum(counts), heads)
    out, lse = alone(b, sum(counts), heads).attend(to_dev(q), starts(counts))
    compare(b, q, counts, out, lse)
    assert b.dev.status() == 0


def graph_us(f, n=10):
    f()
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        for _ in range(n):
            f()
    times = []
    for _ in range(6):
        a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        z.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(z) / n * 1e3)
    return min(times)


@HEIGHTS
def test_what_lies_between_takes_no_time(heads, length):
    """Tokens in the first and last of 1,024 sequences take as long as in the first two: at most
    twice as long, where a look at every sequence between them is a thousand loads one after
    another."""
    n, took = 1024, []
    for held in ([0, 1], [0, 1023]):
        b, rng = holding(5, n, {s: length for s in held})
        counts = [int(s in held) for s in range(n)]
        q, at = to_dev(query(rng, 2, heads)), starts(counts)
        p = alone(b, 2, heads)
        out, lse = p.attend(q, at)
        took.append(graph_us(lambda: p.attend(q, at, out=out, lse=lse)))
    say(f"{heads} heads of {length}: {took[0]:.1f} us side by side, {took[1]:.1f} far apart")
    assert took[1] <= 2 * took[0]

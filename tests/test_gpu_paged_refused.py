"""GPU: a step whose growth is refused leaves the cache as it was, the rows of the
step among it, and can be taken again once there is room."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, paged  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def dev_rows(x):
    return torch.from_numpy(ref.bits(x)).cuda()


def normal(rng, shape):
    return ref.bf16(rng.normal(size=shape))


def full_pool(seed, lens=(10, 64, 70), n_layers=2):
    """Sequences that hold every page of the pool, the first of them with room left."""
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // 64) for n in lens)
    dev = paged.PagedCache.empty(pages, len(lens), 4, n_layers)
    dev.pool.fill_(0xFF)
    want = ref.Cache(pages, len(lens), 4, n_layers)
    assert want.grow(list(lens))
    dev.grow(i32(lens))
    rows = normal(rng, (n_layers, sum(lens), ref.ROW))
    at = np.concatenate([[0], np.cumsum(lens)])
    want.append(rows, at)
    dev.append(dev_rows(rows), i32(at))
    return dev, want, rng


def state(c):
    return [t.clone() for t in (c.pool, c.table, c.lens, c.refs)]


def same(c, before):
    return all(torch.equal(a, b) for a, b in zip(state(c), before))


def check(dev, want):
    assert dev.lens.tolist() == want.lens
    assert np.array_equal(dev.table.cpu().numpy(), want.table())
    assert np.array_equal(dev.refs.cpu().numpy(), want.refs())
    codes, scales = ref.unpack(dev.pool.cpu().numpy())
    for s, n in enumerate(want.lens):
        for p in range(n):
            page, t = want.rows[s][p // 64], p % 64
            assert np.array_equal(ref.VALUES[codes[page, :, t]], ref.VALUES[want.codes[page, :, t]])
            assert np.array_equal(scales[page, :, t // 16],
                                  2.0 ** want.exps[page, :, t // 16].astype(float))


def test_a_step_without_room_and_again_with_it():
    dev, want, rng = full_pool(1)
    before = state(dev)
    rows = normal(rng, (2, 3, ref.ROW)) * np.float32(64)      # (the scales would grow)
    for _ in range(2):
        assert not want.grow([1, 1, 1])
        dev.grow(i32([1, 1, 1]))
        dev.append(dev_rows(rows))
        assert dev.status() == _lib.ABORT_NO_PAGE and same(dev, before)
    # the status is what came since it was cleared: append reports the refusal again
    dev.clear_status()
    assert dev.status() == 0
    dev.append(dev_rows(rows[:, :2]), i32([0, 1, 2, 2]))
    assert dev.status() == _lib.ABORT_NO_PAGE and same(dev, before)
    # a sequence ends, and the step fits
    want.remap([0, 1, -1])
    dev.remap(i32([0, 1, -1]))
    dev.clear_status()
    assert want.grow([1, 1, 1])
    dev.grow(i32([1, 1, 1]))
    want.append(rows, [0, 1, 2, 3])
    dev.append(dev_rows(rows))
    assert dev.status() == 0
    check(dev, want)


@pytest.mark.parametrize("what, bit", [("count", _lib.ABORT_POSITION), ("length", _lib.ABORT_POSITION),
                                       ("page", _lib.ABORT_BAD_PAGE), ("row", _lib.ABORT_NO_PAGE)])
def test_every_refusal_keeps_the_rows(what, bit):
    dev, want, rng = full_pool(2)
    new = [1, 0, 1]
    if what == "count":
        new[1] = -1
    elif what == "length":
        dev.lens[1] = -4
    elif what == "page":
        dev.table[0, 0] = dev.n_pages
    else:
        new[1] = 4 * 64
    before = state(dev)
    dev.grow(i32(new))
    dev.append(dev_rows(normal(rng, (2, 1, ref.ROW))), i32([0, 0, 0, 1]))
    assert dev.status() == bit and same(dev, before)


def test_a_grow_of_nothing_ends_the_refusal():
    """Then append writes the newest positions anew, as it does without a grow before it."""
    dev, want, rng = full_pool(3)
    dev.grow(i32([0, 1, 0]))
    assert dev.status() == _lib.ABORT_NO_PAGE
    dev.clear_status()
    dev.grow(i32([0, 0, 0]))
    rows = normal(rng, (2, 3, ref.ROW))
    want.append(rows, [0, 1, 2, 3])
    dev.append(dev_rows(rows))
    assert dev.status() == 0
    check(dev, want)


def test_a_captured_step_without_room_and_again_with_it():
    dev, want, rng = full_pool(4)
    rows = normal(rng, (2, 3, ref.ROW)) * np.float32(64)
    moved, parents, one = dev_rows(rows), i32([0, 1, 2]), i32([1, 1, 1])
    before = state(dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        dev.clear_status()
        dev.remap(parents)
        dev.grow(one)
        dev.append(moved)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        g.replay()
        assert dev.status() == _lib.ABORT_NO_PAGE and same(dev, before)
    parents.copy_(i32([0, 1, -1]))
    want.remap([0, 1, -1])
    for _ in range(3):
        g.replay()
        parents.copy_(i32([0, 1, 2]))
        assert want.grow([1, 1, 1])
        want.append(rows, [0, 1, 2, 3])
        assert dev.status() == 0
        want.remap([0, 1, 2])
        check(dev, want)


def test_more_rows_than_positions_after_a_refusal():
    """An empty sequence whose prompt finds no room: the refusal is what is reported."""
    dev, want, rng = full_pool(5, (64, 10, 0))
    before = state(dev)
    rows = dev_rows(normal(rng, (2, 70, ref.ROW)))
    dev.grow(i32([0, 0, 70]))
    dev.clear_status()
    dev.append(rows, i32([0, 0, 0, 70]))
    assert dev.status() == _lib.ABORT_NO_PAGE and same(dev, before)
    dev.append(rows, i32([0, 0, 20, 70]))
    assert dev.status() == _lib.ABORT_NO_PAGE and same(dev, before)

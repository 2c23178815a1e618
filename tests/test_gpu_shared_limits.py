"""GPU: attention of sequences that share their first pages, and rows appended as they are
projected, at the ends of the ranges that they accept."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import ops, paged  # noqa: E402
from test_gpu_append_latent import made  # noqa: E402
from test_gpu_paged import SCALE, Both, i32, say, starts, to_dev  # noqa: E402
from test_gpu_shared_prefix import FEW, both_heights, forked, plan, query  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def near(b, q, counts, out, lse, scale, seqs, skip=()):
    """Sequences `seqs` against 64 bits at a scale of fp32; rows [token, heads] of `skip` are NaN."""
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    at = np.concatenate([[0], np.cumsum(counts)])
    for s in seqs:
        total, n = b.ref.lens[s], counts[s]
        with np.errstate(invalid="ignore", over="ignore"):
            o, e, tol, tl = ref.attend(b.ref.values(s), q[at[s]: at[s + 1]], range(total - n, total),
                                       float(np.float32(scale)))
        g, l = got[at[s]: at[s + 1]], gl[at[s]: at[s + 1]]
        sure = np.ones(l.shape, bool)
        for i, heads in skip:
            if at[s] <= i < at[s + 1]:
                assert np.isnan(g[i - at[s], heads]).all() and np.isnan(l[i - at[s], heads]).all()
                sure[i - at[s], heads] = False
        assert (np.abs(g - o)[sure] <= tol[sure]).all(), s
        assert (np.abs(l - e)[sure] <= tl[sure]).all(), s


@both_heights
@pytest.mark.parametrize("scale", [1e-45, 1e-39, 1e-38, 1.6e-38, 1e-37, 1e30, 2.35e38])
def test_scales_at_both_ends(scale, tall):
    b, rng, groups = forked(70, [200], [[30, 100, 3]], tall=FEW * tall)
    counts = [2] * 3 + [1] * FEW * tall
    q = query(rng, sum(counts))
    if scale > 1:
        q = ref.bf16(q * (0.1 / scale))
    say(f"scale {scale}")
    out, lse = plan(b, groups, len(q)).attend(to_dev(q), starts(counts), scale=scale)
    near(b, q, counts, out, lse, scale, range(3))
    assert b.dev.status() == 0


@both_heights
def test_scores_beyond_fp32(tall):
    """Finite products q . row that are infinite times the scale: +infinity makes its token and
    head NaN, and no other, in the common pages and a sequence's own."""
    b, rng, groups = forked(71, [200], [[30, 100, 3]], tall=FEW * tall)
    counts = [1, 2, 1] + [1] * FEW * tall
    scale = 1e20
    q = ref.bf16(rng.normal(size=(sum(counts), 16, ref.ROW)) * 0.05 / scale)
    q[1, ::2] = ref.bf16(rng.normal(size=(8, ref.ROW)) * 1e19)
    z = q[1, ::2].astype(float) @ b.ref.values(1)[:-1].T
    top = float(np.finfo(np.float32).max)
    assert (np.abs(z) < top).all() and (scale * z.max(1) > 2 * top).all()
    out, lse = plan(b, groups, len(q)).attend(to_dev(q), starts(counts), scale=scale)
    near(b, q, counts, out, lse, scale, range(3), [(1, np.arange(0, 16, 2))])


def of_rows(n, common, own, new, heads):
    """n sequences behind `common` rows, each with the rows `own`."""
    pages = -(-len(common) // 64) + n * (-(-len(own) // 64) + 2)
    b = Both(pages, n, -(-(len(common) + len(own)) // 64) + 1, 1)
    assert b.grow([len(common)] + [0] * (n - 1))
    b.append([len(common)] + [0] * (n - 1), common[None])
    b.remap([0] * n)
    assert b.grow([len(own)] * n)
    b.append([len(own)] * n, np.concatenate([own] * n)[None])
    return b, paged.SharedPrefix(b.dev, i32([0, n]), n * new, heads)


@pytest.mark.parametrize("n, common, own, new", [(2, 64, 20, 1), (3, 64, 200, 2), (2, 128, 5, 1),
                                                 (40, 9000, 64, 1)])
def test_scores_of_minus_infinity(n, common, own, new):
    """The first 64 positions have finite products that are -infinity times the scale, the
    others 0: the first have no weight."""
    rng = np.random.default_rng(n)
    rows = np.zeros((common + own, ref.ROW), np.float32)
    rows[:64, :256] = ref.bf16(np.abs(rng.normal(size=(64, 256))) + 1)
    rows[64:, 256:512] = ref.bf16(rng.normal(size=(common + own - 64, 256)))
    b, p = of_rows(n, rows[:common], rows[common:], new, 16)
    assert p.update()[0] == common // 64
    q = np.zeros((n * new, 16, ref.ROW), np.float32)
    q[..., :256] = -1e19
    out, lse = p.attend(to_dev(ref.bf16(q)), starts([new] * n), scale=1e20)
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    for s in (0, n - 1):
        v = b.ref.values(s)[64:]
        o, e, tol, tl = ref.attend(v, q[:new], range(len(v) - new, len(v)), 1.0)
        assert (np.abs(got[s * new: (s + 1) * new] - o) <= tol).all()
        assert (np.abs(gl[s * new: (s + 1) * new] - e) <= tl).all()


@pytest.mark.parametrize("n, common, own, new, heads", [(2, 64, 2, 1, 16), (3, 640, 30, 2, 16),
                                                        (2, 3000, 300, 1, 40)])
def test_weights_that_nearly_cancel(n, common, own, new, heads):
    """Few pages: c is 1 at even positions and -1 at odd ones, whose scores are lower by 11/8192:
    the weights are 1 and 0.99866, which is nearest to 1 in bf16, and the output 0.00067."""
    rows = np.zeros((common + own, ref.ROW), np.float32)
    rows[0::2, :ref.C], rows[1::2, :ref.C] = 1.0, -1.0
    rows[1::2, ref.C] = -11 / 8192
    b, p = of_rows(n, rows[:common], rows[common:], new, heads)
    p.update()
    assert np.array_equal(b.ref.values(0), rows)
    q = np.zeros((n * new, heads, ref.ROW), np.float32)
    q[..., ref.C] = 1.0
    out, lse = p.attend(to_dev(ref.bf16(q)), starts([new] * n), scale=1.0)
    got, gl = ref.values(out.cpu().numpy()), lse.cpu().numpy()
    o, e, _, tl = ref.attend(rows.astype(float), q[:new], range(len(rows) - new, len(rows)), 1.0)
    # half a bf16 step of the output; half a step of 16 bits of each weight, in numerator and
    # denominator, and 2^-20 for exponentials and sums, of sum w |c| = 1
    tol = 2.0**-8 * np.abs(o) + 2 * 2.0**-16 + 2.0**-20
    for s in range(n):
        assert (np.abs(got[s * new: (s + 1) * new] - o) <= tol).all()
        assert (np.abs(gl[s * new: (s + 1) * new] - e) <= tl).all()


def test_offsets_beyond_32_bits():
    """A pool of 5 GB: projected rows and attention in its last pages and layer."""
    layers, pages = 27, 5100
    c = paged.PagedCache.empty(pages, 2, 4, layers)
    named = [[pages - 1, 17, pages - 2], [pages - 1, 17, pages - 3]]
    c.table[:, :3] = i32(named)
    c.refs[[pages - 1, 17, pages - 2, pages - 3]] = 1
    rng = np.random.default_rng(73)
    rope = ops.Rotary(np.zeros(32))             # (neighbours become halves, no more)
    rows = ref.bf16(rng.normal(size=(128 + 20 + 33, ref.ROW)))
    final = made(rows, None, np.zeros(len(rows)))
    c.lens.copy_(i32([128, 0]))
    c.append_latent(to_dev(rows[:128]), rope, start=starts([128, 0]), layer=layers - 1)
    c.refs[[pages - 1, 17]] = 2
    c.lens.copy_(i32([148, 161]))
    c.append_latent(to_dev(rows[128:]), rope, start=starts([20, 33]), layer=layers - 1)
    assert c.status() == 0
    p = paged.SharedPrefix(c, i32([0, 2]), 2, 16)
    assert p.update().tolist() == [2]
    q = query(rng, 2)
    out, lse = p.attend(to_dev(q), layer=layers - 1)
    for s, own in enumerate((final[128:148], final[148:])):
        say(f"sequence {s}")
        codes, scales = ref.unpack(c.pool[named[s]].cpu().numpy())
        wide = np.repeat(np.repeat(scales[:, layers - 1], [512, 64], 2), 16, 1)
        v = (ref.VALUES[codes[:, layers - 1]] * wide).reshape(-1, ref.ROW)[: 128 + len(own)]
        want = np.concatenate([final[:128], own])
        # half a step of 8 bits (below the least normal number 2^-10 of the scale, which is
        # at most 2 / 448 of the largest value), and 2^-18 for the norm in 32 bits
        big = np.abs(want).max()
        tol = np.maximum(2.0**-4 * np.abs(want), 2.0**-10 * big / 224) + 2.0**-18 * big
        assert (np.abs(v - want) <= tol).all()
        o, e, tol, tl = ref.attend(v.astype(float), q[s: s + 1], [len(v) - 1], SCALE)
        assert (np.abs(ref.values(out[s: s + 1].cpu().numpy()) - o) <= tol).all()
        assert (np.abs(lse[s: s + 1].cpu().numpy() - e) <= tl).all()
    assert c.status() == 0


@pytest.mark.parametrize("heads", [1, 16, 128])
def test_the_most_rows(heads):
    """2^20 rows, of which the last tokens of each sequence stand at positions."""
    b, rng, groups = forked(74, [128], [[70, 9]])
    tokens = (1 << 20) // heads
    counts = [tokens - 140, 140]
    last = query(rng, 340, heads)
    q = torch.zeros((tokens, heads, ref.ROW), dtype=torch.int16, device="cuda")
    q[-340:] = to_dev(last)
    say(f"{tokens} tokens of {heads} heads")
    out, lse = plan(b, groups, tokens, heads).attend(q, starts(counts))
    assert b.dev.status() == 0
    assert not out[: tokens - 338].any() and torch.isneginf(lse[: tokens - 338]).all()
    for s, at, seen in ((0, tokens - 140, 198), (1, tokens, 137)):
        pos = np.unique(np.concatenate([np.arange(0, seen, 13), [seen - 1]]))
        i = at - seen + pos
        o, e, tol, tl = ref.attend(b.ref.values(s), last[i - (tokens - 340)], pos, SCALE)
        assert (np.abs(ref.values(out[i.tolist()].cpu().numpy()) - o) <= tol).all()
        assert (np.abs(lse[i.tolist()].cpu().numpy() - e) <= tl).all()
    assert (out[tokens - 140: tokens - 137] == 0).all()

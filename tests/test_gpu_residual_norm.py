"""GPU: the norms around a block with gate and residual (ops.residual_norm) against the
formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_ref as ref  # noqa: E402
from fleet_moe import _lib, ops  # noqa: E402

BITS, F32 = torch.int16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def dev(x, dtype):
    x = np.ascontiguousarray(x, np.float32)
    return torch.from_numpy(x if dtype == F32 else ref.bits(ref.bf16(x))).cuda()


def host(t):
    a = t.cpu()
    return a.numpy().astype(np.float64) if a.dtype == F32 else ref.values(a.numpy()).astype(np.float64)


def unit(v, eps):
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def check(x, y=None, norm=None, post=None, gate=None, scale=1.0, eps=1e-6, got=None):
    """Tolerances: a bf16 result is off by half a step, 2^-8 of it (fp32: 2^-24). The mean of
    squares is a sum of at most 40 roundings a thread and 10 between threads, 50 * 2^-24 of it, so
    its root is off by 25 * 2^-24; with the root, the quotient and the products 2^-19 of u and
    of h. x' is u's error and three roundings: 2^-18 of |x| + |scale gate u|; and h what that
    makes of it, over the rms. Below 2^-126 the step of bf16 is 2^-133 whatever the value: half of
    it, 2^-134, on top of everything."""
    xd = host(x)
    want, slack = xd, np.zeros_like(xd)
    x_out, h = got
    if y is not None:
        u = host(y)
        if post is not None:
            u = unit(u, eps) * host(post)
        if gate is not None:
            u = u * host(gate)
        want = xd + scale * u
        slack = 2.0**-18 * (np.abs(xd) + np.abs(scale * u)) + 2.0**-134
        half = 2.0**-24 if x.dtype == F32 else 2.0**-8
        d = np.abs(host(x_out) - want)
        assert x_out.dtype == x.dtype
        assert (d <= half * np.abs(want) + slack).all(), np.nanmax(d - half * np.abs(want) - slack)
    rms = np.sqrt((want * want).mean(-1, keepdims=True) + eps)
    w = 1.0 if norm is None else host(norm)
    d = np.abs(host(h) - want / rms * w)
    tol = (2.0**-8 + 2.0**-18) * np.abs(want / rms * w) + np.abs(w) * slack / rms + 2.0**-134
    # (the mean takes the errors of x', weighted by x', too)
    tol += np.abs(want / rms * w) * (slack / rms).max(-1, keepdims=True)
    assert (d <= tol).all(), np.nanmax(d - tol)


SIZES = [(1, 2048), (3, 2048), (1100, 2048), (5, 1), (2, 7), (4, 8), (3, 577), (1030, 577), (2, 2056),
         (3, 4100), (2, 8192), (2, 8200), (1, 32768), (1, 12345)]
# the ends of what a number of threads holds
SIZES += [(3, w) for w in (512, 513, 1024, 1025, 1536, 1537, 2049, 4096, 4097, 16384, 16385, 24576, 24577)]


@pytest.mark.parametrize("rows, width", SIZES)
@pytest.mark.parametrize("xt, yt, post, gate", [
    (BITS, BITS, False, None), (F32, BITS, True, "channel"), (BITS, F32, True, "token"),
    (F32, F32, False, "token")])
def test_against_the_formula(rows, width, xt, yt, post, gate):
    rng = np.random.default_rng(rows * 7 + width)
    n = lambda *s: rng.normal(size=s)  # noqa: E731
    x, y = dev(4 * n(rows, width), xt), dev(n(rows, width) * 3, yt)
    norm, p = dev(1 + 0.1 * n(width), BITS), dev(0.5 + 0.1 * n(width), BITS) if post else None
    g = dev(n(*((width,) if gate == "channel" else (rows, width))), BITS) if gate else None
    got = ops.residual_norm(x, y, norm, post_norm=p, gate=g, scale=-0.7)
    check(x, y, norm, p, g, -0.7, got=got)
    x_out, h = ops.residual_norm(x, None, norm)           # the norm alone
    assert x_out is x
    check(x, None, norm, got=(x_out, h))


def test_strides_given_outputs_and_in_place():
    rng = np.random.default_rng(3)
    wide = dev(rng.normal(size=(5, 3 * 640)), BITS)
    x, y, g = wide[:, :640], wide[:, 640:1280], wide[:, 1280:]
    a, h = ops.residual_norm(x, y, gate=g)
    check(x, y, gate=g, got=(a, h))
    # odd columns: not in chunks of 16 bytes
    for lo in (1, 3, 4):
        c = [t[:, lo: lo + 600] for t in (x, y, g)]
        check(c[0], c[1], gate=c[2], got=ops.residual_norm(c[0], c[1], gate=c[2]))
    # one row of y and of the gate for all
    one = y[:1].expand(5, 640)
    check(x, one, gate=g[2:3].expand(5, 640),
          got=ops.residual_norm(x, one, gate=g[2:3].expand(5, 640)))
    xc = x.contiguous()
    out = torch.full_like(xc, -1)
    hb, hf = torch.zeros_like(xc), torch.zeros(xc.shape, device="cuda")
    b = ops.residual_norm(xc, y, gate=g, x_out=out, h=hb, h_f32=hf)
    assert b[0] is out and b[1] is hb and torch.equal(out, a) and torch.equal(hb, h)
    assert torch.equal(hf, ops.bf16_bits_to_f32(hb))
    ops.residual_norm(xc, y, gate=g, x_out=xc, h=hb)
    assert torch.equal(xc, a) and torch.equal(hb, h)


@pytest.mark.parametrize("dtype", [BITS, F32])
def test_values_far_out(dtype):
    """The largest and the smallest numbers, zeros, and what is not finite."""
    rng = np.random.default_rng(4)
    x = rng.normal(size=(9, 2048))
    x[0] *= 5e37
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = 0
    x[4, 5] = 3.3e38
    t = dev(x, dtype)
    norm = dev(np.full(2048, 2.0), BITS)
    check(t[:5], None, norm, got=ops.residual_norm(t[:5], None, norm))
    check(t[5:], None, norm, got=ops.residual_norm(t[5:], None, norm))
    zero = torch.zeros_like(t)
    y = dev(np.abs(x) * 1e-3, dtype)
    check(zero, y, norm, post=norm, got=ops.residual_norm(zero, y, norm, post_norm=norm))
    x[5, 7], x[6, 100], x[7, 3], x[7, 4] = np.inf, np.nan, np.inf, -np.inf
    xo, h = ops.residual_norm(zero, dev(x, dtype), norm)
    h, xo = host(h), host(xo)
    assert np.isnan(h[5, 7]) and (np.delete(h[5], 7) == 0).all() and np.isnan(h[6]).all()
    assert np.isnan(h[7, 3:5]).all() and (h[7, 5:] == 0).all()
    assert np.isinf(xo[5, 7]) and np.isnan(xo[6, 100]) and np.isfinite(np.delete(xo[6], 100)).all()
    assert np.isfinite(h[[0, 1, 2, 3, 4, 8]]).all()


def test_a_row_is_the_same_in_any_batch():
    """Results depend neither on the rows beside a row nor on their number."""
    rng = np.random.default_rng(5)
    x, y = dev(rng.normal(size=(700, 2048)), BITS), dev(rng.normal(size=(700, 2048)), BITS)
    a, h = ops.residual_norm(x, y)
    for i in (0, 5, 699):
        a1, h1 = ops.residual_norm(x[i:i + 1], y[i:i + 1])
        assert torch.equal(a1[0], a[i]) and torch.equal(h1[0], h[i])


def test_refused_and_empty():
    x = torch.zeros((4, 64), dtype=BITS, device="cuda")
    for f in (lambda: ops.residual_norm(x.cpu()), lambda: ops.residual_norm(x[0]),
              lambda: ops.residual_norm(x.half()), lambda: ops.residual_norm(x, x[:3]),
              lambda: ops.residual_norm(x, x.T), lambda: ops.residual_norm(x, gate=x),
              lambda: ops.residual_norm(x, x, gate=x.float()), lambda: ops.residual_norm(x, x_out=x),
              lambda: ops.residual_norm(x, x, norm=x[0, :32]),
              lambda: ops.residual_norm(x, x, x_out=x.float()),
              lambda: ops.residual_norm(x, x, h=x.float()),
              lambda: ops.residual_norm(x, x, h_f32=x)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: ops.residual_norm(x, eps=0.0), lambda: ops.residual_norm(x, x, scale=np.inf),
              lambda: ops.residual_norm(torch.zeros((1, 40000), dtype=BITS, device="cuda"))):
        with pytest.raises(_lib.FleetMoeError):
            f()
    assert ops.residual_norm(x[:0], x[:0])[1].shape == (0, 64)


def test_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(6)
    x, y = dev(rng.normal(size=(33, 2048)), F32), dev(rng.normal(size=(33, 2048)), BITS)
    a, h = ops.residual_norm(x, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a1, h1 = ops.residual_norm(x, y, stream=s)
    s.synchronize()
    assert torch.equal(a1, a) and torch.equal(h1, h)
    xo, hb = torch.zeros_like(a), torch.zeros_like(h)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        ops.residual_norm(x, y, x_out=xo, h=hb)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        xo.zero_(), hb.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(xo, a) and torch.equal(hb, h)
        assert torch.equal(ops.residual_norm(x, y)[1], h)

"""What the calls around a block refuse, and their sizes, without a GPU: the norms with
gate and residual, the rotation, projected rows into pages, shared first pages."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from fleet_moe import _lib
from fleet_moe.rope import RopeParams, frequencies, magnitude, yarn_tables

P = 1 << 20                         # a well aligned address that nothing reads
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    a = dict(pool=P, table=P, lens=P, refs=P, n_pages=64, n_layers=2, n_seqs=4, max_pages=8)
    return _lib.FleetCache(**{**a, **kw})


def rope(**kw):
    return _lib.FleetRope(**{**dict(turns=P, dim=64, halves_in=0, halves_out=1, magnitude=1.0),
                             **kw})


BAD_CACHES = [dict(pool=None), dict(table=None), dict(lens=P + 1), dict(refs=P + 2),
              dict(n_pages=0), dict(n_layers=65), dict(n_seqs=1025), dict(max_pages=0)]
BAD_ROPES = [dict(turns=None), dict(turns=P + 4), dict(dim=0), dict(dim=63), dict(dim=1026),
             dict(dim=-2), dict(halves_in=2), dict(halves_out=-1), dict(magnitude=INF),
             dict(magnitude=NAN)]


def test_norm_refusals(lib):
    def call(**kw):
        a = {**dict(x=P, x_f32=0, xs=2048, y=P, y_f32=0, ys=2048, post=P, gate=P, gs=0, scale=1.0,
                    norm=P, eps=1e-6, x_out=P + 4096, h=P + 8192, hf=P, rows=3, width=2048), **kw}
        return lib.fleet_residual_norm(a["x"], a["x_f32"], a["xs"], a["y"], a["y_f32"], a["ys"],
                                       a["post"], a["gate"], a["gs"], a["scale"], a["norm"],
                                       a["eps"], a["x_out"], a["h"], a["hf"], a["rows"],
                                       a["width"], None)
    for kw in (dict(x=None), dict(x=P + 1), dict(x=P + 2, x_f32=1), dict(x_f32=2), dict(y_f32=-1),
               dict(xs=-1), dict(xs=(1 << 32) + 1), dict(ys=-8), dict(gs=-1), dict(y=P + 1),
               dict(y=P + 2, y_f32=1), dict(post=P + 1), dict(gate=P + 1), dict(norm=P + 1),
               dict(scale=INF), dict(scale=NAN), dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN),
               dict(eps=INF), dict(eps=1e-31), dict(x_out=P + 1), dict(x_out=P + 2, x_f32=1),
               dict(h=None), dict(h=P + 1), dict(hf=P + 2), dict(rows=-1), dict(rows=(1 << 28) + 1),
               dict(width=0), dict(width=32769), dict(x_out=P, xs=4096),
               dict(y=None, post=None, gate=None), dict(y=None, post=None, x_out=None),
               dict(y=None, gate=None, x_out=None)):
        assert call(**kw) == _lib.ERR_ARG, kw
    assert call(rows=0, x=None, h=None) == 0              # nothing to do


def rotations(lib):
    base = dict(x=P, f32=0, xt=1024, xh=64, out=P + 4096, ot=1024, oh=64, n=6, heads=16, width=64,
                at=0)

    def plain(r=None, pos=P, **kw):
        a = {**base, **kw}
        return lib.fleet_rope_rotate(ctypes.byref(r or rope()), a["x"], a["f32"], a["xt"], a["xh"],
                                     a["out"], a["ot"], a["oh"], pos, a["n"], a["heads"],
                                     a["width"], a["at"], None)

    def paged(r=None, c=None, start=P, ws=P, size=lib.fleet_cache_workspace_bytes(64, 4), **kw):
        a = {**base, **kw}
        return lib.fleet_cache_rotate(ctypes.byref(c or cache()), ctypes.byref(r or rope()), a["x"],
                                      a["f32"], a["xt"], a["xh"], a["out"], a["ot"], a["oh"], start,
                                      a["n"], a["heads"], a["width"], a["at"], ws, size, None)
    return plain, paged


def test_rotation_refusals(lib):
    plain, paged = rotations(lib)
    for f in (plain, paged):
        for kw in BAD_ROPES:
            assert f(r=rope(**kw)) == _lib.ERR_ARG, kw
        for kw in (dict(x=None), dict(x=P + 1), dict(x=P + 2, f32=1), dict(f32=2), dict(out=None),
                   dict(out=P + 1), dict(xt=-1), dict(xh=(1 << 32) + 1), dict(ot=-64),
                   dict(n=-1), dict(n=(1 << 28) + 1), dict(heads=0), dict(heads=(1 << 16) + 1),
                   dict(width=62), dict(at=-1), dict(at=1), dict(width=65537), dict(oh=63),
                   dict(ot=1023), dict(ot=0),
                   # in place: the pairs' order, other strides
                   dict(out=P), dict(out=P, r=rope(halves_out=0), ot=2048),
                   dict(out=P, r=rope(halves_out=0), oh=128, ot=2048)):
            assert f(**kw) == _lib.ERR_ARG, kw
        assert f(n=0, x=None, **({"start": P} if f is paged else {})) == 0
    assert plain(pos=None) == _lib.ERR_ARG and plain(pos=P + 2) == _lib.ERR_ARG
    for kw in BAD_CACHES:
        assert paged(c=cache(**kw)) == _lib.ERR_ARG, kw
    assert paged(start=None) == _lib.ERR_ARG              # six tokens, four sequences
    assert paged(start=P + 2) == _lib.ERR_ARG
    assert paged(ws=P + 128) == _lib.ERR_ARG and paged(size=1000) == _lib.ERR_WORKSPACE


def test_latent_refusals(lib):
    n = lib.fleet_cache_workspace_bytes(64, 4)

    def call(c=None, r=None, layer=1, rows=P, stride=576, norm=P, eps=1e-6, start=P, n_rows=10,
             ws=P, size=n):
        return lib.fleet_cache_append_latent(ctypes.byref(c or cache()), layer, rows, stride, norm,
                                             eps, ctypes.byref(r or rope()), start, n_rows, ws, size,
                                             None)
    for kw in BAD_CACHES:
        assert call(c=cache(**kw)) == _lib.ERR_ARG, kw
    for kw in BAD_ROPES + [dict(dim=32), dict(halves_out=0)]:
        assert call(r=rope(**kw)) == _lib.ERR_ARG, kw
    for kw in (dict(layer=-1), dict(layer=2), dict(rows=None), dict(rows=P + 8), dict(stride=568),
               dict(stride=580), dict(stride=1 << 33), dict(norm=P + 8), dict(eps=0.0),
               dict(eps=NAN), dict(eps=INF), dict(start=None), dict(start=P + 2), dict(n_rows=-1),
               dict(n_rows=(1 << 28) + 1), dict(ws=None), dict(ws=P + 128)):
        assert call(**kw) == _lib.ERR_ARG, kw
    assert call(size=n - 1) == _lib.ERR_WORKSPACE
    assert call(n_rows=0, rows=None) == 0


def test_plan_sizes(lib):
    n = lib.fleet_cache_plan_bytes(4, 64, 16)
    assert n % 16 == 0 and (64 << 20) < n < (72 << 20)
    most = lib.fleet_cache_plan_bytes(1024, 1 << 16, 16)
    assert most > (1 << 20) * 4144
    for bad in ((0, 4, 16), (1025, 4, 16), (4, 0, 16), (4, 4, 0), (4, 4, 129),
                (4, (1 << 16) + 1, 16), (4, 2**31 - 1, 128), (4, -1, 16)):
        assert lib.fleet_cache_plan_bytes(*bad) == 0, bad


def test_shared_refusals(lib):
    ws, plan = lib.fleet_cache_workspace_bytes(64, 4), lib.fleet_cache_plan_bytes(4, 6, 16)

    def share(c=None, groups=P, n=2, pages=P, pl=P, pn=plan, w=P, wn=ws):
        return lib.fleet_cache_share(ctypes.byref(c or cache()), groups, n, pages, pl, pn, w, wn,
                                     None)

    def attend(c=None, layer=1, q=P, stride=16 * 576, start=P, n=6, heads=16, scale=0.1, out=P,
               lse=P, pl=P, pn=plan, w=P, wn=ws):
        return lib.fleet_cache_attend_shared(ctypes.byref(c or cache()), layer, q, stride, start, n,
                                             heads, scale, out, lse, pl, pn, w, wn, None)
    for f in (share, attend):
        for kw in BAD_CACHES:
            assert f(c=cache(**kw)) == _lib.ERR_ARG, kw
        for kw in (dict(pl=None), dict(pl=P + 128), dict(w=None), dict(w=P + 16)):
            assert f(**kw) == _lib.ERR_ARG, kw
        assert f(wn=ws - 1) == _lib.ERR_WORKSPACE
    for kw in (dict(groups=None), dict(groups=P + 2), dict(n=0), dict(n=5), dict(pages=P + 1)):
        assert share(**kw) == _lib.ERR_ARG, kw
    assert share(pn=256) == _lib.ERR_WORKSPACE
    for kw in (dict(layer=-1), dict(layer=2), dict(q=None), dict(q=P + 8), dict(stride=16 * 576 - 8),
               dict(stride=16 * 576 + 4), dict(start=P + 2), dict(start=None), dict(n=-1),
               dict(heads=0), dict(heads=129, stride=129 * 576), dict(n=(1 << 16) + 1),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF),
               dict(out=None), dict(out=P + 4), dict(lse=P + 2)):
        assert attend(**kw) == _lib.ERR_ARG, kw
    assert attend(pn=plan - 1) == _lib.ERR_WORKSPACE
    # so many steps that 32 bits would not count them
    wide, n = cache(n_seqs=1024, max_pages=1 << 20), lib.fleet_cache_workspace_bytes(64, 1024)
    assert attend(c=wide, wn=n, pn=1 << 40) == _lib.ERR_ARG
    assert attend(n=0, q=None) == 0


def test_frequencies_are_the_tables():
    p = RopeParams()
    f = frequencies(p)
    assert f.shape == (32,) and f[0] == 1.0 and (np.diff(f) < 0).all()
    # the slowest are stretched by the factor, the fastest as they are
    base = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    assert np.allclose(f[:5], base[:5], rtol=1e-6) and np.allclose(f[-5:], base[-5:] / 40, rtol=1e-6)
    assert magnitude(p) == 1.0
    cos, sin = yarn_tables(100, p)
    a = np.arange(100)[:, None] * np.concatenate([f, f]).astype(np.float64)
    # the tables' angles are rounded to fp32: half a step, 2^-24, of up to 99 radians
    assert np.abs(cos - np.cos(a)).max() < 99 * 2.0**-24 + 2.0**-23
    assert np.abs(sin - np.sin(a)).max() < 99 * 2.0**-24 + 2.0**-23
    other = RopeParams(mscale=1.0, mscale_all_dim=0.5)
    want = (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)
    assert abs(magnitude(other) - want) < 1e-12

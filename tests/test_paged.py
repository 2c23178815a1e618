"""The paged 8-bit cache and the beams' choice without a GPU: every refused
argument of the C entry points, the bounds and index functions that the kernels
share (compiled for the host), and the tests' own restatement."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

import paged_ref as ref
from fleet_moe import _lib

ROOT = Path(__file__).resolve().parents[1]
P = 1 << 20                         # a well aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    a = dict(pool=P, table=P, lens=P, refs=P, n_pages=64, n_layers=2, n_seqs=4, max_pages=8)
    return _lib.FleetCache(**{**a, **kw})


BAD_CACHES = [dict(pool=None), dict(pool=P + 8), dict(table=None), dict(table=P + 2),
              dict(lens=None), dict(lens=P + 1), dict(refs=None), dict(refs=P + 2),
              dict(n_pages=0), dict(n_pages=(1 << 24) + 1), dict(n_layers=0), dict(n_layers=65),
              dict(n_seqs=0), dict(n_seqs=1025), dict(max_pages=0), dict(max_pages=(1 << 20) + 1)]


def test_workspace_sizes(lib):
    n = lib.fleet_cache_workspace_bytes(64, 4)
    assert n % 256 == 0 and (32 << 20) < n < (36 << 20)
    assert lib.fleet_cache_workspace_bytes(1 << 20, 1024) > n
    for pages, seqs in ((0, 4), (64, 0), (-1, 4), (64, 1025), ((1 << 24) + 1, 4)):
        assert lib.fleet_cache_workspace_bytes(pages, seqs) == 0
    assert lib.fleet_beam_workspace_bytes(2, 4, 8, 102400) > 0
    for bad in ((0, 4, 4, 100), (1, 0, 4, 100), (1, 65, 4, 100), (1, 4, 0, 100), (1, 4, 65, 100),
                (1, 4, 4, 0), (1, 4, 4, (1 << 24) + 1), (1100, 64, 4, 100)):
        assert lib.fleet_beam_workspace_bytes(*bad) == 0, bad


def calls(lib, n):
    """Each entry point as a function of keyword changes to good arguments."""
    def remap(c=None, parents=P, ws=P, size=n):
        return lib.fleet_cache_remap(ctypes.byref(c or cache()), parents, ws, size, None)

    def grow(c=None, n_new=P, ws=P, size=n):
        return lib.fleet_cache_grow(ctypes.byref(c or cache()), n_new, ws, size, None)

    def compact(c=None, n_used=P, ws=P, size=n):
        return lib.fleet_cache_compact(ctypes.byref(c or cache()), n_used, ws, size, None)

    def rows(f):
        def call(c=None, layer0=0, layers=2, rows=P, row=576, step=576 * 10, start=P, n_rows=10,
                 ws=P, size=n):
            return f(ctypes.byref(c or cache()), layer0, layers, rows, row, step, start, n_rows,
                     ws, size, None)
        return call

    def attend(c=None, layer=1, q=P, stride=16 * 576, start=P, n_tokens=6, heads=16, max_len=0,
               window=0, sinks=0, scale=0.1, out=P, lse=P, ws=P, size=n):
        return lib.fleet_cache_attend(ctypes.byref(c or cache()), layer, q, stride, start,
                                      n_tokens, heads, max_len, window, sinks, scale, out, lse, ws,
                                      size, None)
    return dict(remap=remap, grow=grow, compact=compact, append=rows(lib.fleet_cache_append),
                read=rows(lib.fleet_cache_read), attend=attend)


def test_refused_caches_and_workspaces(lib):
    n = lib.fleet_cache_workspace_bytes(64, 4)
    for name, f in calls(lib, n).items():
        for kw in BAD_CACHES:
            assert f(c=cache(**kw)) == _lib.ERR_ARG, (name, kw)
        assert f(ws=None) == _lib.ERR_ARG and f(ws=P + 128) == _lib.ERR_ARG, name
        assert f(size=n - 1) == _lib.ERR_WORKSPACE, name


def test_refused_arguments(lib):
    f = calls(lib, lib.fleet_cache_workspace_bytes(64, 4))
    assert f["remap"](parents=None) == _lib.ERR_ARG and f["remap"](parents=P + 2) == _lib.ERR_ARG
    assert f["grow"](n_new=None) == _lib.ERR_ARG and f["grow"](n_new=P + 1) == _lib.ERR_ARG
    assert f["compact"](n_used=P + 2) == _lib.ERR_ARG
    for name in ("append", "read"):
        for kw in (dict(layer0=-1), dict(layer0=1), dict(layers=0), dict(layers=3), dict(rows=None),
                   dict(rows=P + 8), dict(row=568), dict(row=580), dict(row=1 << 33),
                   dict(step=576 * 10 - 8), dict(step=576 * 10 + 4), dict(step=-8),
                   dict(start=P + 2), dict(start=None), dict(n_rows=-1),
                   dict(n_rows=(1 << 28) + 1)):
            assert f[name](**kw) == _lib.ERR_ARG, (name, kw)
        assert f[name](n_rows=0, rows=None) == 0          # nothing to do
    for kw in (dict(layer=-1), dict(layer=2), dict(q=None), dict(q=P + 8), dict(stride=16 * 576 - 8),
               dict(stride=16 * 576 + 4), dict(start=P + 2), dict(start=None), dict(n_tokens=-1),
               dict(heads=0), dict(heads=129, stride=129 * 576), dict(n_tokens=(1 << 22) + 1),
               dict(max_len=-1), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(out=None), dict(out=P + 4), dict(lse=P + 2)):
        assert f["attend"](**kw) == _lib.ERR_ARG, kw
    assert f["attend"](n_tokens=0, q=None) == 0


def test_beam_refusals(lib):
    n = lib.fleet_beam_workspace_bytes(2, 4, 8, 1000)

    def call(**kw):
        a = {**dict(logits=P, ld=1000, scores=P, finished=P, groups=2, beams=4, out=8, vocab=1000,
                    eos=1, o=P, parents=P, tokens=P, ended=P, ws=P, size=n), **kw}
        return lib.fleet_beam_select(a["logits"], a["ld"], a["scores"], a["finished"], a["groups"],
                                     a["beams"], a["out"], a["vocab"], a["eos"], a["o"],
                                     a["parents"], a["tokens"], a["ended"], a["ws"], a["size"],
                                     None)
    for kw in (dict(logits=None), dict(logits=P + 2), dict(ld=999), dict(ld=1 << 41),
               dict(scores=None), dict(scores=P + 1), dict(groups=0), dict(beams=0),
               dict(beams=65), dict(out=0), dict(out=65), dict(vocab=0), dict(eos=1000),
               dict(o=None), dict(o=P + 2), dict(parents=None), dict(parents=P + 1),
               dict(tokens=None), dict(tokens=P + 3), dict(ws=None), dict(ws=P + 64),
               dict(groups=16384, beams=4)):
        assert call(**kw) == _lib.ERR_ARG, kw
    assert call(size=n - 1) == _lib.ERR_WORKSPACE


HOST = r"""
#include <cstdio>
#include <initializer_list>
#include "cache_pages.h"
using namespace fleet_moe::cache;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    // lengths and pages that the kernels refuse
    CHECK(checked_len(0, 4) == 0 && checked_len(256, 4) == 256);
    CHECK(checked_len(257, 4) == -1 && checked_len(-1, 4) == -1);
    CHECK(checked_len(2147483647, 1 << 20) == -1);
    CHECK(page_offset(-1, 8, 0, 3) == -1 && page_offset(8, 8, 0, 3) == -1);
    CHECK(page_offset(-2147483647 - 1, 8, 0, 3) == -1 && page_offset(2147483647, 8, 0, 3) == -1);
    CHECK(page_offset(7, 8, 2, 3) == 23ll * 36992);
    CHECK(page_offset((1 << 24) - 1, 1 << 24, 26, 27) == ((((int64_t)1 << 24) - 1) * 27 + 26) * 36992);
    CHECK(clamp_row(-5, 10) == 0 && clamp_row(11, 10) == 10 && clamp_row(7, 10) == 7);
    // every item of every ragged layout has a unit of its sequence, and no unit two
    const int counts[] = {0, 1, 2, 3, 15, 16, 17, 31, 33, 64, 100};
    for (int mul : {1, 5, 16, 24, 128}) for (int div : {16, 64}) {
        const int pad = mul % div != 0;
        int start = 0, s = 0;
        for (int rep = 0; rep < 3; ++rep) for (int n : counts) {
            const int64_t units = ((int64_t)n * mul + div - 1) / div;
            const int64_t a = first_unit(start, s, mul, div, pad);
            const int64_t b = first_unit(start + n, s + 1, mul, div, pad);
            CHECK(b - a >= units);
            start += n; ++s;
        }
    }
    // append: n rows from any place in a block
    for (int a = 0; a < 40; ++a) for (int n = 1; n < 70; ++n) for (int off = 0; off < 16; ++off) {
        const int64_t have = first_unit(a + n, 1, 1, 16, 2) - first_unit(a, 0, 1, 16, 2);
        CHECK(have >= (off + n + 15) / 16);
    }
    // what a token sees
    for (int pos = 0; pos < 50; ++pos) for (int w = 0; w < 60; ++w) for (int k = 0; k < 60; ++k) {
        const Seen s = seen_of(pos, w, k);
        CHECK(0 <= s.sink && s.sink <= s.lo && s.lo <= pos);
        for (int p = 0; p <= pos; ++p)
            CHECK((p >= s.lo || p < s.sink) == (w == 0 || p > pos - w || p < k));
    }
    CHECK(seen_of(2147483647, 2147483647, 2147483647).lo == 1);
    CHECK(seen_of(5, 2147483647, 0).lo == 0);
    // the least exponent, over every finite bf16 magnitude
    for (unsigned b = 0; b < 0x7f80; ++b) {
        const unsigned u = b << 16;
        float f; __builtin_memcpy(&f, &u, 4);
        const int e = scale_exp(b);
        CHECK(e >= -110 && e <= 120);
        CHECK((double)f <= __builtin_ldexp(448.0, e));
        CHECK(e == -110 || (double)f > __builtin_ldexp(448.0, e - 1));
    }
    return 0;
}
"""


def test_bounds_and_indexes_on_the_host(tmp_path):
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(HOST)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{ROOT}/fleet-mi300x_amd/csrc", "-o", exe, src], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_restated_rounding():
    v = ref.VALUES
    ok = ~np.isnan(v)
    assert (v[ref.to_e4m3(v[ok])] == v[ok]).all()
    assert v[ref.to_e4m3(np.array([447.0, 448.0, 432.0, 2.0**-10, 2.0**-10 * 1.01, -17.0]))].tolist() \
        == [448.0, 448.0, 448.0, 0.0, 2.0**-9, -16.0]
    import torch
    x = np.random.default_rng(1).normal(size=4096) * 2.0 ** np.random.default_rng(2).integers(-12, 8, 4096)
    x = np.clip(x, -448, 448).astype(np.float32)
    t = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert (v[ref.to_e4m3(x)] == t).all()


def test_restated_pages():
    c = ref.Cache(6, 3, 2, 1)
    assert c.grow([10, 0, 0]) and c.rows[0] == [0]
    c.remap([0, 0, -1])
    assert list(c.refs()) == [2, 0, 0, 0, 0, 0]
    assert c.grow([1, 1, 0]) and c.rows == [[1], [0], []]    # the last holder keeps the page
    assert c.grow([0, 60, 0]) and c.rows[1] == [0, 2]
    assert not c.grow([0, 0, 200])                           # wider than the table
    c.remap([-1, 1, 5])
    assert c.compact() == 2 and c.rows == [[], [0, 1], []]


def test_status_bits_are_one_thing_each():
    """The header's bits, and those that kernels keep to themselves."""
    bits = {}
    files = [ROOT / "include" / "fleet_moe.h"] + sorted((ROOT / "fleet-mi300x_amd" / "csrc").iterdir())
    for f in files:
        if f.suffix not in (".h", ".hip"):
            continue
        for name, v in re.findall(r"(FLEET_MOE_ABORT_\w+|kAbort\w+)\s*(?:=\s*)?(0x[0-9a-fA-F]+)u?\b",
                                  f.read_text()):
            bits.setdefault(name, int(v, 16))
    assert {"FLEET_MOE_ABORT_NO_PAGE", "kAbortRouteMismatch"} <= set(bits)
    assert len(set(bits.values())) == len(bits) and all(v & (v - 1) == 0 for v in bits.values())
    for name in ("NO_PAGE", "BAD_PAGE", "POSITION", "BAD_ID"):
        assert getattr(_lib, f"ABORT_{name}") == bits[f"FLEET_MOE_ABORT_{name}"]

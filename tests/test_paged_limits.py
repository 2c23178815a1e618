"""The ends of the ranges that the paged cache's calls accept, without a GPU."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

from fleet_moe import _lib

ROOT = Path(__file__).resolve().parents[1]

ROWS = r"""
#include <cstdio>
#include "cache_pages.h"
using namespace fleet_moe::cache;
int main() {
    // every row of few heads, and the rows beside every token's first for the others
    for (int n = 1; n <= 128; ++n) {
        const uint64_t per = head_divisor(n);
        const int step = n < 4 ? 1 : n;
        for (int64_t at = 0; at < kMaxRows; at += step)
            for (int64_t row = at - (step > 1); row <= at; ++row)
                if (row >= 0 && token_of_row((int)row, per) != row / n) {
                    std::printf("%d heads, row %lld: %d\n", n, (long long)row,
                                token_of_row((int)row, per));
                    return 1;
                }
        if (token_of_row(kMaxRows - 1, per) != (kMaxRows - 1) / n) return 1;
    }
    return 0;
}
"""


def test_the_token_of_every_row(tmp_path):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(ROWS)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{ROOT}/fleet-mi300x_amd/csrc", "-o", exe, src], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_scales_that_are_no_number_in_base_2():
    """scale * log2(e) has to be finite: 2.3586e38 is the largest that is."""
    lib = _lib.load()
    n = lib.fleet_cache_workspace_bytes(64, 4)
    at = 1 << 20                    # a well aligned address that nothing reads
    cache = _lib.FleetCache(at, at, at, at, 64, 2, 4, 8)

    def call(scale, tokens):
        return lib.fleet_cache_attend(ctypes.byref(cache), 0, at, 16 * 576, at, tokens, 16, 0, 0, 0,
                                      scale, at, at, at, n, None)
    for scale in (2.36e38, 3.0e38, 3.4e38, float("inf"), float("nan"), 0.0, -1e-45):
        assert call(scale, 6) == _lib.ERR_ARG, scale
    for scale in (2.35e38, 1.0, 1e-38, 1e-45):
        assert call(scale, 0) == 0, scale           # (no tokens: nothing is launched)

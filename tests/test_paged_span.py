"""The keys that paged attention walks (csrc/paged_span.h), compiled for the
host: every visible key that the table holds, and no more tiles than it has."""

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "torch-mojo-backend_amd" / "csrc"
LAST = 0x7FFFFF00  # the last position

SOURCE = """
#include <algorithm>
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
#include "paged_span.h"
extern "C" int end_of(long long width, long long page) { return mi::table_end(width, page); }
extern "C" void span(int first, int last, int window, int sinks, int end, int tile, int* out, int most) {
  const mi::KeySpan s(first, last, window, sinks, end, tile);
  out[0] = s.tiles;
  for (int i = 0; i < s.tiles && i < most; ++i) out[i + 1] = s.tile(i);
}
extern "C" int sees(int pos, int j, int window, int sinks) { return mi::visible(pos, j, window, sinks); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("span")
    (d / "span.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Xassembler", "--noexecstack", f"-I{CSRC}",
                    str(d / "span.cpp"), "-o", str(d / "span.so")], check=True, timeout=120)
    lib = ctypes.CDLL(str(d / "span.so"))
    lib.end_of.argtypes = [ctypes.c_longlong] * 2
    return lib


def tiles(host, first, last, window, sinks, end, tile):
    out = (ctypes.c_int * 4096)()
    host.span(first, last, window, sinks, end, tile, out, 4095)
    return out[0], list(out[1:1 + min(out[0], 4095)])


def test_end_of_the_table(host):
    assert host.end_of(0, 16) == 0 and host.end_of(3, 16) == 48
    assert host.end_of(2 ** 31 - 1, 2 ** 31 - 1) == host.end_of(2 ** 27, 16) == LAST + 1


@pytest.mark.parametrize("tile", [16, 32])
def test_every_visible_key_once(host, tile):
    rng = random.Random(tile)
    for _ in range(3000):
        end = rng.choice([0, 1, 16, 48, 50, 300])
        first = rng.randrange(-1, 400)
        last = rng.choice([-1, first + rng.randrange(0, 40)])
        window, sinks = rng.choice([(0, 0), (rng.randrange(1, 100), rng.randrange(0, 150)), (1, 0), (399, 500)])
        n, got = tiles(host, first, last, window, sinks, end, tile)
        assert len(set(got)) == n == len(got) and n <= -(-end // tile) and all(0 <= t * tile < max(end, 1) for t in got)
        wanted = {j // tile for p in range(max(first, 0), last + 1) for j in range(min(p + 1, end))
                  if host.sees(p, j, window, sinks)}
        assert wanted <= set(got), (first, last, window, sinks, end)


@pytest.mark.parametrize("tile", [16, 32])
@pytest.mark.parametrize("pos", [48, 48 * 40, 2 ** 30, LAST])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 7), (100, 4), (2 ** 31 - 1, 4), (LAST, LAST), (1, LAST)])
def test_positions_past_the_table_walk_what_it_holds(host, tile, pos, window, sinks):
    for first in (pos, max(pos - 31, 0), -1):
        n, got = tiles(host, first, pos, window, sinks, host.end_of(3, 16), tile)
        assert n <= -(-48 // tile) and all(0 <= t * tile < 48 for t in got)

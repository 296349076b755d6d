"""How the slices of a gradient list go over launches, no GPU (the rule, compiled here for the
CPU): every element once, in grids that a launch can have, up to slices that pass one alone."""

import ctypes
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
THREADS, MOST = 256, 96
ROOM = (2 ** 32 - 1) // THREADS  # blocks a launch

SRC = r"""
#include "grad_slices.h"
extern "C" int walk(const int64_t* sizes, int count, int64_t chunk, int threads, int most, int back, int64_t* v, int room) {
  int n = 0, launch = 0;
  oxi::walk_slices([&](int i) { return sizes[i]; }, count, chunk, threads, most, back != 0,
                   [&](int i, int64_t e0, int64_t len, int64_t nb) {
                     if (n < room) {
                       int64_t* p = v + 5 * n;
                       p[0] = launch, p[1] = i, p[2] = e0, p[3] = len, p[4] = nb;
                     }
                     ++n;
                   },
                   [&]() { ++launch; });
  return n;
}
extern "C" int64_t most_blocks(int64_t threads) { return oxi::most_blocks(threads); }
extern "C" int fits(int64_t blocks, int64_t threads) { return oxi::grid_fits(blocks, threads); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("slices")
    (d / "slices.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", f"-I{ROOT / 'oxitorch_amd' / 'csrc'}",
                    str(d / "slices.cpp"), "-o", str(d / "slices.so")], check=True)
    lib = ctypes.CDLL(str(d / "slices.so"))
    lib.most_blocks.restype = ctypes.c_int64
    return lib


def walk(lib, sizes, chunk, back):
    room = 4 * len(sizes) + 1000
    v = (ctypes.c_int64 * (5 * room))()
    n = lib.walk((ctypes.c_int64 * max(1, len(sizes)))(*sizes), len(sizes), ctypes.c_int64(chunk), THREADS, MOST, int(back),
                 v, room)
    assert n <= room
    return [tuple(v[5 * k:5 * k + 5]) for k in range(n)]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("chunk", [2048, 4096, 32768])
@pytest.mark.parametrize("sizes", [[], [0], [1], [2048, 0, 2049, 5], [7] * 300, [2 ** 35 - 4096], [2 ** 35 - 2048], [2 ** 35 + 1],
                                   [3, 2 ** 37 + 12345, 0, 4097], [2 ** 40], [2 ** 40, 2 ** 40 - 1], [2 ** 34] * 3],
                         ids=lambda s: f"{len(s)}x{max(s, default=0)}")
def test_every_element_once(lib, sizes, chunk, back):
    got = walk(lib, sizes, chunk, back)
    # launches by turns, each with pieces and with blocks that fit
    launches = [g[0] for g in got]
    assert launches == sorted(launches) and set(launches) == set(range(len(set(launches))))
    for k in set(launches):
        mine = [g for g in got if g[0] == k]
        blocks = sum(g[4] for g in mine)
        assert len(mine) <= MOST and 0 < blocks <= ROOM and lib.fits(ctypes.c_int64(blocks), ctypes.c_int64(THREADS))
    # in order or from the end; each slice's pieces lie one after the other, cut between chunks
    order = got[::-1] if back else got
    at = [(i, e0) for _, i, e0, _, _ in order]
    assert at == sorted(at)
    for i, n in enumerate(sizes):
        end = 0
        for _, _, e0, length, nb in (g for g in order if g[1] == i):
            assert e0 == end and e0 % chunk == 0 and length > 0 and nb == -(-length // chunk)
            end += length
        assert end == n
        # a slice that a launch takes is not cut
        assert sum(g[1] == i for g in got) == (0 if n == 0 else -(-(-(-n // chunk)) // ROOM))


def test_grids(lib):
    for threads in (1, 64, 256, 1024):
        most = lib.most_blocks(ctypes.c_int64(threads))
        assert most < 2 ** 31 and most * threads < 2 ** 32 and ((most + 1) * threads >= 2 ** 32 or most + 1 == 2 ** 31)
        assert lib.fits(ctypes.c_int64(most), ctypes.c_int64(threads)) and not lib.fits(ctypes.c_int64(most + 1), ctypes.c_int64(threads))

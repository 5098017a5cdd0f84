"""Which states a token of a sliding window reads, which rows read a state, and how the kernels' walks are cut into parts: the arithmetic of
csrc/mvr_span.cuh itself, compiled for the CPU, against the definition in whole numbers of any size."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

import medvision_b200

CSRC = os.path.join(os.path.dirname(os.path.abspath(medvision_b200.__file__)), "csrc")

SOURCE = r"""
#include "mvr_span.cuh"
#include <cstdint>
using namespace mvr;
struct Call {
  int N, T, L, G, Hk, D, sinks, sink_tiles, sink_parts, row_splits, row_tiles_per;
};
static Call call_of(const int64_t* a, WindowSizes& w) {  // N, T, L, G, Hk, D, before, after, sinks
  w = window_sizes(a[1], a[2], a[3], a[6], a[7], a[8]);
  Call p = {};
  p.N = (int)a[0]; p.T = (int)a[1]; p.L = (int)a[2]; p.G = (int)a[3]; p.Hk = (int)a[4]; p.D = (int)a[5];
  p.sinks = (int)w.sinks;
  return p;
}
extern "C" {
// the states of a token: lo, hi, sink
void token_states(const int64_t* a, int64_t offset, int64_t token, int64_t end, int* to) {
  WindowSizes w;
  const Call p = call_of(a, w);
  const Span s = span_of(p, places_from(offset, a[6], a[7]), (int)token, (int)token, (int)end);
  to[0] = s.lo; to[1] = s.hi; to[2] = s.sink;
}
void state_rows(const int64_t* a, int64_t offset, int64_t state, int* to) {
  WindowSizes w;
  const Call p = call_of(a, w);
  rows_of_state(p, places_from(offset, a[6], a[7]), (int)state, to[0], to[1]);
}
// A tile of `rows` rows from `first` on walks tiles of STEP states in `splits` parts: seen[j] counts the walks over state j.
int walk_states(const int64_t* a, int64_t offset, int64_t end, int first, int rows, int splits, int* seen) {
  constexpr int STEP = 64;
  WindowSizes w;
  const Call p = call_of(a, w);
  const int last = first + rows < p.T * p.G ? first + rows : p.T * p.G, per = (int)parts_of(w.span_tiles(rows, STEP), splits);
  const SpanTiles<STEP> tiles(span_of(p, places_from(offset, a[6], a[7]), first / p.G, (last - 1) / p.G, (int)end));
  for (int part = 0; part < splits; ++part)
    for (int i = part * per; i < (part + 1) * per && i < tiles.count; ++i)
      for (int j = tiles.first(i); j < tiles.first(i) + STEP && j < p.L; ++j) ++seen[j];
  return per * splits >= tiles.count;
}
// All CTAs of the gradients of keys and values: seen[n][tile][row] counts the walks over a row, place[n][part][j] where a state's sums go.
int walk_rows(const int64_t* a, const int64_t* offsets, const int64_t* ends, int tile, int step, int splits, int* seen, int64_t* place, int parts) {
  WindowSizes w;
  Call p = call_of(a, w);
  const int state_tiles = (p.L + tile - 1) / tile, rows = p.T * p.G;
  p.sink_tiles = (int)parts_of(w.sinks, tile);
  p.row_splits = splits;
  p.row_tiles_per = w.row_tiles(tile, step, splits);
  p.sink_parts = p.sink_tiles > 0 ? w.sink_parts(step, p.row_tiles_per) : 1;
  if (p.sink_parts > parts) return -1;
  const int ctas = p.N * (p.sink_tiles * p.sink_parts + (state_tiles - p.sink_tiles) * p.row_splits);
  for (int block = 0; block < ctas; ++block) {
    const StateTile s = state_tile(p, block, state_tiles);
    const Places at = places_from(offsets[s.n], a[6], a[7]);
    const int j0 = s.tile * tile;
    const TileRows r = rows_of_states(p, s, at, j0, tile, (int)ends[s.n], step);
    if (j0 < ends[s.n])  // (else the kernel walks nothing)
      for (int row = r.first; row < r.first + r.count * step && row < r.end; ++row) ++seen[((int64_t)s.n * state_tiles + s.tile) * rows + row];
    for (int j = j0; j < j0 + tile && j < p.L; ++j) {
      const PartPlace to = part_place(p, s, j, 0, tile);
      if (to.parts) place[((int64_t)s.n * parts + s.part) * p.L + j] = to.at;
    }
  }
  return p.sink_parts;
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    folder = tmp_path_factory.mktemp("places")
    source, built = folder / "places.cpp", folder / "places.so"
    source.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fwrapv", "-shared", "-fPIC", "-I", CSRC, "-o", str(built), str(source)])
    return ctypes.CDLL(str(built))


def numbers(values, kind=ctypes.c_int64):
    return (kind * len(values))(*values)


def call(N, T, L, G, before, after, sinks, Hk=1, D=1):
    return numbers([N, T, L, G, Hk, D, before, after, sinks])


def reads(j, place, before, after, sinks, end):
    return j < end and j <= place + after and (j >= place - before or j < sinks)


BIG = 2 ** 63 - 1
REACHES = [(0, 0), (5, 0), (0, 9), (40, 3), (10 ** 12, 0), (0, 10 ** 12), (2 ** 31 - 1, 2 ** 31), (2 ** 41 - 3, 2 ** 41), (BIG, BIG), (BIG - 4, 2)]
OFFSETS = [0, 3, -7, 30, 2 ** 31, -2 ** 31, 3 * 10 ** 9, -3 * 10 ** 9, 2 ** 40, -2 ** 40, 2 ** 41, -2 ** 41 - 2, 10 ** 18, -10 ** 18, BIG, -BIG - 1, BIG - 9, -BIG + 6]


@pytest.mark.parametrize("before,after", REACHES)
def test_states_and_rows_of_any_offset_and_reach(lib, before, after):
    T, L, G = 11, 50, 2
    near = [offset + s * reach + d for offset in (0, 20) for reach, s in ((before, 1), (after, -1)) for d in (-4, 0, 6)]  # (where a window's ends meet the states)
    for offset in OFFSETS + [o for o in near if -BIG - 1 <= o <= BIG]:
        for sinks in (0, 3, 10 ** 12):
            a = call(1, T, L, G, before, after, sinks)
            out = (ctypes.c_int * 3)()
            for end in (0, 1, 33, L):
                for t in range(T):
                    lib.token_states(a, ctypes.c_int64(offset), ctypes.c_int64(t), ctypes.c_int64(end), out)
                    got = [out[0] <= j < out[1] or j < out[2] for j in range(L)]
                    assert got == [reads(j, offset + t, before, after, sinks, end) for j in range(L)], (offset, sinks, end, t)
            for j in range(0, L, 7):
                lib.state_rows(a, ctypes.c_int64(offset), ctypes.c_int64(j), out)
                tokens = [t for t in range(T) if reads(j, offset + t, before, after, sinks, L)]
                rows = range(out[0], out[1])
                assert list(rows) == [t * G + g for t in tokens for g in range(G)], (offset, sinks, j)


def table(T, L, before, after, sinks, offset, end):
    """Token and state: whether it reads it."""
    place = [[offset + t] for t in range(T)]  # (numbers of any size)
    return np.array([[reads(j, p, before, after, sinks, end) for j in range(L)] for p, in place], dtype=bool).reshape(T, L)


def cases(seed, count):
    rng = random.Random(seed)
    for _ in range(count):
        T, L, G = rng.choice([1, 2, 33, 90, 150]), rng.choice([1, 40, 64, 130, 200]), rng.choice([1, 2, 3, 8])
        reach = lambda: rng.choice([0, 0, 7, 60, 500, 10 ** 12, BIG])  # noqa: E731
        before, after, sinks = reach(), reach(), rng.choice([0, 0, 1, 5, 70, 129, 10 ** 12])
        offset = rng.choice([0, 0, L - T, -20, 7, 300, 2 ** 33 - 20, -2 ** 33 + 20])
        yield T, L, G, before, after, sinks, offset, rng.choice([0, 1, L // 2, L, L])


def test_a_row_tile_walks_every_state_that_its_rows_read_once(lib):
    for T, L, G, before, after, sinks, offset, end in cases(0, 100):
        read = table(T, L, before, after, sinks, offset, end)
        for rows, splits in ((64, 1), (128, 3), (32, 5)):
            for first in range(0, T * G, rows):
                seen = (ctypes.c_int * L)()
                enough = lib.walk_states(call(1, T, L, G, before, after, sinks), ctypes.c_int64(offset), ctypes.c_int64(end), first, rows, splits, seen)
                assert enough and max(seen) <= 1
                needed = read[first // G:(min(first + rows, T * G) - 1) // G + 1].any(0)
                assert (np.array(seen)[needed] == 1).all()


def test_the_parts_of_a_state_tile_walk_every_row_that_reads_it_once(lib):
    together = 0
    for T, L, G, before, after, sinks, offset, end in cases(1, 120):
        N, rows, Hk, D = 2, T * G, 2, 3
        offsets, ends = [offset, max(offset - 3, -BIG)], [end, L]
        read = [table(T, L, before, after, sinks, o, e) for o, e in zip(offsets, ends)]
        a = call(N, T, L, G, before, after, sinks, Hk, D)
        for tile, step, splits in ((16, 8, 1), (32, 16, 2), (128, 64, 3), (64, 64, 2)):
            tiles, most = -(-L // tile), 64
            seen, place = (ctypes.c_int * (N * tiles * rows))(), (ctypes.c_int64 * (N * most * L))(*[-1] * (N * most * L))
            sink_parts = lib.walk_rows(a, numbers(offsets), numbers(ends), tile, step, splits, seen, place, most)
            assert sink_parts >= 1 and max(seen) <= 1
            together += splits > 1 and sink_parts > 1 and min(sinks, L) + tile < L
            walked = np.array(seen).reshape(N, tiles, T, G)
            for n in range(N):
                for i in range(tiles):
                    assert (walked[n, i] == read[n][:, i * tile:(i + 1) * tile].any(1)[:, None]).all()  # (others may hold anything)
            # a place of its own for every part's sums of every state, one behind another
            lead = min(L, -(-min(sinks, L) // tile) * tile)
            want = N * ((sink_parts * lead if sink_parts > 1 else 0) + (splits * (L - lead) if splits > 1 else 0))
            place = np.array(place)
            assert (np.sort(place[place >= 0]) == np.arange(want) * Hk * D).all()
    assert together > 10

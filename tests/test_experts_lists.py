"""What an experts' product reads out of its lists, compiled for the CPU and
compared with whole numbers of any size: the lists are the device's, and no value
of theirs may lead out of the buffers."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "dragonwing-edge-rs_amd" / "csrc"
INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1

# Undefined arithmetic ends the program.
FLAGS = ["-fsanitize=undefined", "-fno-sanitize-recover=undefined"]

SOURCE = """
#include <stdio.h>
#include <stdlib.h>
#include "expert_lists.h"
#include "kv_lists.h"

// rows of A and C of every entry given
static int rows(int argc, char** argv) {
  const uint32_t places = atoi(argv[2]), each = atoi(argv[3]);
  for (int i = 4; i < argc; ++i) {
    const int32_t entry = (int32_t)atoll(argv[i]);
    const dw::RowList list{&entry, places, each}, none{nullptr, places, each};
    printf("%u %d %u\\n", list.row(0), dw::row_named(entry, (int)places), none.row(i));
  }
  return 0;
}
// every tile of a grid
static int tiles(char** argv) {
  const int grid = atoi(argv[2]), all = atoi(argv[3]), columns = atoi(argv[4]);
  for (int id = 0; id < grid; ++id) {
    int tile;
    if (dw::tile_number(id, all, columns, &tile)) printf("%d\\n", tile);
  }
  return 0;
}
// an expert's places of each two offsets
static int shares(int argc, char** argv) {
  const int slots = atoi(argv[2]);
  for (int i = 3; i + 1 < argc; i += 2) {
    const dw::NewTokens t = dw::new_tokens((int)atoll(argv[i]), (int)atoll(argv[i + 1]), slots);
    printf("%d %d\\n", t.first, t.count);
  }
  return 0;
}
int main(int argc, char** argv) {
  return argv[1][0] == 'r' ? rows(argc, argv) : argv[1][0] == 't' ? tiles(argv) : shares(argc, argv);
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    at = tmp_path_factory.mktemp("expert_lists")
    (at / "lists.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", *FLAGS, "-D__host__=", "-D__device__=", "-D__forceinline__=inline",
                    f"-I{CSRC}", str(at / "lists.cpp"), "-o", str(at / "lists")], check=True)

    def go(*args):
        out = subprocess.run([str(at / "lists"), *map(str, args)], capture_output=True, text=True)
        assert out.returncode == 0, out.stderr
        return np.array([[int(v) for v in line.split()] for line in out.stdout.splitlines()], np.int64)

    return go


@pytest.mark.parametrize("places,each", [(1, 1), (24, 3), (127, 1), (1 << 24, 32)])
def test_rows_of_any_entry(run, places, each):
    entries = sorted({INT_MIN, INT_MIN + 1, -places, -1, 0, 1, each - 1, each, places - 1, places, places + 1, INT_MAX})
    for i, (entry, (row_a, row_c, unlisted)) in enumerate(zip(entries, run("rows", places, each, *entries))):
        named = 0 <= entry < places
        assert row_a == (entry // each if named else 0) and 0 <= row_a < max(1, places // each)
        assert row_c == entry if named else row_c < 0
        assert unlisted == i + 4


@pytest.mark.parametrize("rows,columns,more", [(1, 1, 0), (7, 1, 3), (8, 3, 0), (13, 5, 40), (100, 7, 9), (1, 1000, 1), (0, 4, 50)])
def test_each_tile_is_one_workgroups(run, rows, columns, more):
    tiles = run("tiles", rows * columns + more, rows, columns).reshape(-1)
    assert sorted(tiles) == list(range(rows * columns))


@pytest.mark.parametrize("rows,columns", [(1 << 24, 128), (1 << 24, 256), (1 << 28, 1 << 18), ((1 << 24) + 3, 257), (1 << 27, 31),
                                          ((1 << 28) - 1, (1 << 18) - 1)])
def test_tiles_of_more_than_31_bits_count(run, rows, columns):
    # lists that overlap: any tile that a workgroup takes is one of the rows' own, and taken once
    assert rows * columns >= 1 << 31
    tiles = run("tiles", 5000, rows, columns).reshape(-1)
    assert len(set(tiles)) == len(tiles)
    assert (tiles >= 0).all() and (tiles // columns < rows).all()


def test_places_of_any_offsets(run):
    slots = 1 << 24
    ends = [INT_MIN, -1, 0, 1, 16, 17, slots - 1, slots, slots + 1, INT_MAX]
    both = [(a, b) for a in ends for b in ends]
    for (a, b), (first, count) in zip(both, run("shares", slots, *[v for pair in both for v in pair])):
        own = range(max(a, 0), min(b, slots))
        assert count == len(own) and 0 <= first and first + count <= slots
        assert not len(own) or first == own[0]

"""What attention reads out of its lists, compiled for the CPU and compared
with whole numbers of any size: the lists are the device's, and no value of
theirs may lead out of the buffers."""
import ctypes as C
import itertools
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "dragonwing-edge-rs_amd" / "csrc"
INT_MIN, INT_MAX = -2 ** 31, 2 ** 31 - 1

SOURCE = """
#include "kv_lists.h"
extern "C" void span(int t0, int t1, int tokens, int* out) {
  const dw::NewTokens t = dw::new_tokens(t0, t1, tokens);
  out[0] = t.first, out[1] = t.count;
}
extern "C" int fits(int slot, int splits, int token, int head, int slots, int tokens, int heads) {
  return dw::entry_fits(slot, splits, token, head, slots, tokens, heads);
}
"""


@pytest.fixture(scope="module")
def lists(tmp_path_factory):
    at = tmp_path_factory.mktemp("kv_lists")
    (at / "lists.cpp").write_text(SOURCE)
    # -fwrapv: as the device's 32-bit instructions do it
    subprocess.run(["g++", "-O1", "-std=c++17", "-fwrapv", "-shared", "-fPIC", "-D__host__=", "-D__device__=",
                    "-D__forceinline__=inline", f"-I{CSRC}", str(at / "lists.cpp"), "-o", str(at / "lists.so")],
                   check=True)
    return C.CDLL(str(at / "lists.so"))


@pytest.mark.parametrize("tokens", [1, 6, 127, (1 << 24) - 1])
def test_new_tokens_of_any_list(lists, tokens):
    ends = sorted({INT_MIN, INT_MIN + 1, INT_MIN + 100, -16, -1, 0, 1, 5, 15, 16, 100, tokens - 1, tokens, tokens + 1,
                   INT_MAX - 15, INT_MAX - 1, INT_MAX})
    for t0, t1 in itertools.product(ends, ends):
        out = (C.c_int * 2)()
        lists.span(t0, t1, tokens, out)
        own = range(max(t0, 0), min(t1, tokens))  # the rows that the list gives the sequence
        assert out[1] == len(own), (t0, t1, list(out))
        assert 0 <= out[0] and out[0] + out[1] <= tokens
        if len(own):
            assert out[0] == own[0]


def test_entries_that_the_joins_follow(lists):
    # every place that is reached from an entry, in 32 bits as the device counts it, is one of the buffers'
    slots, tokens, heads, group, rows = 4160, 400, 4096, 128, 128
    wrap = lambda v: (v + 2 ** 31) % 2 ** 32 - 2 ** 31  # noqa: E731
    any_int = [INT_MIN, -1, 0, 1, 2, 7, 399, 400, 4095, 4096, 4158, 4160, INT_MAX - 126, INT_MAX]
    followed = 0
    for slot, splits, token, head in itertools.product(any_int, [0, 1, 2, 3, 4160, (1 << 24) - 1], any_int, any_int):
        if not lists.fits(slot, splits, token, head, slots, tokens, heads):
            continue
        followed += 1
        assert 0 <= slot and slot + splits <= slots
        for row in (0, group - 1, rows - 1):
            at, end = wrap(head + row), wrap((head // group + 1) * group)
            if at < end and at < heads:
                assert 0 <= at < heads and 0 <= token < tokens
    assert followed
    # what split kernels write is followed
    for slot, splits, token, head in ((0, 2, 0, 0), (slots - 2, 2, tokens - 1, heads - 1), (0, slots, 3, 16)):
        assert lists.fits(slot, splits, token, head, slots, tokens, heads)


def test_entries_whose_heads_would_wrap(lists):
    # a head of an int's last 127 wraps below 0 as rows count from it: such an entry must not be followed
    for head in range(INT_MAX - 126, INT_MAX + 1):
        assert not lists.fits(0, 2, 0, head, 16, 1, 4096)

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

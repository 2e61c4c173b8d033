"""Attention and append with lists at the ends of an int: any rows of a
sequence may come of them, but no access outside the buffers, and the rows
that no sequence has stay as they were."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import ops

pytestmark = pytest.mark.gpu

LEAST, MOST = -2 ** 31, 2 ** 31 - 1


def run(be, c, heads, start, lens, max_pages):
    """y over a pattern; the table has max_pages entries a sequence, the last ones no pages."""
    batch, t = len(lens), c.tokens
    table = np.full((batch, max_pages), -1, np.int32)
    table[:, :c.max_pages] = c.table[0]
    lists = [be.from_numpy(x) for x in (table, np.array(start, np.int32), np.array(lens, np.int32))]
    cache = [be.from_numpy(x) for x in (c.q["k"], c.s["k"], c.q["v"], c.s["v"])]
    sizes = (c.h, c.d, c.page, c.num_pages, max_pages)
    x = np.random.default_rng(1).normal(0, 1, (t, heads, c.d)).astype(np.float16)
    y = be.from_numpy(np.full(x.shape, 777, np.float16))
    ops.attention_mxfp4(be, be.from_numpy(x), heads * c.d, 0, *cache, *lists, y, t, batch, heads, *sizes, 0.1)
    row = 2 * c.h * c.d
    kv = be.from_numpy(np.random.default_rng(2).normal(0, 1, (t, row)).astype(np.float16))
    ops.kv_append_mxfp4(be, kv, row, 0, kv, row, row // 2, *cache, *lists, t, batch, *sizes)
    return be.to_numpy(y, np.float16, x.shape)


STARTS = [(100, LEAST), (5, LEAST), (15, LEAST + 3), (MOST, LEAST), (LEAST, MOST), (MOST, 3), (-1, LEAST),
          (LEAST, 2, LEAST, MOST), (3, LEAST, MOST, 1, LEAST), (MOST, MOST, LEAST, LEAST)]


# a wave for 16 rows, and tiles of 128 rows: few tokens, and enough for 6,144 steps of 64 keys
@pytest.mark.parametrize("tokens,heads,keys,pages", [(6, 2, 100, 9), (400, 16, 16384, 1024)])
@pytest.mark.parametrize("start", STARTS)
def test_starts_at_the_ends_of_an_int(backend, tokens, heads, keys, pages, start):
    c = ref.Cache(np.random.default_rng(3), [tokens], [keys], 1, 64, 16)
    for n in (keys, MOST, LEAST):
        y = run(backend, c, heads, start, [n] * (len(start) - 1), pages)
        owned = np.zeros(tokens, bool)
        for t0, t1 in zip(start, start[1:]):
            owned[max(t0, 0):max(0, min(t1, tokens))] = True
        assert (y[~owned] == 777).all()
    backend.synchronize()

"""Appending to an MXFP4 cache and attention over it against their
definitions in 64 bits, and the layer they are used in."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import HipError, ops

pytestmark = pytest.mark.gpu

F16 = ops.DTYPE_F16


def put(be, c):
    """The cache's buffers, in the order of the calls."""
    return [be.from_numpy(x) for x in (c.q["k"], c.s["k"], c.q["v"], c.s["v"], c.table, c.start, c.len)]


def sizes(c):
    return (c.h, c.d, c.page, c.num_pages, c.max_pages)


def attend(be, c, q, scale, causal=True, window=0, bufs=None, stride=None, off=0):
    """q [tokens, heads, d] f16 in rows of `stride` from column `off`; y comes back over a pattern."""
    t, heads, d = q.shape
    row = heads * d if stride is None else stride
    wide = np.full((t, row), np.nan, np.float16)
    wide[:, off:off + heads * d] = q.reshape(t, -1)
    y = be.from_numpy(np.full((t, heads, d), 777, np.float16))
    ops.attention_mxfp4(be, be.from_numpy(wide), row, off, *(bufs or put(be, c)), y, t, c.batch, heads, *sizes(c),
                        scale, causal=causal, window=window)
    return be.to_numpy(y, np.float16, (t, heads, d)).astype(np.float64)


def check(got, want, off):
    real = ~np.isnan(off).all((1, 2))
    bad = ~((np.abs(got - want) <= off) | (np.isnan(got) & np.isnan(want)))[real]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[real][bad][:3], want[real][bad][:3],
                           off[real][bad][:3])
    assert (got[~real] == 777).all()  # rows of no sequence


HEADS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (7, 1, 64), (16, 1, 256), (6, 2, 256), (40, 2, 64), (8, 8, 64)]


@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_one_new_token_each(backend, heads, kv_heads, d, page):
    rng = np.random.default_rng(heads * 100 + d + page)
    c = ref.Cache(rng, [1] * 9, [1, 2, 15, 16, 17, 33, 64, 129, 300], kv_heads, d, page)
    q = rng.normal(0, 1, (c.tokens, heads, d)).astype(np.float16)
    scale = d ** -0.5
    check(attend(backend, c, q, scale), *ref.attention(q.astype(np.float64), c, scale))


@pytest.mark.parametrize("kv", [1000, 1024, 4097, 9001])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 1, 128), (2, 2, 64), (3, 1, 256)])
def test_one_long_sequence(backend, kv, heads, kv_heads, d):
    rng = np.random.default_rng(kv + d)
    c = ref.Cache(rng, [1], [kv], kv_heads, d, 32)
    q = (rng.normal(0, 1, (1, heads, d)) * 3).astype(np.float16)
    check(attend(backend, c, q, d ** -0.5), *ref.attention(q.astype(np.float64), c, d ** -0.5))


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (5, 1, 128), (4, 2, 256), (24, 1, 64)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 19), (True, 64)])
def test_ragged_prompts(backend, heads, kv_heads, d, causal, window):
    rng = np.random.default_rng(heads + d + window)
    # a sequence without new tokens, one of a single token, one with a cached prefix, rows behind the last
    c = ref.Cache(rng, [17, 0, 1, 70, 5, 2], [17, 40, 100, 130, 261, 2], kv_heads, d, 16, extra=3)
    q = rng.normal(0, 1, (c.tokens, heads, d)).astype(np.float16)
    check(attend(backend, c, q, d ** -0.5, causal, window), *ref.attention(q.astype(np.float64), c, d ** -0.5, causal,
                                                                        window))


@pytest.mark.parametrize("n,kv,page", [(127, 127, 16), (128, 200, 128), (129, 129, 32), (257, 300, 256),
                                       (190, 1000, 64)])
def test_prompt_lengths(backend, n, kv, page):
    rng = np.random.default_rng(n)
    c = ref.Cache(rng, [n, 3], [kv, 50], 2, 128, page)
    q = rng.normal(0, 1, (c.tokens, 8, 128)).astype(np.float16)
    check(attend(backend, c, q, 128 ** -0.5), *ref.attention(q.astype(np.float64), c, 128 ** -0.5))


def test_strides_of_the_queries(backend):
    rng = np.random.default_rng(8)
    for nq, kv in (([1, 1, 1], [40, 3, 100]), ([60, 9], [60, 90])):
        c = ref.Cache(rng, nq, kv, 2, 128, 16)
        q = rng.normal(0, 1, (c.tokens, 4, 128)).astype(np.float16)
        want = ref.attention(q.astype(np.float64), c, 0.1)
        for stride, off in ((512, 0), (1024, 512), (777, 3), (515, 1)):
            check(attend(backend, c, q, 0.1, stride=stride, off=off), *want)


def test_rows_that_see_no_key_are_zero(backend):
    rng = np.random.default_rng(2)
    # no keys; fewer keys than new tokens (the first rows are before all); keys only
    c = ref.Cache(rng, [1, 4, 3, 2], [0, 2, 1, 30], 1, 64, 16)
    c.len[0] = -7  # and a length below zero
    q = rng.normal(0, 1, (c.tokens, 4, 64)).astype(np.float16)
    got = attend(backend, c, q, 0.125)
    want, off = ref.attention(q.astype(np.float64), c, 0.125)
    check(got, want, off)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[5:7] == 0).all() and (got[3] != 0).any()


def test_pages_outside_the_cache_are_seen_by_none(backend):
    rng = np.random.default_rng(4)
    for nq in ([1, 1], [40, 9]):
        c = ref.Cache(rng, nq, [100, 70], 2, 128, 16)
        q = rng.normal(0, 1, (c.tokens, 4, 128)).astype(np.float16)
        bufs = put(backend, c)
        table = c.table.copy()
        table[0, 1], table[1, 0], table[1, 4] = c.num_pages, -1, 2 ** 31 - 1
        bufs[4] = backend.from_numpy(table)
        got = attend(backend, c, q, 0.1, bufs=bufs)
        gone = [set(range(16, 32)), set(range(16)) | set(range(64, 80))]
        for r in range(c.tokens):
            b = int(np.searchsorted(c.start, r, side="right")) - 1
            pos = c.kv[b] - nq[b] + r - c.start[b]
            j = np.array([x for x in range(pos + 1) if x not in gone[b]], int)
            for h in range(4):
                if not len(j):
                    assert (got[r, h] == 0).all()
                    continue
                k, v = c.rows("k", b, h // 2)[j], c.rows("v", b, h // 2)[j]
                e = k @ q[r, h].astype(np.float64) * 0.1
                e = np.exp(e - e.max())
                # f16 of p and of the result, and scores good to 2^-14 of order one
                np.testing.assert_allclose(got[r, h], e @ v / e.sum(), rtol=2.0 ** -10, atol=8 * 2.0 ** -11)


@pytest.mark.parametrize("nq", [[1, 1, 1], [3, 2, 4], [50, 70, 20]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_keys_and_values_reach_only_rows_that_see_them(backend, nq, d):
    rng = np.random.default_rng(d + sum(nq))
    c = ref.Cache(rng, nq, [90, 120, 75], 2, d, 16)
    # a NaN block among the values of sequence 0's last token and of a middle token of sequence 2, a NaN key block in
    # the last but one of sequence 1
    p, s = c.table[0, 89 // 16], 89 % 16
    c.s["v"][p, 1, s, d // 32 - 1] = 255
    p, s = c.table[2, 60 // 16], 60 % 16
    c.s["v"][p, 0, s, 1] = 255
    p, s = c.table[1, 118 // 16], 118 % 16
    c.s["k"][p, 0, s, 0] = 255
    q = rng.normal(0, 1, (c.tokens, 4, d)).astype(np.float16)
    want, off = ref.attention(q.astype(np.float64), c, 0.1)
    got = attend(backend, c, q, 0.1)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    check(got, want, np.where(np.isnan(off), 0, off))
    assert np.isnan(got).any() and not np.isnan(got).all()


def test_scores_out_of_the_ordinary(backend):
    rng = np.random.default_rng(6)
    c = ref.Cache(rng, [1, 1, 1, 40], [70, 70, 70, 90], 1, 128, 16)
    q = rng.normal(0, 1, (c.tokens, 2, 128)).astype(np.float16)
    q[0, 0] *= 200  # one key takes all
    q[1, 0, 5] = np.nan
    q[2, 1] = 0
    q[20, 0, 7] = np.inf
    want, off = ref.attention(q.astype(np.float64), c, 1.0)
    got = attend(backend, c, q, 1.0)
    assert np.isnan(got[1, 0]).all() and np.isnan(got[20, 0]).all()
    ok = ~np.isnan(want)
    assert (np.abs(got - want)[ok] <= off[ok]).all()
    want, off = ref.attention(q.astype(np.float64), c, -0.3)  # a negative scale is a scale
    got = attend(backend, c, q, -0.3)
    ok = ~np.isnan(want)
    assert (np.abs(got - want)[ok] <= off[ok]).all()
    # scale 0: the mean of what is seen
    want, off = ref.attention(np.nan_to_num(q.astype(np.float64), posinf=0, nan=0), c, 0.0)
    check(attend(backend, c, np.nan_to_num(q, posinf=0, nan=0), 0.0), want, off)


def test_growing_scores(backend):
    # the running maximum moves at every tile, by far more than exp's range
    rng = np.random.default_rng(7)

    def values(name, shape):
        x = rng.normal(0, 1, shape + (64,))
        return x

    c = ref.Cache(rng, [1, 33], [700, 700], 1, 64, 16, values=values)
    for b in range(2):
        for j in range(700):
            x = np.full((1, 64), 6.0 * 2 ** (j / 100 - 3))
            qk, sk = ref.encode(x, -23)
            c.q["k"][c.table[b, j // 16], 0, j % 16], c.s["k"][c.table[b, j // 16], 0, j % 16] = qk[0], sk[0]
    q = np.full((c.tokens, 3, 64), 1.0, np.float16)
    q[:, 1] = -1
    q[:, 2] = 0.01
    check(attend(backend, c, q, 1.0), *ref.attention(q.astype(np.float64), c, 1.0))


@pytest.mark.parametrize("most", [1, 9])
def test_many_sequences(backend, most):
    # more than a wave has lanes, some without keys or new tokens
    rng = np.random.default_rng(most)
    nq = [int(x) for x in rng.integers(0, most + 1, 150)]
    kv = [n + int(x) for n, x in zip(nq, rng.integers(0, 90, 150))]
    kv[3] = kv[70] = 0
    kv[140] = 400
    c = ref.Cache(rng, nq, kv, 1, 64, 16, extra=1)
    q = rng.normal(0, 1, (c.tokens, 3, 64)).astype(np.float16)
    check(attend(backend, c, q, 0.125), *ref.attention(q.astype(np.float64), c, 0.125))


def test_many_sequences_of_many_new_tokens(backend):
    rng = np.random.default_rng(31)
    nq = [int(x) for x in rng.integers(0, 40, 80)]
    nq[5], nq[77] = 150, 140
    kv = [n + int(x) for n, x in zip(nq, rng.integers(0, 60, 80))]
    c = ref.Cache(rng, nq, kv, 2, 64, 16)
    q = rng.normal(0, 1, (c.tokens, 16, 64)).astype(np.float16)
    check(attend(backend, c, q, 0.125), *ref.attention(q.astype(np.float64), c, 0.125))


@pytest.mark.parametrize("nq", [[1, 2], [120, 9]])
@pytest.mark.parametrize("heads,kv_heads", [(160, 1), (256, 2), (34, 2)])
def test_many_heads_of_a_kv_head(backend, heads, kv_heads, nq):
    rng = np.random.default_rng(heads)
    c = ref.Cache(rng, nq, [150, 77], kv_heads, 64, 32)
    q = rng.normal(0, 1, (c.tokens, heads, 64)).astype(np.float16)
    check(attend(backend, c, q, 0.125), *ref.attention(q.astype(np.float64), c, 0.125))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 100)])
def test_prompts_of_many_heads(backend, d, causal, window):
    rng = np.random.default_rng(d + window)
    c = ref.Cache(rng, [260, 0, 131], [300, 20, 500], 2, d, 64, extra=2)
    q = rng.normal(0, 1, (c.tokens, 32, d)).astype(np.float16)
    check(attend(backend, c, q, d ** -0.5, causal, window), *ref.attention(q.astype(np.float64), c, d ** -0.5, causal,
                                                                        window))


def test_prompts_with_bad_pages_nan_and_empty_rows(backend):
    rng = np.random.default_rng(77)
    c = ref.Cache(rng, [300, 200], [280, 333], 1, 128, 16)
    for name, b, j, blk in (("v", 0, 250, 3), ("k", 0, 270, 1), ("v", 1, 300, 0)):
        c.s[name][c.table[b, j // 16], 0, j % 16, blk] = 255
    q = rng.normal(0, 1, (c.tokens, 32, 128)).astype(np.float16)
    want, off = ref.attention(q.astype(np.float64), c, 0.1)
    got = attend(backend, c, q, 0.1)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    check(got, want, np.where(np.isnan(off), 0, off))
    assert (got[:20] == 0).all()  # the first 20 of 300 new tokens have no key among 280
    # pages outside the cache: as if their keys were masked
    bufs = put(backend, c)
    table = c.table.copy()
    table[1, 2], table[1, 20] = c.num_pages, -3
    bufs[4] = backend.from_numpy(table)
    got = attend(backend, c, q, 0.1, bufs=bufs)
    r, h = 300 + 150, 5
    pos = 333 - 200 + 150
    j = np.array([x for x in range(pos + 1) if x // 16 not in (2, 20)])
    k, v = c.rows("k", 1, 0)[j], c.rows("v", 1, 0)[j]
    e = k @ q[r, h].astype(np.float64) * 0.1
    e = np.exp(e - e.max())
    np.testing.assert_allclose(got[r, h], e @ v / e.sum(), rtol=2.0 ** -10, atol=8 * 2.0 ** -11)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (7, 1, 128), (32, 2, 128), (3, 1, 256), (40, 1, 256)])
@pytest.mark.parametrize("kv", [65, 200, 512, 1000])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 70)])
def test_few_steps_of_keys(backend, heads, kv_heads, d, kv, causal, window):
    # few enough that a workgroup takes them whole, or just not
    rng = np.random.default_rng(heads + d + kv)
    c = ref.Cache(rng, [1, 0, 5, 2, 1], [kv, 3, kv // 2, 1, 40], kv_heads, d, 16, extra=1)
    for name, b, blk in (("v", 0, 0), ("k", 2, 1), ("v", 2, 1)):
        j = c.kv[b] - 1
        c.s[name][c.table[b, j // 16], 0, j % 16, blk] = 255
    q = rng.normal(0, 1, (c.tokens, heads, d)).astype(np.float16)
    want, off = ref.attention(q.astype(np.float64), c, d ** -0.5, causal, window)
    got = attend(backend, c, q, d ** -0.5, causal, window)
    np.testing.assert_array_equal(np.isnan(got)[:-1], np.isnan(want)[:-1])
    off[:-1][np.isnan(off[:-1])] = 0  # NaN where NaN is wanted; the last row is of no sequence
    check(got, want, off)


def large(rng, nq, kv, heads, kv_heads, d, page, window=0, extra=0):
    """A batch whose prompts are so long that tiles of 128 rows are used (6,144 steps of 64 keys), its queries, and some of
    its rows: all of the first and last tokens of each sequence, and 2% of the others."""
    c = ref.Cache(rng, nq, kv, kv_heads, d, page, extra=extra)
    group = heads // kv_heads
    tile = 128 // group
    assert sum(-(-n // tile) * kv_heads * max(1, -(-min(k, window + tile + 14 if window else k) // 64))
               for n, k in zip(nq, kv) if n * group >= 128) >= 6144
    q = rng.normal(0, 1, (c.tokens, heads, d)).astype(np.float16)
    some = rng.random((c.tokens, heads)) < 0.02
    for b in range(c.batch):
        some[c.start[b]:min(c.start[b] + 2, c.start[b + 1])] = True
        some[max(c.start[b], c.start[b + 1] - 2):c.start[b + 1]] = True
    return c, q, some


def check_some(got, want, off, some, owned):
    bad = ~((np.abs(got - want) <= off) | (np.isnan(got) & np.isnan(want)))[some]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[some][bad][:3], want[some][bad][:3])
    assert (got[owned:] == 777).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1000)])
def test_long_prompts_beside_single_tokens(backend, d, causal, window):
    rng = np.random.default_rng(d + window)
    nq, kv = [1300, 0, 1, 33, 1, 300, 15], [1400, 40, 2500, 2000, 1, 2100, 15]
    c, q, some = large(rng, nq, kv, 32, 4, d, 64, window, extra=2)
    some[-2:] = False
    want, off = ref.attention(q.astype(np.float64), c, d ** -0.5, causal, window, some)
    check_some(attend(backend, c, q, d ** -0.5, causal, window), want, off, some, c.start[-1])


@pytest.mark.parametrize("heads,kv_heads,nq,kv", [(8, 8, 1000, 6200), (7, 1, 900, 8200), (40, 1, 200, 6000), (100, 1, 200, 2200),
                                                  (128, 1, 190, 2100), (16, 1, 130, 24000)])
def test_groups_of_long_prompts(backend, heads, kv_heads, nq, kv):
    # the last: 17 tiles that split over their keys, and a single token's keys with them
    rng = np.random.default_rng(heads)
    c, q, some = large(rng, [nq, 1], [kv, 900], heads, kv_heads, 64, 32)
    want, off = ref.attention(q.astype(np.float64), c, 0.125, some=some)
    check_some(attend(backend, c, q, 0.125), want, off, some, c.start[-1])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_tiles_split_over_keys(backend, d):
    rng = np.random.default_rng(d)
    c, q, some = large(rng, [240, 5, 40], [12000, 3000, 11000], 16, 1, d, 128)
    want, off = ref.attention(q.astype(np.float64), c, d ** -0.5, some=some)
    got = attend(backend, c, q, d ** -0.5)
    check_some(got, want, off, some, c.start[-1])
    for _ in range(3):
        np.testing.assert_array_equal(attend(backend, c, q, d ** -0.5), got)


def test_long_prompts_with_bad_pages_nan_and_empty_rows(backend):
    rng = np.random.default_rng(77)
    c, q, some = large(rng, [600, 200, 1], [580, 17000, 3000], 16, 1, 128, 16)
    for name, b, j, blk in (("v", 0, 550, 3), ("k", 0, 570, 1), ("v", 1, 16950, 0), ("v", 2, 77, 2)):
        c.s[name][c.table[b, j // 16], 0, j % 16, blk] = 255
    # a factor past f16 where only some rows see the value, behind those that are compared
    c.s["v"][c.table[1, 16990 // 16], 0, 16990 % 16, 1] = 200
    some[790:800] = False
    want, off = ref.attention(q.astype(np.float64), c, 0.1, some=some)
    got = attend(backend, c, q, 0.1)
    np.testing.assert_array_equal(np.isnan(got)[some], np.isnan(want)[some])
    check_some(got, want, np.where(np.isnan(off), 0, off), some, c.start[-1])
    assert (got[:20] == 0).all()  # the first 20 of 600 new tokens have no key among 580
    # pages outside the cache: as if their keys were masked
    bufs = put(backend, c)
    table = c.table.copy()
    table[1, 2], table[1, 700] = c.num_pages, -3
    bufs[4] = backend.from_numpy(table)
    got = attend(backend, c, q, 0.1, bufs=bufs)
    r, h = 600 + 20, 5
    j = np.array([x for x in range(17000 - 200 + 20 + 1) if x // 16 not in (2, 700)])
    k, v = c.rows("k", 1, 0)[j], c.rows("v", 1, 0)[j]
    e = k @ q[r, h].astype(np.float64) * 0.1
    e = np.exp(e - e.max())
    np.testing.assert_allclose(got[r, h], e @ v / e.sum(), rtol=2.0 ** -10, atol=8 * 2.0 ** -11)


def test_growing_scores_of_a_long_prompt(backend):
    rng = np.random.default_rng(7)
    c, q, some = large(rng, [1000], [3200], 16, 1, 64, 16)
    j = np.arange(3200)
    x, s = ref.encode(np.full((1, 64), 6.0) * 2.0 ** (j[:, None] / 400 - 3), -23)
    c.q["k"][c.table[0, j // 16], 0, j % 16], c.s["k"][c.table[0, j // 16], 0, j % 16] = x, s
    q[:] = 1
    q[:, 1::3] = -1
    q[:, 2::3] = 0.01
    want, off = ref.attention(q.astype(np.float64), c, 1.0, some=some)
    check_some(attend(backend, c, q, 1.0), want, off, some, 1000)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-40])
def test_scales_out_of_the_ordinary(backend, scale):
    rng = np.random.default_rng(4)
    c = ref.Cache(rng, [1, 30, 4], [90, 40, 3], 2, 64, 16)
    q = rng.normal(0, 1, (c.tokens, 6, 64)).astype(np.float16)
    check(attend(backend, c, q, scale), *ref.attention(q.astype(np.float64), c, scale))


def test_lists_that_overlap_stay_in_bounds(backend):
    # as many sequences as tokens, each of them all tokens: more work than a grid is made for
    rng = np.random.default_rng(3)
    c = ref.Cache(rng, [400] + [0] * 39, [4000] + [0] * 39, 1, 64, 16)
    q = rng.normal(0, 1, (c.tokens, 16, 64)).astype(np.float16)
    for first in (0, -7):
        bufs = put(backend, c)
        start = np.full(41, 400, np.int32)
        start[:40:2] = first
        bufs[5], bufs[6] = backend.from_numpy(start), backend.from_numpy(np.full(40, 4000, np.int32))
        bufs[4] = backend.from_numpy(np.tile(c.table[:1], (40, 1)))
        attend(backend, c, q, 0.1, bufs=bufs)
        attend(backend, c, q[:, :2].copy(), 0.1, bufs=bufs)
    backend.synchronize()


def test_long_splits(backend):
    # so many steps that a split takes more than its first 1,024 keys' pages; some heads against the oracle
    rng = np.random.default_rng(15)
    batch, hk, d, page, keys = 64, 8, 64, 64, 4700
    pages = -(-keys // page)
    n = batch * pages
    table = rng.permutation(n).astype(np.int32).reshape(batch, pages)
    q8 = {x: rng.integers(0, 256, (n, hk, page, d // 2), dtype=np.uint8) for x in "kv"}
    s8 = {x: rng.integers(121, 127, (n, hk, page, d // 32), dtype=np.uint8) for x in "kv"}
    bufs = [backend.from_numpy(x) for x in (q8["k"], s8["k"], q8["v"], s8["v"], table,
                                            np.arange(batch + 1, dtype=np.int32), np.full(batch, keys, np.int32))]
    q = rng.normal(0, 1, (batch, hk, d)).astype(np.float16)
    y = backend.alloc(q.nbytes)
    ops.attention_mxfp4(backend, backend.from_numpy(q), hk * d, 0, *bufs, y, batch, batch, hk, hk, d, page, n, pages,
                        0.125)
    got = backend.to_numpy(y, np.float16, q.shape).astype(np.float64)
    for b, h in ((0, 0), (7, 3), (31, 7), (63, 1)):
        k, v = (ref.decode(q8[x][table[b], h], s8[x][table[b], h], d).reshape(-1, d)[:keys] for x in "kv")
        s = k @ q[b, h].astype(np.float64) * 0.125
        e = np.exp(s - s.max())
        want, mean = e @ v / e.sum(), e @ np.abs(v) / e.sum()
        off = mean * (2.0 ** -11 + 2 * (d + 3) * 2.0 ** -23 * (np.abs(k) @ np.abs(q[b, h].astype(np.float64))).max() / 8
                      + 2.0 ** -20 + keys * 2.0 ** -23) + keys * 2.0 ** -25 * np.abs(v).max() / e.sum()
        assert (np.abs(got[b, h] - want) <= off + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()


def test_a_cache_past_32_bit_offsets(backend):
    # pages of 256 KiB, the last ones past 2^32 bytes: appended to, then attended over
    rng = np.random.default_rng(9)
    hk, d, page, n = 8, 256, 256, 17000
    rows = n * hk * page
    bufs = [backend.alloc(rows * x) for x in (d // 2, d // 32, d // 2, d // 32)]
    table = np.array([[n - 1, 3, n - 2]], np.int32)
    t = 600
    lists = [backend.from_numpy(x) for x in (table, np.array([0, t], np.int32), np.array([t], np.int32))]
    kv = rng.normal(0, 1, (t, 2, hk, d)).astype(np.float16)
    bkv = backend.from_numpy(kv)
    ops.kv_append_mxfp4(backend, bkv, 2 * hk * d, 0, bkv, 2 * hk * d, hk * d, *bufs, *lists, t, 1, hk, d, page, n, 3)
    q = rng.normal(0, 1, (1, hk, d)).astype(np.float16)
    y = backend.alloc(q.nbytes)
    lists[1] = backend.from_numpy(np.array([0, 1], np.int32))
    ops.attention_mxfp4(backend, backend.from_numpy(q), hk * d, 0, *bufs, *lists, y, 1, 1, hk, hk, d, page, n, 3, 0.06)
    got = backend.to_numpy(y, np.float16, q.shape).astype(np.float64)
    for b in bufs:
        b.free()
    for h in range(hk):
        k, v = (ref.decode(*ref.encode(kv[:, i, h].astype(np.float64), -23), d) for i in (0, 1))
        s = k @ q[0, h].astype(np.float64) * 0.06
        e = np.exp(s - s.max())
        want, mean = e @ v / e.sum(), e @ np.abs(v) / e.sum()
        assert (np.abs(got[0, h] - want) <= 1.5 * 2.0 ** -11 * mean + t * 2.0 ** -25 * 8 + 2.0 ** -11 * np.abs(want)).all()


def test_two_backends_at_once(backend):
    import dragonwing_edge_rs_amd as dw
    rng = np.random.default_rng(44)
    other = dw.Backend(0)
    c = ref.Cache(rng, [1, 1, 3], [900, 40, 77], 2, 128, 16)
    q = rng.normal(0, 1, (c.tokens, 8, 128)).astype(np.float16)
    want = attend(backend, c, q, 0.1)
    state = []
    for be in (backend, other):
        y = be.alloc(c.tokens * 8 * 128 * 2)
        state.append((be, be.from_numpy(q), put(be, c), y))
    for _ in range(20):
        for be, bq, bufs, y in state:
            ops.attention_mxfp4(be, bq, 1024, 0, *bufs, y, c.tokens, c.batch, 8, *sizes(c), 0.1)
    for be, _, _, y in state:
        np.testing.assert_array_equal(be.to_numpy(y, np.float16, q.shape).astype(np.float64), want)
    del state, y
    other.close()


def test_attention_is_the_same_every_time(backend):
    rng = np.random.default_rng(12)
    for nq, kv in (([1, 1], [5000, 77]), ([100, 30], [700, 30])):
        c = ref.Cache(rng, nq, kv, 2, 128, 32)
        q = rng.normal(0, 1, (c.tokens, 8, 128)).astype(np.float16)
        first = attend(backend, c, q, 0.1)
        for _ in range(3):
            np.testing.assert_array_equal(attend(backend, c, q, 0.1), first)


@pytest.mark.parametrize("kv_heads,d,page", [(1, 64, 16), (3, 128, 32), (2, 256, 64)])
def test_append(backend, kv_heads, d, page):
    rng = np.random.default_rng(d)
    c = ref.Cache(rng, [1, 0, 40, 5, 3], [33, 20, 40, 70, 2], kv_heads, d, page, extra=2)
    c.table[3, 66 // page] = c.num_pages if page == 16 else c.table[3, 66 // page]  # a page outside the cache
    row, ko, vo = 2 * kv_heads * d + 9, 4, kv_heads * d + 7
    with np.errstate(over="ignore"):  # some are infinities: their blocks are NaN
        x = (rng.normal(0, 1, (c.tokens, row)) * np.exp(rng.normal(0, 4, (c.tokens, row)))).astype(np.float16)
    x[3, ko + 5] = np.inf
    x[4, vo + 40] = np.nan
    x[5, ko:ko + 64] = 0
    x[6, vo:vo + 32] = 2.0 ** -24  # below the least scale
    x[7, vo:vo + 32] = 65504
    bufs = put(backend, c)
    bx = backend.from_numpy(x)
    ops.kv_append_mxfp4(backend, bx, row, ko, bx, row, vo, *bufs, c.tokens, c.batch, *sizes(c))
    want = {n: (c.q[n].copy(), c.s[n].copy()) for n in "kv"}
    for b in range(c.batch):
        for i in range(c.nq[b]):
            pos = c.kv[b] - c.nq[b] + i
            if pos < 0 or not 0 <= c.table[b, pos // page] < c.num_pages:
                continue
            for n, o in (("k", ko), ("v", vo)):
                q, s = ref.encode(x[c.start[b] + i, o:o + kv_heads * d].reshape(kv_heads, d).astype(np.float64), -23)
                want[n][0][c.table[b, pos // page], :, pos % page] = q
                want[n][1][c.table[b, pos // page], :, pos % page] = s
    for n, at in (("k", 0), ("v", 2)):
        np.testing.assert_array_equal(backend.to_numpy(bufs[at], np.uint8, want[n][0].shape), want[n][0])
        np.testing.assert_array_equal(backend.to_numpy(bufs[at + 1], np.uint8, want[n][1].shape), want[n][1])


def test_lists_that_make_no_sense_stay_in_bounds(backend):
    # starts out of order or past the tokens, lengths past the table: any result, but no access outside
    rng = np.random.default_rng(3)
    c = ref.Cache(rng, [2, 3, 1], [20, 30, 9], 1, 64, 16)
    q = rng.normal(0, 1, (c.tokens, 2, 64)).astype(np.float16)
    for start, lens in (([5, 1, 900, -4], [20, 30, 9]), ([0, 2, 5, 6], [2 ** 31 - 1, -2 ** 31, 2 ** 30]),
                        ([-2 ** 31, 2 ** 31 - 1, 0, 6], [2 ** 31 - 1] * 3)):
        bufs = put(backend, c)
        bufs[5], bufs[6] = (backend.from_numpy(np.array(v, np.int32)) for v in (start, lens))
        attend(backend, c, q, 0.1, bufs=bufs)
        x = backend.from_numpy(rng.normal(0, 1, (c.tokens, 128)).astype(np.float16))
        ops.kv_append_mxfp4(backend, x, 128, 0, x, 128, 64, *bufs, c.tokens, c.batch, *sizes(c))
    backend.synchronize()


def test_refused_buffers(backend):
    rng = np.random.default_rng(3)
    c = ref.Cache(rng, [2, 3, 1], [20, 30, 9], 1, 64, 16)
    bufs = put(backend, c)
    x, y = backend.alloc(6 * 128 * 2), backend.alloc(6 * 2 * 64 * 2)

    def go(bufs, x=x, y=y, stride=128):
        ops.attention_mxfp4(backend, x, stride, 0, *bufs, y, 6, 3, 2, *sizes(c), 0.1)

    go(bufs)
    for i in range(7):
        wrong = list(bufs)
        wrong[i] = backend.alloc(bufs[i].len_bytes() + 4)
        with pytest.raises(HipError, match="mismatch"):
            go(wrong)
        with pytest.raises(HipError, match="mismatch"):
            ops.kv_append_mxfp4(backend, x, 128, 0, x, 128, 64, *wrong, 6, 3, *sizes(c))
        wrong[i] = None
        with pytest.raises(HipError, match="null buffer"):
            go(wrong)
    with pytest.raises(HipError, match="mismatch"):
        go(bufs, stride=129)
    with pytest.raises(HipError, match="is an input"):
        go(bufs, y=x)


def test_a_layer_of_them(backend):
    """A decoder layer's attention as a serving program runs it: a prompt, then single tokens, each step quantize ->
    product -> rotary positions in place -> append -> attention -> product; against the same steps in 64 bits from the
    device's own inputs to each step."""
    be, rng = backend, np.random.default_rng(21)
    hidden, hq, hk, d, page, batch, pages = 256, 8, 2, 64, 16, 2, 4
    row = (hq + 2 * hk) * d
    w1 = ref.encode(rng.normal(0, hidden ** -0.5, (row, hidden)))
    w2 = ref.encode(rng.normal(0, (hq * d) ** -0.5, (hidden, hq * d)))
    dev = [be.from_numpy(t) for t in (*w1, *w2)]
    npages = batch * pages
    table = rng.permutation(npages).astype(np.int32).reshape(batch, pages)
    shape = (npages, hk, page)
    cache = [be.from_numpy(np.full(shape + (n,), 255, np.uint8)) for n in (d // 2, d // 32, d // 2, d // 32)]
    btable = be.from_numpy(table)
    lens = [0, 0]
    hist = [[], []]  # keys and values of each sequence as quantized
    for nq in ([21, 9], [1, 1], [1, 1], [1, 3]):
        t = sum(nq)
        start = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
        lens = [a + b for a, b in zip(lens, nq)]
        x = rng.normal(0, 1, (t, hidden)).astype(np.float16)
        pos = np.concatenate([np.arange(m - n, m) for n, m in zip(nq, lens)]).astype(np.int32)
        pos = np.stack([pos, pos // 2, pos % 5]).astype(np.int32)
        bx, bq, bs = be.from_numpy(x), be.alloc(t * hidden // 2), be.alloc(t * hidden // 32)
        qkv, y, out = be.alloc(t * row * 2), be.alloc(t * hq * d * 2), be.alloc(t * hidden * 4)
        ops.quantize_mxfp4(be, F16, bx, bq, bs, t, hidden)
        ops.gemm_mxfp4(be, ops.DTYPE_MXFP4, bq, bs, dev[0], dev[1], None, F16, qkv, t, row, hidden)
        before = be.to_numpy(qkv, np.float16, (t, row))
        ops.rope_axes(be, F16, qkv, row, 0, qkv, row, 0, be.from_numpy(pos), t, hq + hk, d, d, (12, 10, 10))
        args = (btable, be.from_numpy(start), be.from_numpy(np.array(lens, np.int32)))
        ops.kv_append_mxfp4(be, qkv, row, hq * d, qkv, row, (hq + hk) * d, *cache, *args, t, batch, hk, d, page,
                            npages, pages)
        ops.attention_mxfp4(be, qkv, row, 0, *cache, *args, y, t, batch, hq, hk, d, page, npages, pages, d ** -0.5)
        ops.gemm_mxfp4(be, F16, y, None, dev[2], dev[3], None, ops.DTYPE_F32, out, t, hidden, hq * d)
        after = be.to_numpy(qkv, np.float16, (t, row))
        # the product
        a = ref.decode(*ref.encode(x.astype(np.float64)), hidden)
        want, off = ref.product(a, ref.decode(*w1, hidden))
        assert (np.abs(before - want) <= off + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
        # the positions
        src = before[:, :(hq + hk) * d].reshape(t, hq + hk, d).astype(np.float64)
        want = ref.rope(src, pos, d, (12, 10, 10))
        big = 2 * np.abs(src).max()
        assert (np.abs(after[:, :(hq + hk) * d].reshape(want.shape) - want)
                <= big * 2.0 ** -21 + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
        np.testing.assert_array_equal(after[:, (hq + hk) * d:], before[:, (hq + hk) * d:])
        # the cache and the attention
        c = ref.Cache(rng, nq, lens, hk, d, page)
        c.table, c.num_pages, c.max_pages = table, npages, pages
        c.q = {n: be.to_numpy(cache[i], np.uint8, shape + (d // 2,)) for n, i in (("k", 0), ("v", 2))}
        c.s = {n: be.to_numpy(cache[i], np.uint8, shape + (d // 32,)) for n, i in (("k", 1), ("v", 3))}
        kv = after[:, hq * d:].reshape(t, 2, hk, d).astype(np.float64)
        for b in range(batch):
            hist[b].append(ref.decode(*ref.encode(kv[start[b]:start[b + 1]].reshape(-1, d), -23), d).reshape(
                -1, 2, hk, d))
            whole = np.concatenate(hist[b])
            for h in range(hk):
                np.testing.assert_array_equal(c.rows("k", b, h), whole[:, 0, h])
                np.testing.assert_array_equal(c.rows("v", b, h), whole[:, 1, h])
        got = be.to_numpy(y, np.float16, (t, hq, d)).astype(np.float64)
        check(got, *ref.attention(after[:, :hq * d].reshape(t, hq, d).astype(np.float64), c, d ** -0.5))
        want, off = ref.product(got.reshape(t, -1), ref.decode(*w2, hq * d))
        assert (np.abs(be.to_numpy(out, np.float32, (t, hidden)) - want) <= off + np.abs(want) * 2.0 ** -24).all()

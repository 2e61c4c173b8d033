"""Attention where its exponentials are at their ends: scores far from 0, whose
products with the scale f32 rounds by whole numbers, and keys of a millionth of
the largest weight.  Queries, keys and scores are such that every score is an
f32 number with nothing rounded, so that what is left are the roundings that
the kernels state: p to f16 (2^-11 of it, 2^-31 of the largest at least), sums
in f32, the result to f16."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import ops

pytestmark = pytest.mark.gpu


def attend(be, c, q, scale, causal):
    t, heads, d = q.shape
    y = be.from_numpy(np.full(q.shape, 777, np.float16))
    ops.attention_mxfp4(be, be.from_numpy(q), heads * d, 0,
                        *[be.from_numpy(x) for x in (c.q["k"], c.s["k"], c.q["v"], c.s["v"], c.table, c.start, c.len)], y,
                        t, c.batch, heads, c.h, d, c.page, c.num_pages, c.max_pages, scale, causal=causal)
    return be.to_numpy(y, np.float16, q.shape).astype(np.float64)


def attention(scores, v, scale):
    """y of rows that see all keys, from scores [rows, keys] and values [keys, d], and its bound."""
    s = scores.astype(np.float64) * np.float64(np.float32(scale))
    e = np.exp(s - s.max(-1, keepdims=True))
    total = e.sum(-1, keepdims=True)
    y, mean = e @ v / total, e @ np.abs(v) / total
    n = len(v)
    # the exponent: (score - max) * scale log2(e), log2(e) and the product to 2^-24 of it, and exp2's own 2^-22
    arg = np.minimum(np.abs(s - s.max(-1, keepdims=True)), 120) * 2.0 ** -22 + 2.0 ** -21
    wide = (e * (2.0 ** -11 + arg)) @ np.abs(v) / total
    off = (wide + n * 2.0 ** -31 * np.abs(v).max(0) / total + mean * ((e * arg).sum(-1, keepdims=True) / total + (n + 8) * 2.0 ** -23)
           + 2.0 ** -11 * np.abs(y) + 2.0 ** -25)
    return y, off


# new tokens and keys of each sequence, heads, kv heads, keys the table has room for
SHAPES = [
    ([1], [5000], 4, 1, 0),                   # splits of one sequence, joined
    ([1], [300], 4, 1, 0),                    # a workgroup for a few steps
    ([1] * 300, [130] * 300, 2, 2, 0),        # a wave an item
    ([3, 1], [700, 200], 6, 2, 0),            # several tokens a tile
    ([300, 5], [6000, 4000], 16, 1, 0),       # tiles of 128 rows, and few rows beside them
]


def make(shape, d, key_of, value_of, seed):
    """A cache whose key j of a sequence is key_of(j) [d] and whose values are value_of(j)."""
    nq, kv, heads, kv_heads, _ = shape
    rng = np.random.default_rng(seed)
    c = ref.Cache(rng, nq, kv, kv_heads, d, 16)
    for b in range(c.batch):
        j = np.arange(c.kv[b])
        for name, f in (("k", key_of), ("v", value_of)):
            x, s = ref.encode(f(rng, j), -23)
            for h in range(kv_heads):
                c.q[name][c.table[b, j // 16], h, j % 16], c.s[name][c.table[b, j // 16], h, j % 16] = x, s
    return c


def check(be, c, q, scale):
    heads = q.shape[1]
    got = attend(be, c, q, scale, False)
    for b in range(c.batch):
        rows = np.arange(c.start[b], c.start[b + 1])
        for h in sorted({0, heads - 1}):
            k, v = c.rows("k", b, h // (heads // c.h)), c.rows("v", b, h // (heads // c.h))
            scores = q[rows, h].astype(np.float64) @ k.T
            assert (scores == scores.astype(np.float32)).all()
            y, off = attention(scores, v, scale)
            bad = ~(np.abs(got[rows, h] - y) <= off)
            assert not bad.any(), (b, h, int(bad.sum()), got[rows, h][bad][:4], y[bad][:4], off[bad][:4])
        if b == 3 and c.batch > 10:
            break  # the others are alike


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.125, 64.0, 1e30, 1e32])
def test_scores_far_from_zero(backend, shape, d, scale):
    # (d - 1) 2^19 + 0 to 48, many keys with the largest: a tie, and neighbours that count where the scale is 1
    steps = np.array([0, 8, 16, 24, 32, 48, 64, 96])

    def keys(rng, j):
        x = np.full((len(j), d), 64.0)
        x[:, 0] = steps[np.minimum(rng.integers(0, 8, len(j)), 3 + j * 5 // len(j))]  # the largest come late
        return x

    c = make(shape, d, keys, lambda rng, j: rng.normal(0, 1, (len(j), d)), d)
    q = np.full((c.tokens, shape[2], d), 8192.0, np.float16)
    q[:, :, 0] = max(0.5, d / 256)  # so that f32 holds the scores
    if scale < 0:
        q = -q
    check(backend, c, q, scale)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("low", [2.0, 4.0, 6.0])
def test_keys_of_a_millionth_of_the_largest_weight(backend, shape, d, low):
    # one key in 64 has all of the weight and a value of 0: the others' weights, 2^-18.5 to 2^-22.7 of it, are the result
    def keys(rng, j):
        x = np.zeros((len(j), d))
        x[:, 0] = np.where(j % 64 == 5, 24.0, low)
        return x

    def values(rng, j):
        return np.where((j % 64 == 5)[:, None], 0.0, 1024.0 * (1 + 5 * rng.random((len(j), d))))

    c = make(shape, d, keys, values, d + int(low))
    q = np.zeros((c.tokens, shape[2], d), np.float16)
    q[:, :, 0] = 1
    check(backend, c, q, 0.7145)

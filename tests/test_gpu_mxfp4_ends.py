"""Products with MXFP4 weights over all scales of the format, 2^-127 to 2^127,
with elements whose sums f32 holds exactly: the product of the definition has
to come out to the last bit."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import ops

pytestmark = pytest.mark.gpu

K = 64
NORMAL, TOP = 2.0 ** -126, 2.0 ** 128


def product(be, a, q, s, m, n):
    mx = isinstance(a, tuple)
    c = be.from_numpy(np.full((m, n), 777, np.float32))
    ops.gemm_mxfp4(be, ops.DTYPE_MXFP4 if mx else ops.DTYPE_F16, be.from_numpy(a[0] if mx else a),
                   be.from_numpy(a[1]) if mx else None, be.from_numpy(q), be.from_numpy(s), None, ops.DTYPE_F32, c, m, n,
                   K)
    return be.to_numpy(c, np.float32, (m, n)).astype(np.float64)


def weights(rng):
    """Row b of 256: random elements of scale byte b; the last row, of NaN, as quantize writes it (zeros)."""
    q = rng.integers(0, 256, (256, K // 2), dtype=np.uint8)
    q[255] = 0
    return q, np.repeat(np.arange(256, dtype=np.uint8)[:, None], K // 32, 1)


def check(got, a, w):
    """Exact where f32 has room: sums of magnitudes below 2^128, and 2^-126 where they go below the normal numbers."""
    want, size = a @ w.T, np.abs(a) @ np.abs(w).T
    assert np.isnan(got[:, 255]).all()
    room = size[:, :255] < TOP
    off = np.where(size[:, :255] < NORMAL * 2 ** 24, K * NORMAL, 0)  # terms of the sum may lie below 2^-126
    bad = room & ~(np.abs(got - want)[:, :255] <= off)
    assert not bad.any(), (int(bad.sum()), sorted(set(np.argwhere(bad)[:, 1].tolist())), np.argwhere(bad)[:4],
                           got[:, :255][bad][:4], want[:, :255][bad][:4])
    assert room.mean() > 0.8


@pytest.mark.parametrize("m", [1, 4, 5, 20, 40, 150])
@pytest.mark.parametrize("e", [-24, -14, -5, 5])
def test_f16_rows(backend, m, e):
    # all eleven bits of an f16 significand, subnormal numbers among them
    rng = np.random.default_rng(m + 100 * e + 10000)
    q, s = weights(rng)
    a = np.ldexp(rng.integers(-2047, 2048, (m, K)).astype(np.float64), e)
    a[:, ::7] = 0
    w = ref.decode(q, s, K)
    if e == -24:  # the largest scale too has sums that f32 holds
        assert (np.abs(a) @ np.abs(w[254]) < TOP).any()
    check(product(backend, a.astype(np.float16), q, s, m, 256), a, w)


@pytest.mark.parametrize("m", [1, 5, 20, 40, 150])
@pytest.mark.parametrize("e", [-24, -14, 5])
def test_f16_rows_and_scales_that_f16_holds(backend, m, e):
    # 2^-23 to 2^13: no other among them, so that the weights are widened to f16; its subnormal numbers too
    rng = np.random.default_rng(m + 100 * e + 10000)
    q, s = weights(rng)
    own = np.repeat(np.arange(104, 141), 3)
    q, s = q[own], s[own]
    a = np.ldexp(rng.integers(-2047, 2048, (m, K)).astype(np.float64), e)
    got = product(backend, a.astype(np.float16), q, s, m, len(own))
    np.testing.assert_array_equal(got, a @ ref.decode(q, s, K).T)


@pytest.mark.parametrize("m", [1, 20, 40, 150])
@pytest.mark.parametrize("byte", [0, 1, 60, 127, 190, 253, 254])
def test_mxfp4_rows(backend, m, byte):
    rng = np.random.default_rng(m + 1000 * byte)
    q, s = weights(rng)
    a = rng.integers(0, 256, (m, K // 2), dtype=np.uint8), np.full((m, K // 32), byte, np.uint8)
    got = product(backend, a, q, s, m, 256)
    wide, w = ref.decode(*a, K), ref.decode(q, s, K)
    want, size = wide @ w.T, np.abs(wide) @ np.abs(w).T
    assert np.isnan(got[:, 255]).all()
    room = size[:, :255] < TOP
    off = np.where(size[:, :255] < NORMAL * 2 ** 24, K * NORMAL, 0)
    bad = room & ~(np.abs(got - want)[:, :255] <= off)
    assert not bad.any(), (int(bad.sum()), sorted(set(np.argwhere(bad)[:, 1].tolist())), got[:, :255][bad][:4],
                           want[:, :255][bad][:4])

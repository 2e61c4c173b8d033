"""MXFP4 rows and products with MXFP4 weights against their definitions in
64 bits (tests/mxfp4_reference.py; no reference code exists for them)."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import HipError, ops

pytestmark = pytest.mark.gpu

F16, F32, MX = ops.DTYPE_F16, ops.DTYPE_F32, ops.DTYPE_MXFP4


def quantize(be, x):
    rows, k = x.shape
    nb = ref.blocks(k)
    bx, bq, bs = be.from_numpy(x), be.alloc(rows * nb * 16), be.alloc(rows * nb)
    be.upload(bq, np.full(rows * nb * 16, 0xA5, np.uint8))
    ops.quantize_mxfp4(be, F16 if x.dtype == np.float16 else F32, bx, bq, bs, rows, k)
    return be.to_numpy(bq, np.uint8, (rows, nb * 16)), be.to_numpy(bs, np.uint8, (rows, nb))


def dequantize(be, q, s, k, dtype):
    rows = q.shape[0]
    y = be.alloc(rows * k * np.dtype(dtype).itemsize)
    ops.dequantize_mxfp4(be, F16 if dtype == np.float16 else F32, be.from_numpy(q), be.from_numpy(s), y, rows, k)
    return be.to_numpy(y, dtype, (rows, k))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 64), (300, 7), (1000, 40), (7, 1023),
                                    (2, 4099), (129, 8192)])
def test_quantize_and_back(backend, rows, k, dtype):
    rng = np.random.default_rng(rows * 10007 + k)
    with np.errstate(over="ignore"):  # some f16 elements are infinities: their blocks are NaN
        x = (rng.normal(0, 1, (rows, k)) * np.exp(rng.normal(0, 3, (rows, k)))).astype(dtype)
    q, s = quantize(backend, x)
    rq, rs = ref.encode(x)
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(q, rq)
    want = ref.decode(q, s, k)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(dequantize(backend, q, s, k, np.float32), want.astype(np.float32))
        np.testing.assert_array_equal(dequantize(backend, q, s, k, np.float16), want.astype(np.float16))


def test_quantize_every_tie_and_edge(backend):
    # midpoints of the grid and their neighbours, at factors over f32's range
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999])
    v = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(9))])
    rows = []
    for e in (-130, -127, -126, -125, -60, -1, 0, 1, 60, 124, 125):
        for top in (4.0, 6.0, 7.9):
            r = np.zeros(64)
            r[:30] = np.ldexp(v, e)
            r[32:62] = -np.ldexp(v, e)
            r[31] = np.ldexp(top, e)
            r[63] = -np.ldexp(top, e)
            rows.append(r)
    rows.append(np.zeros(64))
    rows.append(np.full(64, -0.0))
    rows.append(np.full(64, np.finfo(np.float32).max))
    rows.append(np.full(64, 2.0 ** -149))
    x = np.array(rows).astype(np.float32)
    q, s = quantize(backend, x)
    rq, rs = ref.encode(x)
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(dequantize(backend, q, s, 64, np.float32), ref.decode(q, s, 64).astype(np.float32))


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_block_with_a_non_number_is_nan_and_only_it(backend, bad):
    x = np.random.default_rng(5).normal(0, 1, (3, 100)).astype(np.float32)
    x[1, 40] = bad
    x[2, 99] = bad
    q, s = quantize(backend, x)
    np.testing.assert_array_equal(q, ref.encode(x)[0])
    np.testing.assert_array_equal(s, ref.encode(x)[1])
    for dtype in (np.float16, np.float32):
        y = dequantize(backend, q, s, 100, dtype)
        want = np.zeros((3, 100), bool)
        want[1, 32:64] = True
        want[2, 96:] = True
        np.testing.assert_array_equal(np.isnan(y), want)


def test_every_byte_at_every_scale_back(backend):
    q = np.repeat(np.arange(256, dtype=np.uint8)[None], 256, 0).reshape(256, 256)
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, 1)
    want = ref.decode(q, s, 512)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(dequantize(backend, q, s, 512, np.float32), want.astype(np.float32))
        np.testing.assert_array_equal(dequantize(backend, q, s, 512, np.float16), want.astype(np.float16))


def weights(rng, n, k, spread=1.0):
    return ref.encode(rng.normal(0, 1 / np.sqrt(k), (n, k)) * np.exp(rng.normal(0, spread, (n, 1))))


def run_product(be, a, q, s, m, n, k, bias, act, dtype):
    """a: f16 rows, or (q, scales) of MXFP4 ones."""
    mx = isinstance(a, tuple)
    c = be.from_numpy(np.full((m, n), np.nan, dtype))
    ops.gemm_mxfp4(be, MX if mx else F16, be.from_numpy(a[0] if mx else a), be.from_numpy(a[1]) if mx else None,
                   be.from_numpy(q), be.from_numpy(s), None if bias is None else be.from_numpy(bias),
                   F16 if dtype == np.float16 else F32, c, m, n, k, act=act)
    return be.to_numpy(c, dtype, (m, n))


def check_product(got, want, off):
    # the sum's own error, then one rounding to the type of C (f16: half a step of 2^-10, or of the subnormals' 2^-24)
    e = np.finfo(got.dtype)
    tol = off + np.abs(want) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


SIZES = [(1, 1, 1), (1, 16, 32), (1, 17, 33), (2, 5, 31), (3, 100, 64), (1, 512, 4096), (5, 130, 1000), (15, 64, 96),
         (16, 48, 128), (17, 33, 129), (31, 200, 160), (33, 80, 257), (48, 64, 2050), (64, 65, 512), (65, 129, 288),
         (100, 300, 320), (127, 128, 256), (129, 257, 224), (200, 140, 999), (256, 512, 768), (300, 260, 1056),
         (513, 384, 320)]


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(backend, m, n, k, kind):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    q, s = weights(rng, n, k)
    w = ref.decode(q, s, k)
    a = (rng.normal(0, 1, (m, k)) * np.exp(rng.normal(0, 1, k))).astype(np.float16)
    wide = a.astype(np.float64)
    if kind == "mxfp4":
        a = ref.encode(wide)
        wide = ref.decode(*a, k)
    bias = rng.normal(0, 1, n)
    for dtype, use, act in ((np.float16, False, 0), (np.float32, True, 2), (np.float16, True, 1)):
        b = bias.astype(dtype) if use else None
        want, off = ref.product(wide, w, None if b is None else b.astype(np.float64), act)
        check_product(run_product(backend, a, q, s, m, n, k, b, act, dtype), want, off)


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(3303, 4001, 100), (1900, 7300, 288), (6500, 2050, 129), (70, 2050, 8200),
                                   (130, 1030, 14000), (31, 5301, 700), (13, 5200, 333), (40, 130, 33000)])
def test_large_product(backend, m, n, k, kind):
    # many tiles, and few with a long K that is shared
    rng = np.random.default_rng(m)
    q, s = weights(rng, n, k)
    a = rng.normal(0, 1, (m, k)).astype(np.float16)
    wide = a.astype(np.float64)
    if kind == "mxfp4":
        a = ref.encode(wide)
        wide = ref.decode(*a, k)
    b = rng.normal(0, 1, n).astype(np.float16)
    want, off = ref.product(wide, ref.decode(q, s, k), b.astype(np.float64), 2)
    check_product(run_product(backend, a, q, s, m, n, k, b, 2, np.float16), want, off)


@pytest.mark.parametrize("kind", ["f16", "mxfp4", "far"])
def test_product_on_the_largest_tiles(backend, kind):
    # enough tiles of 256 x 256 that they are chosen; "far": factors that f16 does not hold among them
    rng = np.random.default_rng(11)
    m, n, k = 4091, 8189, 136
    q, s = weights(rng, n, k, 0.1)
    a = rng.normal(0, 1, (m, k)).astype(np.float16)
    if kind == "far":
        s[n // 3, 2], s[n - 1, 4] = 90, 150
    wide = a.astype(np.float64)
    if kind == "mxfp4":
        a = ref.encode(wide)
        wide = ref.decode(*a, k)
    b = rng.normal(0, 1, n).astype(np.float32)
    want, off = ref.product(wide, ref.decode(q, s, k), b.astype(np.float64))
    check_product(run_product(backend, a, q, s, m, n, k, b, 0, np.float32), want, off)


@pytest.mark.parametrize("m", [1, 20, 150])
def test_silu_over_its_range(backend, m):
    # from -110 to 110, and infinities and NaN, as biases of products of zeros
    bias = np.linspace(-110, 110, 400).astype(np.float32)
    bias[[5, 77, 390]] = np.inf, -np.inf, np.nan
    q, s = ref.encode(np.zeros((400, 64)))
    a = np.zeros((m, 64), np.float16)
    got = run_product(backend, a, q, s, m, 400, 64, bias, 2, np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        y = bias.astype(np.float64)
        want = np.where(np.isinf(y), np.where(y > 0, y, np.nan), y / (1 + np.exp(-y)))
    np.testing.assert_array_equal(np.isnan(got), np.broadcast_to(np.isnan(want), got.shape))
    ok = np.isfinite(want)
    # where e^-y is no f32 number (above 2^128) it is infinite, and the quotient 0
    gone = np.where(y[ok] < -128 * np.log(2), np.abs(want[ok]), 0)
    assert (np.abs(got[:, ok] - want[ok]) <= 8 * 2.0 ** -24 * np.abs(want[ok]) + 2.0 ** -126 + gone).all()
    assert (got[:, want == np.inf] == np.inf).all()


def test_product_past_32_bit_offsets(backend):
    # rows of A that reach past 2^32 bytes: 1,024 rows again and again, so that the oracle is small
    rng = np.random.default_rng(5)
    m, n, k = 70 * 1024, 48, 32768
    q, s = weights(rng, n, k)
    part = rng.normal(0, 1, (1024, k)).astype(np.float16)
    ba, bc = backend.alloc(m * k * 2), backend.alloc(m * n * 4)
    backend.upload(ba, np.tile(part, (m // 1024, 1)))
    ops.gemm_mxfp4(backend, F16, ba, None, backend.from_numpy(q), backend.from_numpy(s), None, F32, bc, m, n, k)
    got = backend.to_numpy(bc, np.float32, (m // 1024, 1024, n))
    ba.free()
    np.testing.assert_array_equal(got, np.broadcast_to(got[:1], got.shape))
    check_product(got[0], *ref.product(part.astype(np.float64), ref.decode(q, s, k)))


def test_products_of_two_threads_on_one_backend(backend):
    import threading
    rng = np.random.default_rng(8)
    work = []
    for m, n, k in ((70, 300, 4100), (3, 500, 1001), (130, 200, 9000), (20, 900, 2050)):
        q, s = weights(rng, n, k)
        a = rng.normal(0, 1, (m, k)).astype(np.float16)
        work.append((a, q, s, m, n, k, run_product(backend, a, q, s, m, n, k, None, 0, np.float32)))
    bad = []

    def run(mine):
        for _ in range(10):
            for a, q, s, m, n, k, want in mine:
                if not np.array_equal(run_product(backend, a, q, s, m, n, k, None, 0, np.float32), want):
                    bad.append((m, n, k))

    threads = [threading.Thread(target=run, args=(w,)) for w in (work[:2], work[2:], work[::-1])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m", [1, 20, 150, 400])
def test_product_of_far_apart_scales(backend, m, kind):
    # factors of one row from 2^-60 to 2^60, and activations that make every
    # block of order one: a sum that loses a small factor is off by whole terms
    rng = np.random.default_rng(m)
    n, k = 70, 32 * 24
    e = rng.integers(-60, 60, (n, 1, k // 32))
    e[:] = e[:1]  # one factor a block of columns
    w = (rng.normal(0, 1, (n, k // 32, 32)) * np.ldexp(1.0, e[:, 0, :, None])).reshape(n, k)
    q, s = ref.encode(w)
    if kind == "mxfp4":
        a = ref.encode((rng.normal(0, 1, (m, k // 32, 32)) * np.ldexp(1.0, -e[:1, 0, :, None])).reshape(m, k))
        wide = ref.decode(*a, k)
    else:
        e16 = np.clip(-e[:1, 0, :, None], -14, 11)  # finite f16 rows
        a = (rng.normal(0, 1, (m, k // 32, 32)) * np.ldexp(1.0, e16)).reshape(m, k).astype(np.float16)
        wide = a.astype(np.float64)
    want, off = ref.product(wide, ref.decode(q, s, k))
    check_product(run_product(backend, a, q, s, m, n, k, None, 0, np.float32), want, off)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_product_of_rows_with_non_numbers(backend, m, value):
    rng = np.random.default_rng(3)
    n, k = 90, 320
    w = np.where(rng.random((n, k)) < 0.5, 1.0, 2.0)  # no zero, no sign: inf stays inf
    q, s = ref.encode(w)
    a = rng.normal(0, 1, (m, k)).astype(np.float16)
    a[m // 2, 77] = value
    got = run_product(backend, a, q, s, m, n, k, None, 0, np.float32)
    with np.errstate(invalid="ignore"):
        want = a.astype(np.float64) @ w.T
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.isinf(got), np.isinf(want))
    rest = [i for i in range(m) if i != m // 2]
    check_product(got[rest], *ref.product(a[rest].astype(np.float64), w))


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_with_nan_blocks(backend, m, kind):
    rng = np.random.default_rng(9)
    n, k = 80, 352
    q, s = weights(rng, n, k)
    s[11, 4] = 255
    a = rng.normal(0, 1, (m, k)).astype(np.float16)
    bad_rows = np.zeros(m, bool)
    wide = a.astype(np.float64)
    if kind == "mxfp4":
        a = ref.encode(wide)
        a[1][m - 1, 7] = 255
        bad_rows[m - 1] = True
        wide = ref.decode(*a, k)
    got = run_product(backend, a, q, s, m, n, k, None, 0, np.float32)
    want = np.zeros((m, n), bool)
    want[bad_rows] = True
    want[:, 11] = True
    np.testing.assert_array_equal(np.isnan(got), want)
    cols = [i for i in range(n) if i != 11]
    check_product(got[~bad_rows][:, cols], *ref.product(wide[~bad_rows], ref.decode(q, s, k)[cols]))


def test_product_is_the_same_every_time(backend):
    rng = np.random.default_rng(1)
    for m, n, k in ((1, 700, 2048), (24, 300, 4000), (260, 300, 512)):
        q, s = weights(rng, n, k)
        a = rng.normal(0, 1, (m, k)).astype(np.float16)
        first = run_product(backend, a, q, s, m, n, k, None, 0, np.float32)
        for _ in range(3):
            np.testing.assert_array_equal(run_product(backend, a, q, s, m, n, k, None, 0, np.float32), first)


def test_refused_buffers(backend):
    be = backend
    x, q, s = be.alloc(4 * 64 * 2), be.alloc(4 * 32), be.alloc(4 * 2)
    with pytest.raises(HipError, match="mismatch"):
        ops.quantize_mxfp4(be, F32, x, q, s, 4, 64)
    with pytest.raises(HipError, match="mismatch"):
        ops.quantize_mxfp4(be, F16, x, q, s, 4, 65)
    with pytest.raises(HipError, match="mismatch"):
        ops.dequantize_mxfp4(be, F16, q, s, x, 4, 63)
    c = be.alloc(4 * 4 * 2)
    ops.gemm_mxfp4(be, F16, x, None, q, s, None, F16, c, 4, 4, 64)
    with pytest.raises(HipError, match="mismatch"):
        ops.gemm_mxfp4(be, F16, x, None, q, s, None, F32, c, 4, 4, 64)
    with pytest.raises(HipError, match="mismatch"):
        ops.gemm_mxfp4(be, F16, x, None, q, s, s, F16, be.alloc(5 * 4 * 2), 4, 5, 64)
    with pytest.raises(HipError, match="operand"):
        ops.gemm_mxfp4(be, F16, x, None, be.alloc(64 * 32), be.alloc(64 * 2), None, F16, x, 4, 64, 64)
    tiny = be.alloc(3 * 16)
    with pytest.raises(HipError, match="overlap"):
        ops.quantize_mxfp4(be, F16, tiny, tiny, be.alloc(3), 3, 8)
    with pytest.raises(HipError, match="overlap"):
        ops.dequantize_mxfp4(be, F16, tiny, be.alloc(3), tiny, 3, 8)
    with pytest.raises(HipError, match="null buffer"):
        ops.gemm_mxfp4(be, F16, x, None, None, s, None, F16, c, 4, 4, 64)

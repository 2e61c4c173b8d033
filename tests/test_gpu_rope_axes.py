"""Rotary positions over several axes against their definition in 64 bits
(no reference code exists for them)."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import HipError, ops

pytestmark = pytest.mark.gpu

F16, F32 = ops.DTYPE_F16, ops.DTYPE_F32


def limit(x, y, rotary, dtype):
    """What an element may be off: the angle's fraction of a turn rounds to f32 (2^-25 of a turn, 2^-22.3 rad), sine
    and cosine are good to 4 half-ulps, two products and a sum round, and the result rounds to its type.  Each is
    relative to the pair's magnitudes, taken as twice the head's largest."""
    big = 2 * np.abs(x).max(-1, keepdims=True)
    e = np.finfo(dtype)
    return big * (2.0 ** -22.3 + 8 * 2.0 ** -24) + np.abs(y) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2


CASES = [
    # tokens, heads, dim, rotary, sections
    (1, 1, 64, 64, (32,)),
    (1, 40, 128, 128, (16, 24, 24)),
    (7, 5, 128, 128, (64, 0, 0)),
    (7, 5, 128, 128, (0, 40, 24)),
    (33, 3, 80, 72, (12, 12, 12)),
    (20, 3, 80, 40, (10, 10)),
    (5, 9, 96, 18, (3, 4, 2)),
    (9, 2, 67, 66, (11, 11, 11)),
    (3, 2, 5, 2, (1,)),
    (300, 12, 256, 256, (32, 48, 48)),
    (2, 2, 300, 256, (16, 16, 16, 16, 16, 16, 16, 16)),
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("tokens,heads,dim,rotary,sections", CASES)
def test_rope(backend, tokens, heads, dim, rotary, sections, dtype):
    rng = np.random.default_rng(tokens * 100 + heads + dim)
    x = rng.normal(0, 2, (tokens, heads, dim)).astype(dtype)
    pos = rng.integers(-1000, 1000, (len(sections), tokens)).astype(np.int32)
    pos[0] = rng.integers(0, 2 ** 31 - 1, tokens)  # far beyond what an f32 angle resolves
    bx, bp, by = backend.from_numpy(x), backend.from_numpy(pos), backend.alloc(x.nbytes)
    row = heads * dim
    for order, pairs, freq, base in ((0, 0, 0, 10000.0), (1, 1, 1, 500000.0), (1, 0, 0, 100.0), (0, 1, 1, 0.5)):
        ops.rope_axes(backend, F16 if dtype == np.float16 else F32, bx, row, 0, by, row, 0, bp, tokens, heads, dim,
                      rotary, sections, order=order, pairs=pairs, freq=freq, base=base)
        got = backend.to_numpy(by, dtype, x.shape).astype(np.float64)
        want = ref.rope(x.astype(np.float64), pos, rotary, sections, order, pairs, freq, base)
        tol = limit(x.astype(np.float64), want, rotary, dtype)
        # the angle itself: up to 2^31 / base turns in f64, products of up to 128 80-bit factors
        far = np.abs(pos).max() * max(1.0, 1 / base) / (2 * np.pi)
        tol = tol + 2 * np.abs(x).max() * 2 * np.pi * far * 2.0 ** -52
        assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
        np.testing.assert_array_equal(got[..., rotary:], x[..., rotary:].astype(np.float64))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (80, 40), (96, 18)])
def test_strided_columns_and_in_place(backend, dim, rotary, dtype):
    # queries and keys of a fused projection turn in place; the values and a
    # ragged end of the row are left as they were
    rng = np.random.default_rng(dim)
    t, hq, hk, tail = 13, 4, 2, 5
    row = (hq + 2 * hk) * dim + tail
    x = rng.normal(0, 1, (t, row)).astype(dtype)
    pos = rng.integers(0, 5000, (2, t)).astype(np.int32)
    half = rotary // 2
    sections = (half - half // 3, half // 3)
    buf, bp = backend.from_numpy(x), backend.from_numpy(pos)
    dt = F16 if dtype == np.float16 else F32
    ops.rope_axes(backend, dt, buf, row, 0, buf, row, 0, bp, t, hq + hk, dim, rotary, sections)
    got = backend.to_numpy(buf, dtype, x.shape)
    n = (hq + hk) * dim
    src = x[:, :n].reshape(t, hq + hk, dim).astype(np.float64)
    want = ref.rope(src, pos, rotary, sections)
    assert (np.abs(got[:, :n].reshape(want.shape) - want) <= limit(src, want, rotary, dtype)).all()
    np.testing.assert_array_equal(got[:, n:], x[:, n:])
    # from odd columns of one buffer to odd columns of another, whose other columns stay
    y0 = rng.normal(0, 1, (t, hk * dim + 7)).astype(dtype)
    by = backend.from_numpy(y0)
    bx = backend.from_numpy(x)
    ops.rope_axes(backend, dt, bx, row, hq * dim + 3, by, hk * dim + 7, 5, bp, t, hk, dim, rotary, sections)
    got = backend.to_numpy(by, dtype, y0.shape)
    src = x[:, hq * dim + 3:hq * dim + 3 + hk * dim].reshape(t, hk, dim).astype(np.float64)
    want = ref.rope(src, pos, rotary, sections)
    assert (np.abs(got[:, 5:5 + hk * dim].reshape(want.shape) - want) <= limit(src, want, rotary, dtype)).all()
    np.testing.assert_array_equal(got[:, :5], y0[:, :5])
    np.testing.assert_array_equal(got[:, 5 + hk * dim:], y0[:, 5 + hk * dim:])
    # to other columns of its own buffer
    wide = np.concatenate([x, y0], 1)
    w = wide.shape[1]
    bw = backend.from_numpy(wide)
    ops.rope_axes(backend, dt, bw, w, 0, bw, w, row + 2, bp, t, hk, dim, rotary, sections)
    got = backend.to_numpy(bw, dtype, wide.shape)
    src = x[:, :hk * dim].reshape(t, hk, dim).astype(np.float64)
    want = ref.rope(src, pos, rotary, sections)
    assert (np.abs(got[:, row + 2:row + 2 + hk * dim].reshape(want.shape) - want) <= limit(src, want, rotary,
                                                                                          dtype)).all()
    np.testing.assert_array_equal(got[:, :row + 2], wide[:, :row + 2])


def test_the_three_axes_are_one_where_their_positions_agree(backend):
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (11, 3, 128)).astype(np.float32)
    p = rng.integers(0, 9999, 11).astype(np.int32)
    out = []
    for sections, order in (((64,), 0), ((16, 24, 24), 0), ((24, 20, 20), 1)):
        by = backend.alloc(x.nbytes)
        ops.rope_axes(backend, F32, backend.from_numpy(x), 384, 0, by, 384, 0,
                      backend.from_numpy(np.stack([p] * len(sections))), 11, 3, 128, 128, sections, order=order)
        out.append(backend.to_numpy(by, np.float32, x.shape))
    np.testing.assert_array_equal(out[0], out[1])
    np.testing.assert_array_equal(out[0], out[2])


def test_refused_buffers(backend):
    x, p = backend.alloc(4 * 128 * 2), backend.alloc(2 * 4 * 4)
    with pytest.raises(HipError, match="mismatch"):
        ops.rope_axes(backend, F32, x, 128, 0, x, 128, 0, p, 4, 2, 64, 64, (16, 16))
    with pytest.raises(HipError, match="mismatch"):
        ops.rope_axes(backend, F16, x, 128, 0, x, 128, 0, p, 4, 2, 64, 64, (16, 8, 8))
    with pytest.raises(HipError, match="null buffer"):
        ops.rope_axes(backend, F16, x, 128, 0, x, 128, 0, None, 4, 2, 64, 64, (16, 16))
    z = backend.alloc(4 * 4 * 4)
    with pytest.raises(HipError, match="positions"):
        ops.rope_axes(backend, F16, backend.alloc(4 * 8 * 2), 8, 0, z, 8, 0, z, 4, 2, 4, 2, (1, 0, 0, 0))

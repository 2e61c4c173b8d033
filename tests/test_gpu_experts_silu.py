"""SiLU and the gated activation of experts' products over the whole range of f32
sums: the sums are the biases, since the rows are zeros."""
import numpy as np
import pytest

from dragonwing_edge_rs_amd import ops

pytestmark = pytest.mark.gpu

F16, F32, MX = ops.DTYPE_F16, ops.DTYPE_F32, ops.DTYPE_MXFP4
LOST = 2.0 ** -121  # values of SiLU below it may be


def sums(rng, n):
    """n sums: of order one, large ones of both signs, those whose SiLU is near f32's end, and special ones."""
    s = np.concatenate([rng.normal(0, 3, n // 4), rng.uniform(-110, 110, n // 4), rng.uniform(-92, -84, n // 4),
                        np.exp(rng.uniform(-80, 80, n)) * rng.choice([-1, 1], n)])[:n].astype(np.float32)
    s[:6] = 0, -0.0, np.inf, np.nan, 3e38, -3e38
    return s


def run(be, s, rows, k, mx, act, dtype):
    """act of the sums s [n], for each of `rows` rows of one expert."""
    n, blocks, half = s.size, -(-k // 32), dtype == np.float16
    cols = n // 2 if act == ops.ACT_SWIGLU else n
    a = be.from_numpy(np.zeros((rows, blocks * 16) if mx else (rows, k), np.uint8 if mx else np.float16))
    scales = be.from_numpy(np.full((rows, blocks), 127, np.uint8)) if mx else None
    w, ws = be.from_numpy(np.zeros((n, blocks * 16), np.uint8)), be.from_numpy(np.full((n, blocks), 127, np.uint8))
    c = be.from_numpy(np.full((rows, cols), 7.5, dtype))
    ops.gemm_mxfp4_experts(be, MX if mx else F16, a, scales, w, ws, be.from_numpy(s.astype(dtype)), F16 if half else F32, c,
                           be.from_numpy(np.array([0, rows], np.int32)), None, rows, 1, n, k, act=act)
    return be.to_numpy(c, dtype, (rows, cols))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("rows", [3, 40, 150, 300])  # each of the kernels
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_silu_of_all_sums(backend, rows, mx, dtype):
    rng = np.random.default_rng(rows)
    s = sums(rng, 3000)
    if dtype == np.float16:
        s = np.clip(s, -140, 140).astype(np.float16)
        s[:6] = 0, -0.0, np.inf, np.nan, 60000, -60000
    u = np.where(rng.random(s.size) < 0.5, 1.0, rng.uniform(0.5, 2, s.size)).astype(dtype)
    wide = s.astype(np.float64)
    with np.errstate(all="ignore"):
        silu = wide / (1 + np.exp(-wide))
        off = np.abs(silu) * (2.0 ** -17 if dtype == np.float16 else 2.0 ** -22) + LOST
    e = np.finfo(dtype)
    for act in (ops.ACT_SILU, ops.ACT_SWIGLU):
        pairs = np.stack([s, u], 1).reshape(-1)
        got = run(backend, s if act == ops.ACT_SILU else pairs, rows, 64, mx, act, dtype).astype(np.float64)
        with np.errstate(invalid="ignore"):
            want = silu if act == ops.ACT_SILU else silu * u.astype(np.float64)
            # the product's rounding in f32, and that to the result's type
            tol = (off if act == ops.ACT_SILU else off * np.abs(u.astype(np.float64)) + np.abs(want) * 2.0 ** -24)
            tol = tol + np.abs(want) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2
        finite = np.isfinite(want)
        np.testing.assert_array_equal(np.isnan(got), np.broadcast_to(np.isnan(want), got.shape))
        np.testing.assert_array_equal(got[:, np.isinf(want)], np.broadcast_to(want[np.isinf(want)], got[:, np.isinf(want)].shape))
        bad = ~(np.abs(got[:, finite] - want[finite]) <= tol[finite])
        assert not bad.any(), (int(bad.sum()), wide[finite][bad.any(0)][:5], got[:, finite][bad][:5], want[finite][bad.any(0)][:5])

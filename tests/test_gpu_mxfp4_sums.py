"""Products whose sums f32 holds exactly, whatever their order: any element of
K that a kernel drops, takes twice or takes from another row changes the result,
however long the sum is."""
import numpy as np
import pytest

import mxfp4_reference as ref
from dragonwing_edge_rs_amd import ops

pytestmark = pytest.mark.gpu

SIZES = [(1, 40, 33000), (1, 700, 8192), (2, 33, 16384), (3, 70, 16500), (4, 5200, 4100), (4, 16, 31),  # rows through LDS
         (5, 48, 33000), (16, 5130, 2100), (16, 260, 12288), (17, 40, 20000), (20, 300, 33000), (32, 5200, 900),
         (32, 17, 513),  # up to 32 rows
         (33, 128, 8192), (40, 130, 33000), (64, 8192, 2048), (70, 2050, 8200), (130, 1030, 14000), (129, 257, 999),
         (300, 260, 1056), (513, 384, 4100), (257, 130, 511),  # tiles, K shared
         (1900, 7300, 288), (4091, 8189, 136), (6500, 2050, 129), (2048, 4096, 1536)]  # large tiles


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sums_to_the_last_bit(backend, m, n, k, kind):
    be = backend
    a, q, s, _, _, want = ref.whole_product(np.random.default_rng(m + n + k), m, n, k, kind)
    c = be.from_numpy(np.full((m, n), np.nan, np.float32))
    mx = kind == "mxfp4"
    ops.gemm_mxfp4(be, ops.DTYPE_MXFP4 if mx else ops.DTYPE_F16, be.from_numpy(a[0] if mx else a),
                   be.from_numpy(a[1]) if mx else None, be.from_numpy(q), be.from_numpy(s), None, ops.DTYPE_F32, c, m, n, k)
    np.testing.assert_array_equal(be.to_numpy(c, np.float32, (m, n)), want)

"""Calls after one that the device had no memory for."""
import numpy as np
import pytest

from dragonwing_edge_rs_amd import HipError, ops

pytestmark = pytest.mark.gpu


def test_calls_after_a_refused_allocation(backend):
    # more than any device has: the runtime says so and allocates nothing
    be = backend
    ids = be.from_numpy(np.array([1, 0, 1, 2], np.int32))
    offsets, order = be.alloc(4 * 4), be.alloc(4 * 4)
    with pytest.raises(HipError):
        be.alloc(1 << 46)
    ops.order_experts(be, ids, offsets, order, 4, 3)
    np.testing.assert_array_equal(be.to_numpy(order, np.int32, (4,)), [1, 0, 2, 3])
    np.testing.assert_array_equal(be.to_numpy(offsets, np.int32, (4,)), [0, 1, 3, 4])

"""That exact sums notice a lost block of K, wherever it is, where a bound that
grows with K does not."""
import numpy as np
import pytest

import mxfp4_reference as ref


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(4, 40, 33000), (40, 16, 999), (1, 300, 129)])
def test_each_block_changes_the_product(m, n, k, kind):
    _, _, _, a, w, want = ref.whole_product(np.random.default_rng(k), m, n, k, kind)
    # exact: as in 64 bits, and with the terms in another order
    np.testing.assert_array_equal(want, a @ w.T)
    back = np.ascontiguousarray(a[:, ::-1], np.float32) @ np.ascontiguousarray(w[:, ::-1], np.float32).T
    np.testing.assert_array_equal(want, back)
    for at in range(0, k, 32):
        part = a[:, at:at + 32] @ w[:, at:at + 32].T  # what a kernel without this block leaves out
        assert (part != 0).mean() > 0.9


def test_a_block_that_the_bound_of_long_sums_lets_pass():
    # why the sums above are exact: for random elements the worst case of 33,000 roundings hides 32 elements
    rng = np.random.default_rng(40)
    q, s = ref.encode(rng.normal(0, 33000 ** -0.5, (16, 33000)))
    a, w = rng.normal(0, 1, (4, 33000)), ref.decode(q, s, 33000)
    want, off = ref.product(a, w)
    a[:, 512:544] = 0
    assert (np.abs(a @ w.T - want) <= off).all()

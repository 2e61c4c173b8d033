"""Routing by logits that are zeros of either sign: they are equal, and ties go
to the lowest index."""
import numpy as np
import pytest

from test_gpu_experts import check_route

pytestmark = pytest.mark.gpu


def zeros(rng, tokens, experts, top, dtype):
    """Rows of zeros, half of them negative, with some other numbers; and rows of two zeros of unlike signs, the last
    one to be chosen and the first that is not, or both chosen."""
    x = np.where(rng.random((tokens, experts)) < 0.5, -0.0, 0.0)
    x = np.where(rng.random((tokens, experts)) < 1.5 / experts, 1.0, x)
    x = np.where(rng.random((tokens, experts)) < 0.2, -1.0, x)
    x[0], x[1] = 0.0, -0.0
    x[0, 0], x[1, -1] = -0.0, 0.0
    tiny = np.finfo(dtype).smallest_subnormal
    x[2, ::3] = -tiny  # numbers beside them are no zeros
    x[3, ::3] = tiny
    for t in range(4, tokens // 2):
        x[t] = -1 - rng.permutation(experts) / 64
        above = max(0, top - 1 - t % 3)
        some = rng.permutation(experts)[:above + 2]
        x[t, some] = 1 + np.arange(len(some)) / 64
        x[t, np.sort(some[:2])] = (-0.0, 0.0) if t % 4 else (0.0, -0.0)
    return x.astype(dtype)


@pytest.mark.parametrize("experts,top", [(2, 1), (8, 2), (16, 16), (30, 5), (64, 8), (67, 9), (128, 8), (256, 8), (256, 20), (500, 3),
                                         (1024, 32)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_zeros_of_either_sign_tie(backend, experts, top, dtype):
    x = zeros(np.random.default_rng(experts + top), 40, experts, top, dtype)
    for sigmoid in (False, True):
        check_route(backend, x, top, sigmoid=sigmoid, renorm=not sigmoid)


@pytest.mark.parametrize("experts,groups,kept", [(8, 2, 1), (30, 3, 2), (64, 8, 3), (128, 8, 4), (256, 8, 4), (1024, 32, 5)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_zeros_of_either_sign_tie_within_groups(backend, experts, groups, kept, dtype):
    x = zeros(np.random.default_rng(experts + groups), 40, experts, 3, dtype)
    bias = np.where(np.arange(experts) % 2, 0.0, -0.0).astype(np.float32)
    for best in (1, 2):
        check_route(backend, x, 3, groups=groups, kept=kept, best=best)
        check_route(backend, x, 3, sigmoid=True, groups=groups, kept=kept, best=best, bias=bias)

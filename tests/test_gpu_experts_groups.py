"""Routing within groups whose experts lie in whole lanes (65 to 256 experts in
groups of one, two, four or eight lanes), and beside them in groups that do not."""
import numpy as np
import pytest

from test_gpu_experts import check_route

pytestmark = pytest.mark.gpu

# experts, groups, kept.  16 experts a lane: up to 128 have 8 lanes a token, up to 256 16.
SHAPES = [(128, 8, 4), (128, 8, 1), (128, 4, 2), (128, 2, 1), (80, 5, 2), (96, 6, 3), (96, 3, 2), (112, 7, 6), (128, 1, 1),
          (256, 16, 5), (256, 16, 15), (256, 8, 3), (256, 4, 2), (256, 4, 1), (256, 2, 1), (192, 3, 2), (192, 12, 7), (144, 9, 4),
          (240, 15, 2), (160, 5, 2), (224, 7, 4),
          (120, 5, 2), (126, 7, 3), (144, 3, 2), (250, 5, 3)]  # groups that share lanes or have three


@pytest.mark.parametrize("experts,groups,kept", SHAPES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_groups_of_whole_lanes(backend, experts, groups, kept, dtype):
    rng = np.random.default_rng(experts * 7 + groups + kept)
    x = rng.normal(0, 1.5, (37, experts)).astype(dtype)
    bias = rng.normal(0, 0.05, experts).astype(np.float32)
    for top in (1, 8, min(32, kept * (experts // groups))):
        for best in (1, 2):
            check_route(backend, x, top, groups=groups, kept=kept, best=best)
            check_route(backend, x, top, sigmoid=True, groups=groups, kept=kept, best=best, bias=bias, renorm=False, scale=2.5)
            check_route(backend, x, top, groups=groups, kept=kept, best=best, bias=bias)


def shaped(experts, groups, kept):
    return pytest.param(experts, groups, kept, id=f"{experts}-{groups}-{kept}")


SOME = [shaped(*s) for s in ((128, 8, 4), (128, 4, 2), (128, 2, 1), (80, 5, 2), (256, 16, 5), (256, 8, 3), (256, 4, 2), (256, 2, 1),
                             (192, 3, 2), (120, 5, 2))]


@pytest.mark.parametrize("experts,groups,kept", SOME)
def test_ties_of_groups_and_experts(backend, experts, groups, kept):
    rng = np.random.default_rng(experts + groups)
    x = rng.integers(-1, 2, (40, experts)).astype(np.float32)
    x[0] = 0
    size = experts // groups
    x[1:9] = np.tile(x[1:9, :size], groups)  # all groups alike
    x[9:20, size:] = x[9:20, :-size]  # and neighbours
    bias = rng.integers(-1, 2, experts).astype(np.float32) * 0.125
    for dtype in (np.float16, np.float32):
        for best in (1, 2):
            check_route(backend, x.astype(dtype), 8, groups=groups, kept=kept, best=best)
            check_route(backend, x.astype(dtype), 8, sigmoid=True, groups=groups, kept=kept, best=best, bias=bias)
            check_route(backend, x.astype(dtype), 8, groups=groups, kept=kept, best=best, bias=np.zeros_like(bias))


@pytest.mark.parametrize("experts,groups,kept", SOME)
def test_near_ties_of_groups(backend, experts, groups, kept):
    # sums that f32 rounds to one value, in an order of their own
    rng = np.random.default_rng(experts + groups)
    bias = rng.integers(0, 3, experts).astype(np.float32)
    for x in (20 + rng.integers(0, 40, (40, experts)) * 0.25, rng.normal(0, 1e-6, (40, experts))):
        x = x.astype(np.float32)
        for best in (1, 2):
            check_route(backend, x, 8, sigmoid=True, bias=bias, groups=groups, kept=kept, best=best)
            check_route(backend, x, 8, bias=bias, groups=groups, kept=kept, best=best)


@pytest.mark.parametrize("experts,groups,kept", SOME)
def test_masks_infinities_and_nan_in_groups(backend, experts, groups, kept):
    rng = np.random.default_rng(experts + groups)
    size = experts // groups
    x = rng.normal(0, 2, (40, experts)).astype(np.float32)
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4, experts - 1] = np.inf
    x[5, [3, experts // 2]] = np.inf
    x[6] = np.inf
    x[7] = np.finfo(np.float32).min
    x[8, :experts - size] = -np.inf  # the last group alone
    x[9, size:] = -np.inf  # the first
    for g in range(groups):  # one expert a group
        x[10, g * size:(g + 1) * size - 1] = -np.inf
    x[11:20][rng.random((9, experts)) < 0.97] = -np.inf
    x[20:30] = rng.normal(-150, 3, (10, experts))
    bias = rng.normal(0, 0.1, experts).astype(np.float32)
    off = bias.copy()
    off[[0, 7, size, experts - 1]] = -np.inf, np.nan, np.inf, -1e30
    for sigmoid in (False, True):
        for b in (None, bias, off):
            for best in (1, 2):
                check_route(backend, x, 6, sigmoid=sigmoid, renorm=sigmoid, bias=b, groups=groups, kept=kept, best=best)

"""Routing where the sums of two groups lie as far apart in f32 as their roundings
can bring equal ones: the groups that are kept are those of the sums in 64 bits."""
import numpy as np
import pytest

from test_gpu_experts import run_route

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -3  # of f32 numbers from 2^20 on
HIGH, LOW = 2.0 ** 20 + 64, 2.0 ** 20  # biases, so that the two experts of a group lie apart
# whole steps of each group's two scores, half a step below them: sums with the biases are an odd number of steps, so
# that one group's may round down three times and the other's up three times
PAIRS = [((5, 0), (3, 2)), ((3, 2), (5, 0)), ((5, 4), (7, 2)), ((7, 2), (5, 4)), ((4, 5), (2, 7)), ((2, 7), (4, 5)),
         ((4, 1), (2, 3)), ((3, 6), (5, 4))]


def rows():
    """Four logits a row, two of each group: every choice of the f32 numbers around those of which the sigmoids are half
    a step above the whole ones."""
    ulps = np.stack(np.meshgrid(*[np.arange(-4, 5, dtype=np.int32)] * 4, indexing="ij"), -1).reshape(-1, 4)
    parts = []
    for a, b in PAIRS:
        p = (np.array(a + b) + 0.5) * STEP
        parts.append((np.log(p / (1 - p)).astype(np.float32).view(np.int32) + ulps).view(np.float32))
    return np.concatenate(parts)


@pytest.mark.parametrize("experts", [4, 64, 128, 256, 512])
def test_groups_are_those_of_sums_in_64_bits(backend, experts):
    some = rows()
    x = np.full((len(some), experts), -np.inf, np.float32)
    bias = np.full(experts, LOW, np.float32)
    half = experts // 2
    at = [0, 1, half, half + 1]
    x[:, at] = some
    bias[[0, half]] = HIGH
    c = 1 / (1 + np.exp(-some.astype(np.float64))) + bias[at].astype(np.float64)
    want = np.where(c[:, 2] + c[:, 3] > c[:, 0] + c[:, 1], half, 0)
    ids, weights = run_route(backend, x, 1, bias=bias, sigmoid=True, groups=2, kept=1, best=2)
    wrong = np.flatnonzero(ids[:, 0] != want)
    assert not len(wrong), (len(wrong), len(some), some[wrong[:3]], ids[wrong[:3], 0])
    assert (weights == 1).all()

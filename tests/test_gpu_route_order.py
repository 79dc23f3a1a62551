"""The order of apus_hip_route_dev where fp32 scores of very different size meet: large
scores beside ordinary ones, biases that swamp the scores, groups whose second value is tiny.
The choice has to be that of the 64-bit values (tests/test_gpu_route.py says what is compared)."""
import numpy as np
import pytest

from test_gpu_route import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,k", [(64, 8), (256, 6), (320, 8), (64, 12)])
@pytest.mark.parametrize("large", [40.0, 2000.0, 1e4, 1e6])
@pytest.mark.parametrize("fine", [0.0, 2.0 ** -22, 2.0 ** -20])
def test_route_large_scores_beside_small_ones(hip, rng, E, k, large, fine):
    """three scores a few fp32 steps apart among ones near 1: sqrt-softplus has no upper end, so
    the largest scores have the largest errors. The bias is a step or so of the large ones."""
    s = 4000
    z = rng.standard_normal((s, E)) - 2.0
    near = large * (1 + rng.integers(0, 64, (s, 3)) * 2.0 ** -23)
    at = np.argsort(rng.random((s, E)), axis=1)[:, :3]
    np.put_along_axis(z, at, near, axis=1)
    bias = (fine * np.sqrt(large) * rng.standard_normal(E)).astype(np.float32) if fine else None
    check(hip, "softplus", z, bias, k, least=0.5)

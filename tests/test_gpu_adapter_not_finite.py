"""Rank sums of f16 adapters that are not finite beside such as f16 does not hold."""
import numpy as np
import pytest

import feed_forward_reference as ref
from feed_forward_reference import values
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["f32", "f16"])
@pytest.mark.parametrize("rank", [4, 16, 30, 64, 100])
@pytest.mark.parametrize("m,tile", [(5, (1, 16, 16)), (40, (1, 16, 16)), (40, (5, 7, 6))])
def test_an_infinite_sum_beside_a_large_one(gpu_lib, m, tile, rank, out):  # noqa: F811
    # The one rank's sum is infinite, another's -2^20 and more: with positive `up` every result is infinite, of the first one's sign.
    rng = np.random.default_rng(rank)
    n, k, count = 70 if tile[1] == 7 else 80, 72 if tile[2] == 6 else 80, 3
    x = np.abs(values(rng, m, k, "f16")) + 1
    x, down = ref.to_type(x.astype(np.float32), "f16").astype(np.float64), values(rng, count * rank, k, "f16").reshape(count, rank, k)
    up_ = ref.to_type((np.abs(values(rng, count * n, rank, "f16", 0.3)) + 0.25).astype(np.float32), "f16").astype(np.float64).reshape(count, n, rank)
    index = (np.arange(m) % count).astype(np.int32)
    down[:, 1] = -30000
    clean, _ = ref.run_adapters(gpu_lib, x, down, up_, index, None, tile, "f16", "f32")
    assert np.isfinite(clean).all() and (clean < -2.0 ** 17).all()
    down[1, rank - 1, 7] = np.inf
    got, _ = ref.run_adapters(gpu_lib, x, down, up_, index, None, tile, "f16", out)
    assert (got[index == 1] == np.inf).all()
    if out == "f32":
        np.testing.assert_array_equal(got[index != 1], clean[index != 1])

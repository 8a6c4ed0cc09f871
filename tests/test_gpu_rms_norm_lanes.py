"""The norm's row kernels with different numbers of lanes to a row, on the GPU: of 513 to 1024 columns a row has 64 lanes with two
pieces each among more than 512 rows, and 256 lanes with one otherwise. Its codes are the same."""
import numpy as np
import pytest

from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_rms_norm import inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("format", ["s8", "e4m3", "e2m1"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(600, 1000), (513, 544), (601, 1024)])
def test_a_row_does_not_depend_on_its_lanes(gpu_lib, rows, cols, type, format):  # noqa: F811
    x, r, w = inputs(np.random.default_rng(cols), rows, cols, type)
    out_cols = -(-cols // 32) * 32
    many = run(gpu_lib, x, r, w, type, format, out_cols)
    few = [run(gpu_lib, x[i:i + 300], r[i:i + 300], w, type, format, out_cols) for i in range(0, rows, 300)]
    for a, b in zip(many, zip(*few)):
        np.testing.assert_array_equal(a, np.concatenate(b))

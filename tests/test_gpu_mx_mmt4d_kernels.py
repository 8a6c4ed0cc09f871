"""Every kernel of the products of microscaled operands on the GPU, with one chunk of K and with many: exact sums (see
test_gpu_mx_mmt4d.py), from the kernel that is meant."""
import numpy as np
import pytest

from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_mmt4d import check_exact
from test_mx_mmt4d_choice_on_host import KERNELS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,kernel", KERNELS)
def test_exact_sums(gpu_lib, lhs, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    used = check_exact(gpu_lib, np.random.default_rng(rows + cols), rows, cols, k, (m0, n0, 128), lhs, out)
    assert used.decode() == "mx_mmt4d_" + kernel


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,kernel", [q for q in KERNELS if q[4] > 128 and q[2] * q[3] < 1 << 20])
def test_accumulate(gpu_lib, lhs, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    check_exact(gpu_lib, np.random.default_rng(rows + cols), rows, cols, k, (m0, n0, 128), lhs, out, accumulate=True)

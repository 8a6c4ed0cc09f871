"""Every kernel of the gated products and their gradients on the GPU against 64 bits (feed_forward_kernels.py)."""
import pytest

import test_gpu_gated_backward as backward
import test_gpu_gated_mmt4d as gated
from feed_forward_kernels import GATED, GATED_LINES, LHS_GRADS, WEIGHT_GRADS
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("kernel,m,n,k,tile", GATED)
def test_gated(gpu_lib, kernel, m, n, k, tile, type):  # noqa: F811
    mode, pre_type = ("store", type) if k < 100 else ("load", "f32")
    name = gated.check_case(gpu_lib, m, n, k, tile, type, "f32" if k < 100 else type, "silu", mode, pre_type)
    assert name.decode() == "gated_mmt4d_" + kernel


@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("kernel,m,n,k,tile", GATED_LINES)
def test_gated_of_whole_lines(gpu_lib, kernel, m, n, k, tile, type):  # noqa: F811
    name = gated.check_case(gpu_lib, m, n, k, tile, type, type, "gelu")
    assert name.decode() == "gated_mmt4d_" + kernel


@pytest.mark.parametrize("type,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("kernel,m,n,k,tile", LHS_GRADS)
def test_lhs_grad(gpu_lib, kernel, m, n, k, tile, type, out):  # noqa: F811
    backward.check_case(gpu_lib, m, n, k, tile, type, out, type, "silu", which="l")


@pytest.mark.parametrize("type,out,accumulate", [("bf16", "bf16", False), ("f16", "f32", True)])
@pytest.mark.parametrize("kernel,m,n,k,tile", WEIGHT_GRADS)
def test_weight_grads(gpu_lib, kernel, m, n, k, tile, type, out, accumulate):  # noqa: F811
    backward.check_case(gpu_lib, m, n, k, tile, type, out, type, "gelu", accumulate, which="gu")

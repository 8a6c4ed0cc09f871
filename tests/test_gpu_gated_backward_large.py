"""The backward pass of gated products where workspace, operands and gradients have more than 2^31 elements, and where strides are beyond
the fast kernels' 31 bits; the bounds are derived in feed_forward_reference.py."""
import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu
NAMES = ("lhs", "gate", "up", "gate_pre", "up_pre", "out_grad", "lhs_grad", "gate_grad", "up_grad")


def bits(x, t0, t1, type="bf16"):
    """[rows][cols] -> panels of tiles, a row each."""
    return torch.from_numpy(ref.raw(ref.tiled(x, t0, t1), type).view(np.int16).reshape(x.shape[0] // t0, -1)).cuda()


def call(lib, m, n, k, tile, held, stride={}, type="bf16"):
    p = abi.GatedMmt4dBackwardParams()
    ref.tiles_into(p, m, n, k, tile)
    m0, n0, _ = tile
    panel = {"lhs": m0 * k, "lhs_grad": m0 * k, "gate": n0 * k, "up": n0 * k, "gate_grad": n0 * k, "up_grad": n0 * k}
    for name in NAMES:
        setattr(p, name + "_buffer", held[name].data_ptr())
        setattr(p, name + "_stride0", stride.get(name, panel.get(name, m0 * n)))
    p.flags = ref.type_flag("GATED_MMT4D", type, type) | abi.GATED_MMT4D_SILU
    keep, size = ref.workspace(lib, "gated_mmt4d_backward", p)
    ref.call(lib, "gated_mmt4d_backward", p)
    assert bool((keep[size:] == 0xFF).all())
    return size


def problem(seed, m, n, k, type="bf16"):
    rng = np.random.default_rng(seed)
    return dict(x=values(rng, m, k, type), gate=values(rng, n, k, type, 0.2), up_=values(rng, n, k, type, 0.2),
                g=values(rng, m, n, type, 1.5), u=values(rng, m, n, type, 1.5), grad=values(rng, m, n, type))


def matrix_of(panels, t0, t1, type="bf16"):
    """Panels of tiles in device memory -> [rows][cols]"""
    x = panels.view(torch.float16 if type == "f16" else torch.bfloat16).float().cpu().numpy().astype(np.float64)
    return ref.untiled(x.reshape(x.shape[0], -1, t0, t1))


def all_zero(panels):
    return all(bool((panels[i:i + 1024] == 0).all()) for i in range(0, panels.shape[0], 1024))


# The gradient of out is zero but in the last 48 rows: those of lhs_grad are not zero, and the weights' gradients are sums over them.
@pytest.mark.parametrize("n,k", [(8192, 64), (64, 16384)])
@pytest.mark.parametrize("m0,type", [(1, "bf16"), (16, "bf16"), (16, "f16")])
def test_many_rows(gpu_lib, m0, type, n, k):  # noqa: F811
    m, last, tile = 139264, 48, (m0, 16, 16)
    assert m * max(2 * n, k) > 2 ** 31
    given = problem(n, last, n, k, type)
    held = {name: torch.full((m // m0, m0 * cols), 0x3F80, dtype=torch.int16, device="cuda")
            for name, cols in (("lhs", k), ("lhs_grad", k), ("gate_pre", n), ("up_pre", n), ("out_grad", n))}
    held["out_grad"].zero_()
    for name, of, t1 in (("lhs", "x", 16), ("gate_pre", "g", 16), ("up_pre", "u", 16), ("out_grad", "grad", 16)):
        held[name][-last // m0:] = bits(given[of], m0, t1, type)
    for name, of in (("gate", "gate"), ("up", "up_")):
        held[name], held[name + "_grad"] = bits(given[of], 16, 16, type), torch.full((n // 16, 16 * k), 0x3F80, dtype=torch.int16, device="cuda")
    assert call(gpu_lib, m, n, k, tile, held, type=type) >= 4 * m * n
    want, off = ref.backward(activation="silu", type=type, **given)
    assert all_zero(held["lhs_grad"][:-last // m0])
    check(matrix_of(held["lhs_grad"][-last // m0:], m0, 16, type), want[0], off[0], type)
    # (Rows of zeros add nothing, exactly.)
    check(matrix_of(held["gate_grad"], 16, 16, type), want[1], off[1], type)
    check(matrix_of(held["up_grad"], 16, 16, type), want[2], off[2], type)


# The gradient of out is zero but in the last 64 columns: only theirs of the weights' gradients are not zero.
@pytest.mark.parametrize("m", [24, 300])
def test_many_columns(gpu_lib, m):  # noqa: F811
    n, k, last, tile = 139264, 16384, 64, (1, 16, 16)
    given = problem(m, m, last, k)
    held = {name: torch.full((n // 16, 16 * k), 0x3F80, dtype=torch.int16, device="cuda") for name in ("gate", "up", "gate_grad", "up_grad")}
    for name, of in (("gate", "gate"), ("up", "up_")):
        held[name][-last // 16:] = bits(given[of], 16, 16)
    for name, of in (("gate_pre", "g"), ("up_pre", "u"), ("out_grad", "grad")):
        held[name] = torch.zeros((m, n), dtype=torch.int16, device="cuda")
        held[name][:, -last:] = bits(given[of], 1, 16)
    held["lhs"], held["lhs_grad"] = bits(given["x"], 1, 16), torch.full((m, k), 0x3F80, dtype=torch.int16, device="cuda")
    call(gpu_lib, m, n, k, tile, held)
    want, off = ref.backward(activation="silu", type="bf16", **given)
    for i, name in ((1, "gate_grad"), (2, "up_grad")):
        assert all_zero(held[name][:-last // 16])
        check(matrix_of(held[name][-last // 16:], 16, 16), want[i], off[i], "bf16")
    check(matrix_of(held["lhs_grad"], 1, 16), want[0], off[0], "bf16")


# Panels of one matrix 4 GiB and more from first to last, each of a GiB or a 64 MiB's distance: not the fast kernels'.
@pytest.mark.parametrize("name,apart", [("lhs", 1 << 25), ("gate", 1 << 29), ("up", 1 << 29), ("lhs_grad", 1 << 25), ("gate_grad", 1 << 29), ("gate_pre", 1 << 25),
                                        ("out_grad", 1 << 25)])
def test_panels_far_apart(gpu_lib, name, apart):  # noqa: F811
    m, n, k, tile = 70, 96, 128, (1, 16, 16)
    given = problem(7, m, n, k)
    sides = {"lhs": ("x", 1), "gate": ("gate", 16), "up": ("up_", 16), "gate_pre": ("g", 1), "up_pre": ("u", 1), "out_grad": ("grad", 1)}
    held = {of: bits(given[of_given], t0, 16) for of, (of_given, t0) in sides.items()}
    for of in ("lhs", "gate", "up"):
        held[of + "_grad"] = torch.zeros_like(held[of])
    panels, width = held[name].shape
    whole = torch.full(((panels - 1) * apart + width,), 0x7FFF, dtype=torch.int16, device="cuda")  # (NaN between)
    far = whole.as_strided((panels, width), (apart, 1))
    far.copy_(held[name])
    held[name] = far
    call(gpu_lib, m, n, k, tile, held, {name: apart})
    want, off = ref.backward(activation="silu", type="bf16", **given)
    for i, of in enumerate(("lhs", "gate", "up")):
        check(matrix_of(held[of + "_grad"].contiguous(), 1 if of == "lhs" else 16, 16), want[i], off[i], "bf16")
    for i in range(panels - 1):
        between = whole[i * apart + width:(i + 1) * apart]
        assert bool((between[:4096] == 0x7FFF).all()) and bool((between[-4096:] == 0x7FFF).all())

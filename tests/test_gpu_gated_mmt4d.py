"""Gated products on the GPU against 64 bits; the bounds are derived in feed_forward_reference.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, up, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(seed, m, n, k, tile, type):
    """Padded to whole tiles with zeros, but for the values that fill them."""
    rng = np.random.default_rng(seed)
    rows, cols, depth = up(m, tile[0]), up(n, tile[1]), up(k, tile[2])
    scale = 1.5 / np.sqrt(max(1, depth))
    return rng, values(rng, rows, depth, type), values(rng, cols, depth, type, scale), values(rng, cols, depth, type, scale)


def check_case(lib, m, n, k, tile, type, out, activation, mode="none", pre_type="f32", layout={}, host=False):
    rng, x, gate, up_ = inputs(m + n + k, m, n, k, tile, type)
    pre = tuple(values(rng, x.shape[0], gate.shape[0], pre_type) for _ in range(2)) if "load" in mode else None
    got, kernel = ref.run_gated(lib, x, gate, up_, activation, tile, type, out, pre, mode, pre_type, layout, host)
    want, off = ref.gated(x, gate, up_, activation, pre)
    check(got[0], want[0], off[0], out)
    for i in (1, 2):
        if "store" in mode:
            check(got[i], want[i], off[i], pre_type)
        elif "load" in mode:
            np.testing.assert_array_equal(got[i], pre[i - 1])
    return kernel


# From one token to a small prompt, odd sizes, tiles that the fast kernels take and tiles that only the general one does.
PROBLEMS = [
    (1, 16, 16, (1, 16, 16)), (1, 100, 300, (1, 16, 16)), (1, 1000, 4096, (1, 16, 16)), (2, 512, 1024, (1, 16, 16)),
    (3, 200, 640, (1, 1, 8)), (5, 77, 1000, (1, 16, 16)), (8, 300, 2048, (8, 16, 16)), (16, 1040, 3000, (16, 16, 16)),
    (16, 64, 14336, (1, 16, 16)), (17, 333, 257, (1, 16, 16)), (31, 96, 96, (1, 1, 32)), (33, 500, 640, (16, 16, 16)),
    (64, 640, 1152, (1, 16, 16)), (65, 129, 2000, (1, 16, 32)), (100, 1000, 384, (4, 8, 16)), (128, 128, 512, (16, 16, 16)),
    (130, 700, 1000, (1, 16, 16)), (200, 264, 4096, (1, 1, 64)), (257, 513, 896, (1, 16, 8)), (300, 300, 130, (16, 16, 16)),
    (512, 1000, 640, (16, 16, 16)), (777, 1040, 544, (1, 16, 32)), (40, 50, 70, (5, 7, 6)), (9, 30, 500, (3, 5, 16)),
    (20, 20, 1030, (2, 4, 24)), (70, 90, 24, (1, 16, 8)), (300, 200, 8, (1, 16, 8)), (1, 31, 7, (1, 1, 1)), (40, 48, 100, (1, 16, 4)),
    (90, 257, 2056, (1, 1, 2056)), (33, 100, 1000, (1, 4, 16)),
]


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
def test_products(gpu_lib, m, n, k, tile, type, out):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, type, type if out == "same" else out, "silu")


@pytest.mark.parametrize("mode,pre_type", [("load", "f32"), ("load", "same"), ("store", "same"), ("store", "f32"), ("load_store", "f32"),
                                           ("load_store", "same")])
@pytest.mark.parametrize("type,activation", [("bf16", "gelu"), ("f16", "sigmoid")])
@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (2, 7, 9, 11, 16, 18, 20, 22, 30)])
def test_products_with_terms_before_the_activation(gpu_lib, m, n, k, tile, type, activation, mode, pre_type):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, type, type, activation, mode, type if pre_type == "same" else pre_type)


def test_a_bias_for_every_row(gpu_lib):  # noqa: F811
    # Terms whose panels coincide (a stride of zero): one row of them, for tiles one row tall.
    rng, x, gate, up_ = inputs(5, 70, 96, 200, (1, 16, 8), "bf16")
    bias = [values(rng, 1, 96, "f32") for _ in range(2)]
    held = {"lhs": ref.matrix(x, 1, 8, "bf16"), "gate": ref.matrix(gate, 16, 8, "bf16"), "up": ref.matrix(up_, 16, 8, "bf16"),
            "gate_pre": ref.matrix(bias[0], 1, 16, "f32"), "up_pre": ref.matrix(bias[1], 1, 16, "f32"),
            "out": ref.empty(70, 96, 1, "f32")}
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, 70, 96, 200, (1, 16, 8))
    for name, b in held.items():
        b.into(p, name)
    p.gate_pre_stride0 = p.up_pre_stride0 = 0
    p.flags = abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_PRE_LOAD | abi.GATED_MMT4D_PRE_F32
    ref.call(gpu_lib, "gated_mmt4d", p)
    want, off = ref.gated(x, gate, up_, "silu", [np.repeat(b, 70, 0) for b in bias])
    check(ref.fetched(held["out"], 1, 16), want[0], off[0], "f32")


@pytest.mark.parametrize("gap,offset", [(8, 8), (16, 24), (3, 5), (8, 1)])
@pytest.mark.parametrize("m,n,k,tile", [(1, 100, 300, (1, 16, 16)), (40, 100, 384, (1, 16, 16)), (48, 80, 384, (16, 16, 16)),
                                        (300, 200, 512, (1, 1, 32)), (200, 300, 264, (4, 4, 8))])
def test_strides_and_offsets(gpu_lib, m, n, k, tile, gap, offset):  # noqa: F811
    layout = {name: dict(gap=gap + 8 * i, offset=offset + 8 * i) for i, name in enumerate(("lhs", "gate", "up", "gate_pre", "up_pre", "out"))}
    check_case(gpu_lib, m, n, k, tile, "bf16", "bf16", "silu", "load_store", "f32", layout)


@pytest.mark.parametrize("mode", ["none", "load_store"])
def test_host_operands(gpu_lib, mode):  # noqa: F811
    layout = {name: dict(gap=2, offset=3) for name in ("lhs", "gate", "up", "gate_pre", "up_pre", "out")}
    check_case(gpu_lib, 20, 48, 256, (4, 16, 16), "f16", "f32", "gelu", mode, "f16", layout, host=True)


@pytest.mark.parametrize("mode", ["none", "load"])
def test_no_depth(gpu_lib, mode):  # noqa: F811
    check_case(gpu_lib, 5, 32, 0, (1, 16, 16), "bf16", "f32", "sigmoid", mode)


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_activations_over_their_range(gpu_lib, m, activation):  # noqa: F811
    # Products with one term: g runs from far below to far above what the exponential takes, u is one.
    cols = 512
    at = np.concatenate([np.linspace(-30, 30, cols // 2), np.geomspace(1e-30, 1e30, cols // 4), -np.geomspace(1e-30, 1e30, cols // 4)])
    gate = np.zeros((cols, 32))
    up_ = np.zeros((cols, 32))
    gate[:, 0], up_[:, 0] = ref.to_type(at, "bf16"), 1
    x = np.zeros((m, 32))
    x[:, 0] = 1
    got, _ = ref.run_gated(gpu_lib, x, gate, up_, activation, (1, 16, 16), "bf16", "f32")
    value, _, _ = ref.act(gate[:, 0], activation)
    check(got[0], np.repeat(value[None], m, 0), np.repeat(ref.act_off(gate[:, 0], 0, activation)[None], m, 0), "f32")


@pytest.mark.parametrize("m", [1, 20, 300])
def test_values_that_are_not_finite_stay_in_their_row_and_column(gpu_lib, m):  # noqa: F811
    rng, x, gate, up_ = inputs(7, m, 96, 272, (1, 16, 16), "bf16")
    clean, _ = ref.run_gated(gpu_lib, x, gate, up_, "silu", (1, 16, 16), "bf16", "f32")
    x[m // 2, 270] = np.nan
    gate[40, 3], up_[41, 5] = np.nan, np.inf
    got, _ = ref.run_gated(gpu_lib, x, gate, up_, "silu", (1, 16, 16), "bf16", "f32")
    rows, cols = np.arange(m) != m // 2, ~np.isin(np.arange(96), (40, 41))
    assert np.isnan(got[0][m // 2]).all() and np.isnan(got[0][:, 40]).all()
    assert not np.isfinite(got[0][:, 41][x[:, 5] != 0]).any()
    np.testing.assert_array_equal(got[0][rows][:, cols], clean[0][rows][:, cols])


def test_panels_that_coincide(gpu_lib):  # noqa: F811
    rng, x, gate, up_ = inputs(1, 1, 64, 512, (1, 16, 16), "f16")
    held = {"lhs": ref.matrix(x, 1, 16, "f16"), "gate": ref.matrix(gate, 16, 16, "f16"), "up": ref.matrix(up_, 16, 16, "f16"),
            "out": ref.empty(70, 64, 1, "f32")}
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, 70, 64, 512, (1, 16, 16))
    for name, b in held.items():
        b.into(p, name)
    p.lhs_stride0 = 0
    p.flags = abi.GATED_MMT4D_TYPE_F16F16F32 | abi.GATED_MMT4D_SILU
    ref.call(gpu_lib, "gated_mmt4d", p)
    want, off = ref.gated(np.repeat(x, 70, 0), gate, up_, "silu")
    check(ref.fetched(held["out"], 1, 16), want[0], off[0], "f32")


def test_gate_and_up_may_be_one_matrix(gpu_lib):  # noqa: F811
    rng, x, gate, _ = inputs(2, 40, 64, 512, (1, 16, 16), "bf16")
    held = {"lhs": ref.matrix(x, 1, 16, "bf16"), "gate": ref.matrix(gate, 16, 16, "bf16"), "out": ref.empty(40, 64, 1, "bf16")}
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, 40, 64, 512, (1, 16, 16))
    for name, b in held.items():
        b.into(p, name)
    held["gate"].into(p, "up")
    p.flags = abi.GATED_MMT4D_TYPE_BF16BF16BF16 | abi.GATED_MMT4D_SIGMOID
    ref.call(gpu_lib, "gated_mmt4d", p)
    want, off = ref.gated(x, gate, gate, "sigmoid")
    check(ref.fetched(held["out"], 1, 16), want[0], off[0], "bf16")


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (50, 1024, 4096), (512, 1024, 2048)])
def test_the_same_call_gives_the_same_bits(gpu_lib, m, n, k):  # noqa: F811
    rng, x, gate, up_ = inputs(7, m, n, k, (1, 16, 16), "bf16")
    first, _ = ref.run_gated(gpu_lib, x, gate, up_, "silu", (1, 16, 16), "bf16", "f32")
    for _ in range(3):
        np.testing.assert_array_equal(ref.run_gated(gpu_lib, x, gate, up_, "silu", (1, 16, 16), "bf16", "f32")[0][0], first[0])


@pytest.mark.parametrize("m0,m", [(1, 1), (1, 40), (1, 300), (16, 304)])
def test_weights_beyond_32_bits(gpu_lib, m, m0):  # noqa: F811
    # 4.5 GiB of each of the weights, zeros but for the last 48 columns: there is one depth for all of them.
    cols, k = 73728, 32768
    rng, x, gate, up_ = inputs(m, m, 48, k, (m0, 16, 16), "bf16")
    weights = [torch.zeros(cols * k, dtype=torch.int16, device="cuda") for _ in range(2)]
    for w, v in zip(weights, (gate, up_)):
        w[-48 * k:] = torch.from_numpy(ref.raw(ref.tiled(v, 16, 16), "bf16").view(np.int16).reshape(-1)).cuda()
    lhs = ref.matrix(x, m0, 16, "bf16")
    out = torch.full((m // m0, cols // 16, m0, 16), 7.0, device="cuda")
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, m, cols, k, (m0, 16, 16))
    lhs.into(p, "lhs")
    p.gate_buffer, p.up_buffer, p.out_buffer = weights[0].data_ptr(), weights[1].data_ptr(), out.data_ptr()
    p.gate_stride0 = p.up_stride0 = 16 * k
    p.out_stride0 = cols * m0
    p.flags = abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_SILU
    ref.call(gpu_lib, "gated_mmt4d", p)
    assert bool((out[:, :-3] == 0).all())
    want, off = ref.gated(x, gate, up_, "silu")
    check(ref.untiled(out[:, -3:].contiguous().cpu().numpy()), want[0], off[0], "f32")


@pytest.mark.parametrize("m0", [1, 16])
def test_a_result_beyond_32_bits(gpu_lib, m0):  # noqa: F811
    # 4.5 GiB of bf16, of a lhs that is zero but for its last 48 rows.
    rows, cols, k = 73728, 32768, 32
    rng, x, gate, up_ = inputs(m0, 48, cols, k, (m0, 16, 16), "bf16")
    lhs = torch.zeros(rows * k, dtype=torch.int16, device="cuda")
    lhs[-48 * k:] = torch.from_numpy(ref.raw(ref.tiled(x, m0, 16), "bf16").view(np.int16).reshape(-1)).cuda()
    held = {"gate": ref.matrix(gate, 16, 16, "bf16"), "up": ref.matrix(up_, 16, 16, "bf16")}
    out = torch.full((rows // m0, cols // 16, m0, 16), 7, dtype=torch.bfloat16, device="cuda")
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, rows, cols, k, (m0, 16, 16))
    for name, b in held.items():
        b.into(p, name)
    p.lhs_buffer, p.lhs_stride0, p.out_buffer, p.out_stride0 = lhs.data_ptr(), k * m0, out.data_ptr(), cols * m0
    p.flags = abi.GATED_MMT4D_TYPE_BF16BF16BF16 | abi.GATED_MMT4D_SILU
    ref.call(gpu_lib, "gated_mmt4d", p)
    for first in range(0, rows - 48, 8192):
        assert bool((out[first // m0:min(first + 8192, rows - 48) // m0] == 0).all())
    want, off = ref.gated(x, gate, up_, "silu")
    check(ref.untiled(out[-48 // m0:].float().cpu().numpy()), want[0], off[0], "bf16")


def test_in_another_stream_and_replayed(gpu_lib):  # noqa: F811
    rng, x, gate, up_ = inputs(3, 40, 256, 512, (1, 16, 16), "bf16")
    held = {"lhs": ref.matrix(x, 1, 16, "bf16"), "gate": ref.matrix(gate, 16, 16, "bf16"), "up": ref.matrix(up_, 16, 16, "bf16"),
            "out": ref.empty(40, 256, 1, "f32")}
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, 40, 256, 512, (1, 16, 16))
    for name, b in held.items():
        b.into(p, name)
    p.flags = abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_SILU
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.stream(stream):
            gpu_lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            gpu_lib.iree_uk_mi355x_gated_mmt4d_p(C.byref(p))
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                gpu_lib.iree_uk_mi355x_gated_mmt4d_p(C.byref(p))
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)
    want, off = ref.gated(x, gate, up_, "silu")
    for _ in range(3):
        inner = held["out"].device[:40 * 256 * 4].view(torch.float32)
        inner.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(ref.fetched(held["out"], 1, 16), want[0], off[0], "f32")

"""The backward pass of gated products on the GPU against 64 bits; the bounds are derived in feed_forward_reference.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, up, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(seed, m, n, k, tile, type, out, pre_type):
    rng = np.random.default_rng(seed)
    rows, cols, depth = up(m, tile[0]), up(n, tile[1]), up(k, tile[2])
    scale = 1.5 / np.sqrt(max(1, depth))
    return dict(x=values(rng, rows, depth, type), gate=values(rng, cols, depth, type, scale),
                up_=values(rng, cols, depth, type, scale), g=values(rng, rows, cols, pre_type, 1.5),
                u=values(rng, rows, cols, pre_type, 1.5), grad=values(rng, rows, cols, out)), rng


def check_case(lib, m, n, k, tile, type, out, pre_type, activation, accumulate=False, which="lgu", layout={}, host=False):
    given, rng = inputs(m + n + k, m, n, k, tile, type, out, pre_type)
    shape = given["gate"].shape
    old = [values(rng, *shape, out, 3.0) for _ in range(2)] if accumulate else None
    got, kernel = ref.run_backward(lib, activation=activation, tile=tile, type=type, out=out, pre_type=pre_type, accumulate=old,
                                   which=which, layout=layout, host=host, **given)
    want, off = ref.backward(activation=activation, type=type, **given)
    for i, name in enumerate("lgu"):
        if name not in which:
            assert got[i] is None
        elif accumulate and i:
            total = want[i] + old[i - 1]
            check(got[i], total, off[i] + ref.U * np.abs(total), out)
        else:
            check(got[i], want[i], off[i], out)
    return kernel


PROBLEMS = [
    (1, 16, 16, (1, 16, 16)), (1, 300, 200, (1, 16, 16)), (3, 100, 77, (1, 16, 16)), (16, 256, 128, (16, 16, 16)),
    (33, 200, 120, (1, 1, 8)), (64, 640, 512, (1, 16, 16)), (100, 333, 257, (4, 8, 16)), (130, 1000, 500, (1, 16, 16)),
    (257, 300, 400, (1, 16, 8)), (300, 130, 1000, (16, 16, 16)), (777, 264, 328, (1, 16, 32)), (512, 512, 512, (16, 16, 16)),
    (40, 50, 70, (5, 7, 6)), (20, 20, 30, (2, 4, 24)), (9, 17, 31, (1, 1, 1)), (520, 96, 64, (1, 16, 16)), (50, 90, 100, (1, 16, 4)),
    (31, 1030, 40, (1, 1, 40)), (1000, 40, 24, (8, 8, 8)),
]


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
def test_gradients(gpu_lib, m, n, k, tile, type, out):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, type, type if out == "same" else out, type, "silu")


@pytest.mark.parametrize("type,activation,pre_type,accumulate", [("bf16", "gelu", "f32", False), ("f16", "sigmoid", "f32", True),
                                                                 ("bf16", "silu", "bf16", True), ("f16", "gelu", "f16", True)])
@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (1, 4, 7, 9, 11, 12, 16)])
def test_activations_types_and_accumulation(gpu_lib, m, n, k, tile, type, activation, pre_type, accumulate, out):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, type, type if out == "same" else out, pre_type, activation, accumulate)


# Few rows and a long K of lhs_grad (the gate's and up's rows): it is split, and its parts added.
SPLIT = [(1, 2080, 64, (1, 16, 16)), (17, 1200, 264, (1, 16, 8)), (40, 4096, 128, (1, 1, 8)), (64, 3001, 200, (16, 16, 16)),
         (100, 2048, 512, (4, 8, 8)), (130, 5000, 72, (1, 32, 24))]


@pytest.mark.parametrize("type,out,accumulate", [("bf16", "bf16", False), ("f16", "f32", True)])
@pytest.mark.parametrize("m,n,k,tile", SPLIT)
def test_split_sums(gpu_lib, m, n, k, tile, type, out, accumulate):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, type, out, type, "silu", accumulate, which="l" if n == 4096 else "lgu")


@pytest.mark.parametrize("which", ["l", "g", "u", "gu", "lu"])
@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (7, 9, 12)])
def test_some_of_the_gradients(gpu_lib, m, n, k, tile, which):  # noqa: F811
    check_case(gpu_lib, m, n, k, tile, "bf16", "bf16", "bf16", "silu", which=which)


NAMES = ("lhs", "gate", "up", "gate_pre", "up_pre", "out_grad", "lhs_grad", "gate_grad", "up_grad")


@pytest.mark.parametrize("gap,offset", [(8, 8), (16, 24), (3, 5)])
@pytest.mark.parametrize("m,n,k,tile", [(40, 100, 384, (1, 16, 16)), (48, 80, 384, (16, 16, 16)), (300, 200, 512, (1, 1, 32)),
                                        (200, 300, 264, (4, 4, 8))])
def test_strides_and_offsets(gpu_lib, m, n, k, tile, gap, offset):  # noqa: F811
    layout = {name: dict(gap=gap + 8 * i, offset=offset + 8 * i) for i, name in enumerate(NAMES)}
    check_case(gpu_lib, m, n, k, tile, "bf16", "bf16", "f32", "silu", layout=layout)


def test_host_operands(gpu_lib):  # noqa: F811
    layout = {name: dict(gap=2, offset=3) for name in NAMES}
    check_case(gpu_lib, 20, 48, 96, (4, 16, 16), "f16", "f32", "f16", "gelu", accumulate=True, layout=layout, host=True)


@pytest.mark.parametrize("m,n", [(0, 32), (8, 0)])
def test_sums_over_nothing_are_zero(gpu_lib, m, n):  # noqa: F811
    given, _ = inputs(1, m, n, 48, (1, 16, 16), "bf16", "f32", "bf16")
    got, _ = ref.run_backward(gpu_lib, activation="silu", tile=(1, 16, 16), type="bf16", out="f32", pre_type="bf16", **given)
    for x in got:
        assert (x == 0).all()


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
def test_slopes_over_their_range(gpu_lib, activation):  # noqa: F811
    # One weight of each matrix is one: lhs_grad is the sum of dg and du, gate_grad and up_grad are them.
    at = ref.to_type(np.concatenate([np.linspace(-30, 30, 384), np.geomspace(1e-30, 1e30, 64), -np.geomspace(1e-30, 1e30, 64)]), "f32")
    n = len(at)
    x = np.zeros((1, 16))
    x[0, 0] = 1
    given = dict(x=x, gate=np.zeros((n, 16)), up_=np.zeros((n, 16)), g=at[None].astype(np.float64), u=np.ones((1, n)), grad=np.ones((1, n)))
    got, _ = ref.run_backward(gpu_lib, activation=activation, tile=(1, 16, 16), type="bf16", out="f32", pre_type="f32", **given)
    with np.errstate(over="ignore", invalid="ignore"):
        want, off = ref.backward(activation=activation, type="bf16", **given)
        # (From 1e15 on the derivative's own terms are beyond what f64 holds of zero times them; the limits are 0 and 1.)
        value, slope, _ = ref.act(np.clip(given["g"], -1e4, 1e4), activation)
    large = np.abs(at) > 1e4
    want[1][large, 0] = slope[0, large]
    off[1][large, 0] = 2.0 ** -8
    check(got[1], want[1], off[1], "f32")
    check(got[2], want[2], off[2], "f32")


def test_against_differences(gpu_lib):  # noqa: F811
    # The formulas themselves: central differences of the loss sum(out * grad) in 64 bits.
    rng = np.random.default_rng(4)
    m, n, k = 6, 16, 16
    for activation in ("silu", "gelu", "sigmoid"):
        x, gate, up_ = (values(rng, r, k, "bf16", 0.4) for r in (m, n, n))
        grad = values(rng, m, n, "f32")
        g, u = x @ gate.T, x @ up_.T
        want, _ = ref.backward(x, gate, up_, g, u, grad, activation, "bf16")

        def loss():
            return (ref.act(x @ gate.T, activation)[0] * (x @ up_.T) * grad).sum()

        for of, gradient in ((x, want[0]), (gate, want[1]), (up_, want[2])):
            for _ in range(10):
                i = tuple(rng.integers(0, s) for s in of.shape)
                kept, step = of[i], 1e-5
                of[i] = kept + step
                above = loss()
                of[i] = kept - step
                below = loss()
                of[i] = kept
                assert abs((above - below) / (2 * step) - gradient[i]) < 1e-7
        got, _ = ref.run_backward(gpu_lib, x, gate, up_, ref.to_type(g, "f32").astype(np.float64), ref.to_type(u, "f32").astype(np.float64),
                                  grad, activation, (1, 16, 16), "bf16", "f32", "f32")
        want, off = ref.backward(x, gate, up_, ref.to_type(g, "f32").astype(np.float64), ref.to_type(u, "f32").astype(np.float64), grad,
                                 activation, "bf16")
        for i in range(3):
            check(got[i], want[i], off[i], "f32")


def test_values_that_are_not_finite_stay_in_their_row_and_column(gpu_lib):  # noqa: F811
    given, _ = inputs(9, 70, 96, 80, (1, 16, 16), "bf16", "f32", "bf16")
    run = dict(activation="silu", tile=(1, 16, 16), type="bf16", out="f32", pre_type="bf16")
    clean, _ = ref.run_backward(gpu_lib, **run, **given)
    given["grad"][20, 30] = np.nan
    got, _ = ref.run_backward(gpu_lib, **run, **given)
    rows, cols = np.arange(70) != 20, np.arange(96) != 30
    assert np.isnan(got[0][20]).all() and np.isnan(got[1][30]).all() and np.isnan(got[2][30]).all()
    np.testing.assert_array_equal(got[0][rows], clean[0][rows])
    np.testing.assert_array_equal(got[1][cols], clean[1][cols])
    np.testing.assert_array_equal(got[2][cols], clean[2][cols])


@pytest.mark.parametrize("m,n,k", [(40, 640, 512), (700, 520, 328)])
def test_the_same_call_gives_the_same_bits(gpu_lib, m, n, k):  # noqa: F811
    given, _ = inputs(3, m, n, k, (1, 16, 16), "bf16", "f32", "bf16")
    run = dict(activation="silu", tile=(1, 16, 16), type="bf16", out="f32", pre_type="bf16", **given)
    first, _ = ref.run_backward(gpu_lib, **run)
    for _ in range(3):
        for a, b in zip(ref.run_backward(gpu_lib, **run)[0], first):
            np.testing.assert_array_equal(a, b)


def test_in_another_stream_and_replayed(gpu_lib):  # noqa: F811
    # Forward and backward captured together, with the eager calls between the replays using another workspace.
    rng = np.random.default_rng(8)
    m, n, k, tile = 70, 208, 160, (1, 16, 16)
    x, gate, up_ = values(rng, m, k, "bf16"), values(rng, n, k, "bf16", 0.1), values(rng, n, k, "bf16", 0.1)
    grad = values(rng, m, n, "f32")
    held = {"lhs": ref.matrix(x, 1, 16, "bf16"), "gate": ref.matrix(gate, 16, 16, "bf16"), "up": ref.matrix(up_, 16, 16, "bf16"),
            "out_grad": ref.matrix(grad, 1, 16, "f32"), "gate_pre": ref.empty(m, n, 1, "f32"), "up_pre": ref.empty(m, n, 1, "f32"),
            "out": ref.empty(m, n, 1, "f32"), "lhs_grad": ref.empty(m, k, 1, "f32"), "gate_grad": ref.empty(n, k, 16, "f32"),
            "up_grad": ref.empty(n, k, 16, "f32")}
    f, b = abi.GatedMmt4dParams(), abi.GatedMmt4dBackwardParams()
    for p in (f, b):
        ref.tiles_into(p, m, n, k, tile)
        p.flags = abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_GELU | abi.GATED_MMT4D_PRE_F32
        for name, buffer in held.items():
            if hasattr(p, name + "_buffer"):
                buffer.into(p, name)
    f.flags |= abi.GATED_MMT4D_PRE_STORE
    keep, _ = ref.workspace(gpu_lib, "gated_mmt4d_backward", b)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def step():
        gpu_lib.iree_uk_mi355x_gated_mmt4d_p(C.byref(f))
        gpu_lib.iree_uk_mi355x_gated_mmt4d_backward_p(C.byref(b))

    try:
        with torch.cuda.stream(stream):
            gpu_lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            step()
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                step()
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)
    results = ("lhs_grad", "gate_grad", "up_grad")
    eager = [ref.fetched(held[r], 1 if r == "lhs_grad" else 16, 16) for r in results]
    (_, g, u), (_, g_off, u_off) = ref.gated(x, gate, up_, "gelu")
    want, off = ref.backward(x, gate, up_, g, u, grad, "gelu", "bf16", g_off, u_off)
    for i in range(3):
        check(eager[i], want[i], off[i], "f32")
    for _ in range(3):
        for name in results + ("out", "gate_pre", "up_pre"):
            inner = held[name].device[:-64].view(torch.float32)
            inner.fill_(5.0)
        keep.fill_(0xFF)
        ref.run_backward(gpu_lib, x, gate, up_, ref.to_type(g, "f32"), ref.to_type(u, "f32"), grad, "gelu", tile, "bf16", "f32", "f32")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for r, e in zip(results, eager):
            np.testing.assert_array_equal(ref.fetched(held[r], 1 if r == "lhs_grad" else 16, 16), e)

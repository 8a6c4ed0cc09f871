"""Gradients of f16 products far outside f16's range, on the GPU against 64 bits. Bounds as in feed_forward_reference.py, but that the
gradients of g and u are rounded to f16 after a power of two has brought the call's largest to between 2^14 and 2^15: half a step of
f16's subnormals, 2^-25, is 2^-39 of the largest then at most."""
import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_gated_backward import inputs

pytestmark = pytest.mark.gpu


def check_case(lib, monkeypatch, given, tile, out, pre_type, activation="silu", old=None):
    value, slope, _ = ref.act(given["g"], activation)
    largest = max(np.abs(given["grad"] * given["u"] * slope).max(), np.abs(given["grad"] * value).max())
    monkeypatch.setitem(ref.TINY, "f16", max(2.0 ** -39 * largest, 2.0 ** -149))
    want, off = ref.backward(activation=activation, type="f16", **given)
    if out == "f16":
        monkeypatch.setitem(ref.TINY, "f16", 2.0 ** -25)  # (the results' own rounding)
    got, _ = ref.run_backward(lib, activation=activation, tile=tile, type="f16", out=out, pre_type=pre_type, accumulate=old, **given)
    for i in range(3):
        total = want[i] if old is None or i == 0 else want[i] + old[i - 1]
        check(got[i], total, off[i] + (0 if old is None else ref.U * np.abs(total)), out)


# Both products in one launch, one after the other, lhs_grad's sums in parts; eight columns at a time in front of them or one; one thread
# for each result in front and behind.
PROBLEMS = [
    (64, 640, 512, (1, 16, 16)), (100, 333, 257, (1, 1, 8)), (777, 264, 328, (16, 16, 16)), (130, 5000, 72, (1, 32, 24)),
    (300, 2000, 1000, (1, 16, 16)), (1, 2080, 64, (1, 16, 16)), (40, 50, 70, (5, 7, 6)), (9, 17, 31, (1, 1, 1)), (1, 1, 1, (1, 1, 1)),
]


@pytest.mark.parametrize("power", [17, -24, 90, -80])
@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
def test_large_and_small_gradients(gpu_lib, monkeypatch, m, n, k, tile, power):  # noqa: F811
    given, _ = inputs(m + n + k, m, n, k, tile, "f16", "f32", "f32")
    given["grad"] = given["grad"] * 2.0 ** power
    check_case(gpu_lib, monkeypatch, given, tile, "f32", "f32")


@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (0, 2, 3, 6)])
def test_added_to_what_is_there(gpu_lib, monkeypatch, m, n, k, tile):  # noqa: F811
    given, rng = inputs(m + n + k, m, n, k, tile, "f16", "f32", "f16")
    given["grad"] = given["grad"] * 2.0 ** 20
    old = [values(rng, *given["gate"].shape, "f32", 2.0 ** 20) for _ in range(2)]
    check_case(gpu_lib, monkeypatch, given, tile, "f32", "f16", "gelu", old)


@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (0, 1, 3, 6)])
def test_f16_results_that_f16_holds(gpu_lib, monkeypatch, m, n, k, tile):  # noqa: F811
    # dg and du go to 2^19 and beyond; weights and lhs are small.
    given, _ = inputs(m + n + k, m, n, k, tile, "f16", "f16", "f32")
    given["grad"], given["u"], given["g"] = given["grad"] * 2.0 ** 12, given["u"] * 64, given["g"] * 64
    for name in ("x", "gate", "up_"):
        given[name] = ref.to_type((given[name] * 2.0 ** -10).astype(np.float32), "f16").astype(np.float64)
    check_case(gpu_lib, monkeypatch, given, tile, "f16", "f32")


@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (0, 1, 4, 6)])
def test_rows_of_different_sizes(gpu_lib, monkeypatch, m, n, k, tile):  # noqa: F811
    given, _ = inputs(m + n + k, m, n, k, tile, "f16", "f32", "f32")
    given["grad"] = given["grad"] * 2.0 ** -(np.arange(given["grad"].shape[0])[:, None] % 28.0)
    check_case(gpu_lib, monkeypatch, given, tile, "f32", "f32")


def test_nothing_but_zeros(gpu_lib):  # noqa: F811
    given, _ = inputs(1, 70, 96, 80, (1, 16, 16), "f16", "f32", "f32")
    given["grad"] = np.zeros_like(given["grad"])
    got, _ = ref.run_backward(gpu_lib, activation="silu", tile=(1, 16, 16), type="f16", out="f32", pre_type="f32", **given)
    for x in got:
        assert (x == 0).all()


@pytest.mark.parametrize("m,n", [(0, 32), (8, 0)])
def test_sums_over_nothing(gpu_lib, m, n):  # noqa: F811
    given, _ = inputs(1, m, n, 48, (1, 16, 16), "f16", "f32", "f32")
    got, _ = ref.run_backward(gpu_lib, activation="silu", tile=(1, 16, 16), type="f16", out="f32", pre_type="f32", **given)
    for x in got:
        assert (x == 0).all()


@pytest.mark.parametrize("strange", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("power", [0, 30, -30])
def test_values_that_are_not_finite_are_not_the_largest(gpu_lib, strange, power):  # noqa: F811
    given, _ = inputs(9, 70, 96, 80, (1, 16, 16), "f16", "f32", "f32")
    given["grad"] = given["grad"] * 2.0 ** power
    given["grad"][20, 30] = 0  # (not the largest one)
    run = dict(activation="silu", tile=(1, 16, 16), type="f16", out="f32", pre_type="f32")
    clean, _ = ref.run_backward(gpu_lib, **run, **given)
    given["grad"][20, 30] = strange
    got, _ = ref.run_backward(gpu_lib, **run, **given)
    rows, cols = np.arange(70) != 20, np.arange(96) != 30
    assert not np.isfinite(got[0][20]).any() and not np.isfinite(got[1][30]).any() and not np.isfinite(got[2][30]).any()
    assert np.isfinite(clean[0]).all() and np.isfinite(clean[1]).all()
    np.testing.assert_array_equal(got[0][rows], clean[0][rows])
    np.testing.assert_array_equal(got[1][cols], clean[1][cols])
    np.testing.assert_array_equal(got[2][cols], clean[2][cols])


# (more pieces of work than the first pass has threads, eight columns each and one)
@pytest.mark.parametrize("at", [(0, 0), (-1, -1), (500, 170), (-1, 0)])
@pytest.mark.parametrize("m,n,k,tile", [(1040, 2064, 32, (1, 16, 16)), (700, 399, 12, (5, 7, 6))])
def test_the_largest_wherever_it_is(gpu_lib, monkeypatch, m, n, k, tile, at):  # noqa: F811
    given, _ = inputs(m + n + k, m, n, k, tile, "f16", "f32", "f32")
    given["grad"][at], given["u"][at], given["g"][at] = 2.0 ** 19, 1.0, 1.0
    check_case(gpu_lib, monkeypatch, given, tile, "f32", "f32")


@pytest.mark.parametrize("m,n,k", [(50, 640, 256), (24, 2048, 256), (400, 1008, 512)])
def test_replayed_with_gradients_of_another_size(gpu_lib, m, n, k):  # noqa: F811
    rng = np.random.default_rng(m)
    p, held = abi.GatedMmt4dBackwardParams(), {"lhs": ref.matrix(values(rng, m, k, "f16"), 1, 16, "f16"), "lhs_grad": ref.empty(m, k, 1, "f32")}
    ref.tiles_into(p, m, n, k, (1, 16, 16))
    p.flags = abi.GATED_MMT4D_TYPE_F16F16F32 | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_PRE_F32
    for name in ("gate", "up"):
        held[name] = ref.matrix(values(rng, n, k, "f16", 0.1), 16, 16, "f16")
        held[name + "_pre"] = ref.matrix(values(rng, m, n, "f32"), 1, 16, "f32")
        held[name + "_grad"] = ref.empty(n, k, 16, "f32")
    held["out_grad"] = ref.matrix(values(rng, m, n, "f32"), 1, 16, "f32")
    for name, buffer in held.items():
        buffer.into(p, name)
    keep, size = ref.workspace(gpu_lib, "gated_mmt4d_backward", p)
    results = lambda: [ref.fetched(held[name], t0, 16) for name, t0 in (("lhs_grad", 1), ("gate_grad", 16), ("up_grad", 16))]  # noqa: E731
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=stream):
            gpu_lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            ref.call(gpu_lib, "gated_mmt4d_backward", p)
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)
    first = held["out_grad"].device[:4 * m * n].view(torch.float32).clone()
    clean = None
    for power in (0, 25, -30, 3):
        held["out_grad"].device[:4 * m * n].view(torch.float32).copy_(first * 2.0 ** power)
        keep[:size].fill_(0xFF)
        ref.call(gpu_lib, "gated_mmt4d_backward", p)
        want = results()
        clean = want if clean is None else clean
        for name in ("lhs_grad", "gate_grad", "up_grad"):
            held[name].device[:-64].fill_(0x55)
        keep[:size].fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, eager, plain in zip(results(), want, clean):
            np.testing.assert_array_equal(got, eager)
            np.testing.assert_array_equal(got, plain * 2.0 ** power)  # (a power of two changes no bits of these)

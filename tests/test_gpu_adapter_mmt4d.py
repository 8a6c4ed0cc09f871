"""Low-rank adapters on the GPU against 64 bits; the bounds are derived in feed_forward_reference.py."""
import ctypes as C

import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, up, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


def indices(rng, rows, count, order):
    """Of every row: its adapter, or none."""
    if order == "one":
        return np.full(rows, rng.integers(0, count), np.int32)
    if order == "mixed":
        return rng.integers(-1, count, rows).astype(np.int32)
    if order == "all":
        return (rng.permutation(max(rows, count))[:rows] % count).astype(np.int32)
    index = np.sort(rng.integers(-1, count, rows)).astype(np.int32)  # runs
    return rng.permutation(count).astype(np.int32)[index] * (index >= 0) - (index < 0)


def inputs(seed, m, n, k, rank, count, tile, type, order):
    rng = np.random.default_rng(seed)
    rows, cols, depth = up(m, tile[0]), up(n, tile[1]), up(k, tile[2])
    x = values(rng, rows, depth, type)
    down = values(rng, count * rank, depth, type, 1 / np.sqrt(max(1, depth))).reshape(count, rank, depth)
    up_ = values(rng, count * cols, rank, type, 0.3).reshape(count, cols, rank)
    return rng, x, down, up_, indices(rng, rows, count, order), (rng.random(count) + 0.5).astype(np.float32)


def check_case(lib, m, n, k, rank, count, tile, type, out, order, accumulate=True, scaled=True, **layout):
    rng, x, down, up_, index, scales = inputs(m + n + k + rank, m, n, k, rank, count, tile, type, order)
    scales = scales if scaled else None
    init = values(rng, x.shape[0], up_.shape[1], out) if accumulate else None
    got, kernel = ref.run_adapters(lib, x, down, up_, index, scales, tile, type, out, init, **layout)
    part, off = ref.adapters(x, down, up_, index, scales)
    total = part if init is None else part + init
    check(got, total, off + (ref.U * np.abs(total) if accumulate else 0), out)
    without = (index < 0) | (index >= count)
    np.testing.assert_array_equal(got[without], 0 if init is None else init[without])
    return kernel


# m, n, k, rank, count, tile, order
PROBLEMS = [
    (1, 16, 16, 4, 1, (1, 16, 16), "one"), (1, 1000, 4096, 16, 8, (1, 16, 16), "one"), (2, 100, 300, 8, 3, (1, 16, 16), "all"),
    (5, 77, 1000, 16, 9, (1, 16, 16), "mixed"), (16, 1040, 3000, 16, 16, (16, 16, 16), "all"), (17, 333, 257, 13, 4, (1, 16, 16), "mixed"),
    (31, 96, 96, 32, 31, (1, 1, 32), "all"), (40, 200, 640, 64, 5, (1, 16, 16), "runs"), (64, 640, 1152, 16, 64, (1, 16, 16), "all"),
    (65, 129, 2000, 24, 7, (1, 16, 32), "mixed"), (100, 1000, 384, 8, 2, (4, 8, 16), "runs"), (130, 500, 500, 100, 6, (1, 16, 16), "runs"),
    (200, 264, 1024, 1, 3, (1, 1, 64), "mixed"), (257, 513, 300, 128, 3, (1, 16, 8), "runs"), (300, 300, 130, 16, 300, (16, 16, 16), "mixed"),
    (777, 544, 328, 64, 11, (1, 16, 32), "runs"), (600, 100, 200, 16, 40, (1, 16, 16), "mixed"), (40, 50, 70, 5, 4, (5, 7, 6), "mixed"),
    (9, 30, 500, 300, 3, (3, 5, 16), "all"), (20, 20, 1030, 2, 5, (2, 4, 24), "runs"), (12, 31, 7, 3, 2, (1, 1, 1), "mixed"),
    (90, 257, 2056, 16, 5, (1, 1, 2056), "mixed"), (33, 64, 128, 256, 4, (1, 16, 16), "runs"), (48, 100, 64, 20, 2, (1, 4, 16), "one"),
    (530, 48, 40, 12, 3, (1, 16, 8), "runs"), (70, 90, 300, 45, 5, (1, 16, 16), "mixed"), (33, 100, 200, 64, 4, (1, 4, 16), "runs"),
]


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,rank,count,tile,order", PROBLEMS)
def test_added_to_a_result(gpu_lib, m, n, k, rank, count, tile, order, type, out):  # noqa: F811
    check_case(gpu_lib, m, n, k, rank, count, tile, type, type if out == "same" else out, order)


@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("m,n,k,rank,count,tile,order", [PROBLEMS[i] for i in (1, 3, 4, 7, 8, 10, 11, 13, 15, 17, 19, 22)])
def test_alone_and_without_scales(gpu_lib, m, n, k, rank, count, tile, order, out):  # noqa: F811
    check_case(gpu_lib, m, n, k, rank, count, tile, "bf16", "bf16" if out == "same" else out, order, accumulate=False, scaled=False)


# Many rows of few adapters, which are put in order first: all sorts of tiles, ranks and columns, rows of one adapter, of few and of many.
ORDERED = [
    (1000, 1000, 1024, 64, 12, (1, 16, 16), "mixed"), (905, 520, 2000, 100, 30, (1, 16, 8), "mixed"), (704, 2048, 512, 64, 9, (16, 16, 16), "mixed"),
    (2100, 300, 1500, 64, 500, (1, 4, 16), "mixed"), (1500, 1040, 2050, 16, 21, (4, 8, 16), "runs"), (6000, 512, 512, 30, 4, (1, 16, 32), "one"),
    (3000, 400, 3000, 32, 2047, (1, 16, 16), "mixed"), (500, 2000, 3104, 64, 7, (1, 1, 1552), "mixed"),
    (9001, 256, 256, 16, 40, (1, 16, 16), "mixed"), (5000, 256, 256, 16, 5, (1, 16, 16), "runs"),
]


@pytest.mark.parametrize("accumulate", [True, False])
@pytest.mark.parametrize("type,out", [("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("m,n,k,rank,count,tile,order", ORDERED)
def test_many_rows_of_few_adapters(gpu_lib, m, n, k, rank, count, tile, order, type, out, accumulate):  # noqa: F811
    check_case(gpu_lib, m, n, k, rank, count, tile, type, out, order, accumulate)


def test_rows_in_order_give_the_same_bits_and_strange_indices_name_nobody(gpu_lib):  # noqa: F811
    rng, x, down, up_, index, scales = inputs(5, 1000, 512, 2048, 64, 12, (1, 16, 16), "bf16", "mixed")
    run = lambda i: ref.run_adapters(gpu_lib, x, down, up_, i, scales, (1, 16, 16), "bf16", "f32")[0]  # noqa: E731
    first = run(index)
    for _ in range(3):
        np.testing.assert_array_equal(run(index), first)
    others = index.copy()
    others[::3] = rng.choice([-2 ** 31, -1, 12, 13, 2 ** 31 - 1], others[::3].size)
    got = run(others)
    np.testing.assert_array_equal(got[1::3], first[1::3])
    assert not got[::3].any()
    assert not run(np.full_like(index, 12)).any()


@pytest.mark.parametrize("gap,offset", [(8, 8), (16, 24), (3, 5)])
@pytest.mark.parametrize("m,n,k,rank,tile", [(1, 100, 300, 16, (1, 16, 16)), (40, 100, 384, 8, (1, 16, 16)), (48, 80, 384, 12, (16, 16, 16)),
                                             (300, 200, 512, 64, (1, 1, 32))])
def test_strides_and_offsets(gpu_lib, m, n, k, rank, tile, gap, offset):  # noqa: F811
    check_case(gpu_lib, m, n, k, rank, 5, tile, "f16", "f16", "mixed", layout={name: dict(gap=gap, offset=offset) for name in
                                                                            ("lhs", "out")}, down_gap=(gap, gap), up_gap=(8, gap))


def test_host_operands(gpu_lib):  # noqa: F811
    layout = {"lhs": dict(gap=2, offset=3), "out": dict(gap=2, offset=3)}
    check_case(gpu_lib, 20, 48, 96, 8, 5, (4, 16, 16), "f16", "f32", "mixed", layout=layout, host=True)
    check_case(gpu_lib, 20, 48, 96, 8, 5, (4, 16, 16), "f16", "f32", "mixed", accumulate=False, layout=layout, host=True)


@pytest.mark.parametrize("rank,count,k", [(0, 3, 64), (8, 0, 64), (8, 3, 0)])
def test_nobody_has_an_adapter(gpu_lib, rank, count, k):  # noqa: F811
    rng = np.random.default_rng(0)
    x, down, up_ = values(rng, 20, k, "bf16"), np.zeros((count, rank, k)), np.zeros((count, 32, rank))
    index = np.zeros(20, np.int32)
    got, _ = ref.run_adapters(gpu_lib, x, down, up_, index, None, (1, 16, 16), "bf16", "f32")
    assert (got == 0).all()
    init = values(rng, 20, 32, "f32")
    got, _ = ref.run_adapters(gpu_lib, x, down, up_, index, None, (1, 16, 16), "bf16", "f32", init)
    np.testing.assert_array_equal(got, init)


def test_indices_out_of_range_name_nobody(gpu_lib):  # noqa: F811
    rng, x, down, up_, index, scales = inputs(1, 40, 64, 128, 16, 4, (1, 16, 16), "bf16", "all")
    index[[0, 7, 20, 39]] = [4, -5, 2 ** 31 - 1, -2 ** 31]
    init = values(rng, 40, 64, "f32")
    got, _ = ref.run_adapters(gpu_lib, x, down, up_, index, scales, (1, 16, 16), "bf16", "f32", init)
    part, off = ref.adapters(x, down, up_, index, scales)
    check(got, init + part, off + ref.U * np.abs(init + part), "f32")
    np.testing.assert_array_equal(got[[0, 7, 20, 39]], init[[0, 7, 20, 39]])


@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("m,rank", [(40, 16), (300, 64), (300, 8)])
def test_values_that_are_not_finite_stay_with_their_rows(gpu_lib, m, rank, order):  # noqa: F811
    rng, x, down, up_, index, scales = inputs(2, m, 96, 272, rank, 5, (1, 16, 16), "bf16", order)
    clean, _ = ref.run_adapters(gpu_lib, x, down, up_, index, scales, (1, 16, 16), "bf16", "f32")
    down[1, 0, 5], up_[2, 30, 1], scales[3], x[m // 2, 100] = np.nan, np.inf, np.inf, np.nan
    got, _ = ref.run_adapters(gpu_lib, x, down, up_, index, scales, (1, 16, 16), "bf16", "f32")
    rows = ~np.isin(index, (1, 2, 3)) & (np.arange(m) != m // 2)
    np.testing.assert_array_equal(got[rows], clean[rows])
    assert rows.sum() > 10
    assert np.isnan(got[index == 1]).all()
    touched = (index == 2) & (np.arange(m) != m // 2)
    assert not np.isfinite(got[touched, 30]).any()
    np.testing.assert_array_equal(np.delete(got[touched], 30, 1), np.delete(clean[touched], 30, 1))


@pytest.mark.parametrize("m,order", [(1, "one"), (64, "all"), (600, "runs")])
def test_the_same_call_gives_the_same_bits_whoever_else_is_there(gpu_lib, m, order):  # noqa: F811
    rng, x, down, up_, index, scales = inputs(3, m, 256, 2048, 16, 8, (1, 16, 16), "bf16", order)
    run = lambda i: ref.run_adapters(gpu_lib, x, down, up_, i, scales, (1, 16, 16), "bf16", "f32")[0]  # noqa: E731
    first = run(index)
    for _ in range(3):
        np.testing.assert_array_equal(run(index), first)
    # A row's result depends on its adapter and not on the rows beside it.
    others = index.copy()
    others[::2] = (others[::2] + 3) % 8
    np.testing.assert_array_equal(run(others)[1::2], first[1::2])


@pytest.mark.parametrize("m", [3, 200])
def test_a_pool_beyond_32_bits(gpu_lib, m):  # noqa: F811
    # 70 adapters whose parts lie 2^25 elements apart: 4.6 GiB of each.
    rng, x, down, up_, index, scales = inputs(4, m, 64, 256, 16, 70, (1, 16, 16), "bf16", "all")
    index[-1] = 69
    gap = 1 << 25
    pools = [torch.zeros(69 * gap + 16 * 256, dtype=torch.int16, device="cuda") for _ in range(2)]
    for pool, v in zip(pools, (down, up_)):
        bits = torch.from_numpy(ref.raw(v, "bf16").view(np.int16).reshape(70, -1)).cuda()
        for a in range(70):
            pool[a * gap:a * gap + bits.shape[1]] = bits[a]
    held = {"lhs": ref.matrix(x, 1, 16, "bf16"), "out": ref.empty(m, 64, 1, "f32")}
    d_index, d_scales = torch.from_numpy(index).cuda(), torch.from_numpy(scales).cuda()
    p = abi.AdapterMmt4dParams()
    ref.tiles_into(p, m, 64, 256, (1, 16, 16))
    p.rank, p.count = 16, 70
    for name, b in held.items():
        b.into(p, name)
    p.down_buffer, p.up_buffer, p.down_stride0, p.up_stride0, p.down_stride1, p.up_stride1 = \
        pools[0].data_ptr(), pools[1].data_ptr(), gap, gap, 256, 16
    p.index_buffer, p.scales_buffer = d_index.data_ptr(), d_scales.data_ptr()
    p.flags = abi.ADAPTER_MMT4D_TYPE_BF16BF16F32
    keep, _ = ref.workspace(gpu_lib, "adapter_mmt4d", p)
    ref.call(gpu_lib, "adapter_mmt4d", p)
    part, off = ref.adapters(x, down, up_, index, scales)
    check(ref.fetched(held["out"], 1, 16), part, off, "f32")


@pytest.mark.parametrize("m0", [1, 16])
def test_a_result_beyond_32_bits(gpu_lib, m0):  # noqa: F811
    # 4.5 GiB of bf16; rows without an adapter but for the last 48.
    rows, cols, k = 73728, 32768, 32
    rng, x, down, up_, index, scales = inputs(5, 48, cols, k, 8, 3, (m0, 16, 16), "bf16", "all")
    whole = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    whole[-48:] = torch.from_numpy(index).cuda()
    lhs = torch.zeros(rows * k, dtype=torch.int16, device="cuda")
    lhs[-48 * k:] = torch.from_numpy(ref.raw(ref.tiled(x, m0, 16), "bf16").view(np.int16).reshape(-1)).cuda()
    out = torch.full((rows // m0, cols // 16, m0, 16), 7, dtype=torch.bfloat16, device="cuda")
    held = {"down": ref.Buffer(3, 8 * k, "bf16", data=down), "up": ref.Buffer(3, cols * 8, "bf16", data=up_)}
    p = abi.AdapterMmt4dParams()
    ref.tiles_into(p, rows, cols, k, (m0, 16, 16))
    p.rank, p.count = 8, 3
    for name, b in held.items():
        b.into(p, name)
    p.down_stride1, p.up_stride1 = k, 8
    p.lhs_buffer, p.lhs_stride0, p.out_buffer, p.out_stride0 = lhs.data_ptr(), k * m0, out.data_ptr(), cols * m0
    p.index_buffer = whole.data_ptr()
    p.flags = abi.ADAPTER_MMT4D_TYPE_BF16BF16BF16
    keep, _ = ref.workspace(gpu_lib, "adapter_mmt4d", p)
    ref.call(gpu_lib, "adapter_mmt4d", p)
    for first in range(0, rows - 48, 8192):
        assert bool((out[first // m0:min(first + 8192, rows - 48) // m0] == 0).all())
    part, off = ref.adapters(x, down, up_, index, None)
    check(ref.untiled(out[-48 // m0:].float().cpu().numpy()), part, off, "bf16")

"""Which kernels the host picks for gated products, their gradients and adapters, on the CPU (host_launches.py): every kernel is picked
for a problem of the GPU tests, and where every kernel was timed the one picked is near the best."""
import re

import pytest

from feed_forward_kernels import GATED, GATED_LINES, GATED_TIMES, LHS_GRADS, WEIGHT_GRADS, WEIGHT_GRADS_TIMES
from feed_forward_reference import up
from host_launches import recorder  # noqa: F401
from iree_amd import abi
from test_gpu_adapter_mmt4d import ORDERED, PROBLEMS as ADAPTERS
from test_gpu_gated_backward import PROBLEMS as BACKWARD, SPLIT

GIB = 1 << 30
F32, SAME = {"f16": 1, "bf16": 3}, {"f16": 2, "bf16": 4}


def filled(p, m, n, k, tile, operands, flags):
    (p.M0, p.N0, p.K0), p.M, p.N, p.K = tile, up(m, tile[0]) // tile[0], up(n, tile[1]) // tile[1], up(k, tile[2]) // tile[2]
    panel = {"m": p.K * p.M0 * p.K0, "n": p.K * p.N0 * p.K0, "o": p.N * p.M0 * p.N0}
    for i, (name, of) in enumerate(operands):
        setattr(p, name + "_buffer", (i + 1) * 16 * GIB)
        setattr(p, name + "_stride0", panel[of])
    p.flags = flags
    return p


def gated(recorder, m, n, k, tile, type="bf16"):  # noqa: F811
    p = filled(abi.GatedMmt4dParams(), m, n, k, tile, (("lhs", "m"), ("gate", "n"), ("up", "n"), ("out", "o")), SAME[type] | abi.GATED_MMT4D_SILU)
    return recorder.call("iree_uk_mi355x_gated_mmt4d_p", p)


def backward(recorder, m, n, k, tile, which, type="bf16"):  # noqa: F811
    given = [("lhs", "m"), ("gate", "n"), ("up", "n"), ("gate_pre", "o"), ("up_pre", "o"), ("out_grad", "o")]
    grads = [("lhs_grad", "m")] * ("l" in which) + [("gate_grad", "n"), ("up_grad", "n")] * ("w" in which)
    p = filled(abi.GatedMmt4dBackwardParams(), m, n, k, tile, given + grads, SAME[type] | abi.GATED_MMT4D_SILU)
    p.workspace_buffer, p.workspace_size = 512 * GIB, 256 * GIB
    kernel = recorder.call("iree_uk_mi355x_gated_mmt4d_backward_p", p)[0]
    tile = re.search(r"product16_block_kernelILNS_5FloatE\dELi(\d)ELi(\d)ELi\dELb0ENS_%s" % ("7LhsGrad" if which == "l" else "11WeightGrads"), kernel)
    if tile is None:
        assert "gated_lhs_grad_sums" in kernel, kernel
        return 0, 0
    return int(tile[1]), int(tile[2])


@pytest.mark.parametrize("type", ["bf16", "f16"])
def test_every_gated_kernel_is_picked(recorder, type):  # noqa: F811
    picked = set()
    for kernel, m, n, k, tile in GATED:
        assert gated(recorder, m, n, k, tile, type)[1] == "gated_mmt4d_" + kernel, (m, n, k, tile)
        picked.add(kernel)
    assert len(picked) == 17


def test_rows_of_whole_lines(recorder):  # noqa: F811
    picked = set()
    for kernel, m, n, k, tile in GATED_LINES:
        symbol, name = gated(recorder, m, n, k, tile)
        form = re.search(r"product16_lines_kernelILNS_5FloatE\dELi\dELi\dELb(\d)", symbol)
        assert form and name == "gated_mmt4d_" + kernel, (m, n, k, tile)
        picked.add((kernel, form[1]))
    assert len(picked) == 11  # (two of the nine with weights past the caches too)
    # (K not a multiple of 64, rows in tiles, and two workgroups to a compute unit)
    for m, n, k, tile in ((1371, 3273, 96, (1, 16, 16)), (1371, 3273, 130, (1, 16, 8)), (2048, 4096, 512, (16, 16, 16)),
                          (1573, 4882, 128, (1, 16, 16)), (914, 8341, 64, (1, 16, 16)), (314, 12557, 64, (1, 16, 16))):
        assert "product16_block_kernel" in gated(recorder, m, n, k, tile)[0]


@pytest.mark.parametrize("type", ["bf16", "f16"])
def test_every_tile_of_the_gradients_is_picked(recorder, type):  # noqa: F811
    for problems, which, count in ((LHS_GRADS, "l", 8), (WEIGHT_GRADS, "w", 7)):
        for picked, m, n, k, tile in problems:
            assert backward(recorder, m, n, k, tile, which, type) == picked, (m, n, k, tile)
        assert len({x[0] for x in problems}) == count


def test_what_is_picked_is_near_the_fastest(recorder):  # noqa: F811
    slower = {"gated": [], "weights": []}
    for m, n, k, m0, times in GATED_TIMES:
        name = gated(recorder, m, n, k, (m0, 16, 16))[1].replace("gated_mmt4d_", "")
        assert name in times, (m, n, k, m0, name)
        slower["gated"].append(times[name] / min(times.values()))
    for m, n, k, m0, times in WEIGHT_GRADS_TIMES:
        picked = backward(recorder, m, n, k, (m0, 16, 16), "w")
        assert picked in times, (m, n, k, m0, picked)
        slower["weights"].append(times[picked] / min(times.values()))
    for of, x in slower.items():
        assert sum(x) / len(x) < 1.05 and max(x) < 1.2, (of, x)


def all_gradients(recorder, m, n, k, tile):  # noqa: F811
    given = [("lhs", "m"), ("gate", "n"), ("up", "n"), ("gate_pre", "o"), ("up_pre", "o"), ("out_grad", "o")]
    p = filled(abi.GatedMmt4dBackwardParams(), m, n, k, tile, given + [("lhs_grad", "m"), ("gate_grad", "n"), ("up_grad", "n")], SAME["bf16"] | abi.GATED_MMT4D_SILU)
    p.workspace_buffer, p.workspace_size = 512 * GIB, 256 * GIB
    kernel = recorder.call("iree_uk_mi355x_gated_mmt4d_backward_p", p)[0]
    return next((x for x in ("both_grads", "11WeightGrads", "gated_lhs_grad_sums") if x in kernel), None)


# Both products in one launch, the parts of lhs_grad's sums behind it; or one after the other.
@pytest.mark.parametrize("m,n,k,last", [(130, 1000, 512, "gated_lhs_grad_sums"), (206, 353, 749, "both_grads"), (16, 256, 128, "both_grads"),
                                        (4096, 11008, 4096, "11WeightGrads"),
                                        (30, 8567, 3462, "gated_lhs_grad_sums")])
def test_small_gradients_in_one_launch(recorder, m, n, k, last):  # noqa: F811
    assert all_gradients(recorder, m, n, k, (1, 16, 16)) == last


def test_both_products_in_one_launch_are_tested(recorder):  # noqa: F811
    assert sum(all_gradients(recorder, m, n, k, tile) == "both_grads" for m, n, k, tile in BACKWARD) > 5


def test_split_sums_are_tested(recorder):  # noqa: F811
    for m, n, k, tile in SPLIT:
        assert backward(recorder, m, n, k, tile, "l") == (0, 0), (m, n, k, tile)


# Large weights that few rows read go past the caches.
@pytest.mark.parametrize("m,n,k,streams", [(1, 14336, 4096, True), (1, 2048, 2048, False), (1, 28672, 8192, True), (64, 14336, 4096, True), (64, 28672, 8192, True),
                                           (100, 4100, 4096, False), (40, 11008, 4096, True), (128, 11008, 4096, True), (129, 28672, 8192, False)])
def test_weights_past_the_caches(recorder, m, n, k, streams):  # noqa: F811
    kernel, _ = gated(recorder, m, n, k, (1, 16, 16))
    past = re.search(r"few_kernelILNS_5FloatE\dELi\dELi\dELb(\d)|block_kernelILNS_5FloatE\dELi\dELi\dELi\dELb(\d)|lines_kernelILNS_5FloatE\dELi\dELi\dELb(\d)", kernel)
    assert (past is not None and (past[1] or past[2] or past[3]) == "1") == streams, kernel



def adapters(recorder, m, n, k, rank, count, tile, type, out):  # noqa: F811
    p = filled(abi.AdapterMmt4dParams(), m, n, k, tile, (("lhs", "m"), ("out", "o")), (SAME if out == "same" else F32)[type])
    p.rank, p.count = rank, count
    depth, cols = p.K * p.K0, p.N * p.N0
    p.down_buffer, p.down_stride0, p.down_stride1 = 64 * GIB, rank * depth, depth
    p.up_buffer, p.up_stride0, p.up_stride1 = 80 * GIB, rank * cols, rank
    p.index_buffer, p.scales_buffer, p.workspace_buffer, p.workspace_size = 96 * GIB, 112 * GIB, 512 * GIB, 256 * GIB
    kernel = recorder.call("iree_uk_mi355x_adapter_mmt4d_p", p)[0]
    form = re.search(r"adapter_up_kernelILNS_5FloatE\dELS2_\dELb(\d)ELi(\d)ELi\dELb(\d)ELb(\d)", kernel)
    return tuple(form.groups()) if form else kernel


@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["f32", "same"])
def test_every_adapter_kernel_is_tested(recorder, type, out):  # noqa: F811
    picked = {adapters(recorder, m, n, k, rank, count, tile, type, out) for m, n, k, rank, count, tile, _ in ADAPTERS}
    # up to 16 ranks, up to 32, up to 64, more; each with whole sixteens of columns and without
    forms = {(half, chunks, fast, many) for half, chunks, many in (("1", "1", "0"), ("0", "1", "0"), ("0", "2", "0"), ("0", "2", "1")) for fast in "01"}
    assert forms == {x for x in picked if isinstance(x, tuple)}
    assert any("adapter_up_generic" in x for x in picked)


def test_many_rows_of_few_adapters_are_put_in_order(recorder):  # noqa: F811
    for m, n, k, rank, count, tile, _ in ORDERED:
        adapters(recorder, m, n, k, rank, count, tile, "bf16", "f32")
        assert recorder.lib.recorded_launches() == 3, (m, n, k, rank, count, tile)
    # Few rows, as many adapters as rows, little to read, one adapter, and more than have numbers in LDS.
    for m, n, k, rank, count in ((16, 14336, 4096, 64, 2), (64, 14336, 4096, 16, 64), (40, 11008, 4096, 16, 16), (300, 300, 300, 16, 3),
                                 (4096, 4096, 4096, 64, 1), (4096, 4096, 4096, 64, 2048)):
        adapters(recorder, m, n, k, rank, count, (1, 16, 16), "bf16", "f32")
        assert recorder.lib.recorded_launches() == 2, (m, n, k, rank, count)

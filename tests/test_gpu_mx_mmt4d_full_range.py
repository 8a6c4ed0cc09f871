"""Products of E4M3 codes of the format's whole range, on the GPU: 448 next to 2^-9, NaN codes.

A row of the lhs has magnitudes that add up to 2688 at most, times 6 of the rhs less than 2^14, and every product is a multiple
of 2^-10: with scales of one every sum of some of them is exact in f32, in any order and for every type of result, and the result
is that of 64 bits, rounded once. The eights of most rows cancel against the columns of the rhs that are equal
within an eight, so that what the small codes add is all that is left, in results of 16 bits too."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_mmt4d import PROBLEMS, exact_codes, in_64_bits, product
from test_gpu_mx_pack import on_device
from test_mx_mmt4d_choice_on_host import KERNELS, RESIDENT

pytestmark = pytest.mark.gpu


def code_of(value):
    return int(np.flatnonzero(ref.E4M3 == abs(value))[0]) + (128 if value < 0 else 0)


# Eights whose products lie farthest apart: largest and least of the format, of the codes below 4 and of those from 4 on, and
# next to 4. The first ones cancel.
EDGES = [[448, -448, 2.0 ** -9, 0, 0, 0, 0, 0], [3.75, -3.75, 2.0 ** -9, 3.75, 0, 0, 0, -3.75], [448, 0.5, -448, 0, 0, 0, 0, 0],
         [-448, 0, 3.5, 0, 448, 0, 2.0 ** -8, -3.5], [4.5, 3.75, -4.5, -3.75, 2.0 ** -9, 0, 0, 0],
         [448, 2.0 ** -9, 0, 0, 0, 0, 0, 0], [3.75, 2.0 ** -9, 0, 0, 0, 0, 0, 0], [448, 4.5, 0, 0, 0, 0, 0, 0],
         [4, 3.75, 4.5, -4, 2.0 ** -6, 0, 0, 0], [0, 0, 0, 0, 7 * 2.0 ** -9, 2.0 ** -9, 1.875, 240]]
CANCEL = 5


def lhs_of_the_whole_range(rng, rows, k):
    codes = np.zeros((rows, k // 8, 8), np.uint8)
    edges = np.array([[code_of(v) for v in e] for e in EDGES], np.uint8)
    for row in range(rows):
        left, all_cancel = 2688.0, rng.random() < 0.75
        for eight in rng.permutation(k // 8)[:32]:
            if rng.random() < 0.5:
                new = rng.permutation(edges[rng.integers(CANCEL if all_cancel else len(edges))])
            else:
                new = rng.integers(0, 256, 8).astype(np.uint8)
                new[new % 128 == 127] -= 1
                if all_cancel:
                    new[4:] = new[:4] ^ 128          # each with its opposite, but for two small ones
                    new[[3, 7]] = rng.integers(1, 9, 2)
                new = rng.permutation(new)
            size = ref.E4M3[new & 127].sum()
            if size <= left:
                codes[row, eight] = new
                left -= size
    return codes.reshape(rows, k), np.full((rows, k // 32), 127, np.uint8)


def rhs_of_ones(rng, rows, k):
    """Random codes with scales of one; in three rows of four the same code (not zero) for each eight of K."""
    codes, _ = ref.random_codes(rng, rows, k, "e2m1")
    level = rng.random(rows) < 0.75
    same = (rng.integers(1, 8, (rows, k // 8)) | 8 * rng.integers(0, 2, (rows, k // 8))).astype(np.uint8).repeat(8, 1)
    codes[level] = same[level]
    return codes, np.full((rows, k // 32), 127, np.uint8)


def wanted(lhs, rhs, out_type):
    bound = np.abs(ref.widen(*lhs, "e4m3")).sum(1).max() * 6
    assert bound <= 2.0 ** 14 and (np.abs(ref.widen(*lhs, "e4m3")) * 512 % 1 == 0).all()
    return ref.to_type(in_64_bits(lhs, rhs, "e4m3").astype(np.float32), out_type)


def check(lib, rows, cols, k, tile, out_type):
    rng = np.random.default_rng(rows + cols + k)
    lhs, rhs = lhs_of_the_whole_range(rng, rows, k), rhs_of_ones(rng, cols, k)
    got, kernel = product(lib, lhs, rhs, tile, "e4m3", out_type)
    np.testing.assert_array_equal(got, ref.raw(wanted(lhs, rhs, out_type), out_type))
    return kernel


@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
def test_sums(gpu_lib, m, n, k, tile, out_type):  # noqa: F811
    check(gpu_lib, *(ref.up(v, t) for v, t in zip((m, n, k), tile)), tile, out_type)


@pytest.mark.parametrize("out,rows,cols,k,m0,n0,kernel", [q[1:] for q in KERNELS if q[0] == "e4m3"])
def test_sums_of_every_kernel(gpu_lib, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    assert check(gpu_lib, rows, cols, k, (m0, n0, 128), out).decode() == "mx_mmt4d_" + kernel


@pytest.mark.parametrize("out,rows,cols,k,m0,n0", [q[1:] for q in RESIDENT if q[0] == "e4m3"])
def test_sums_with_the_lhs_in_registers(gpu_lib, out, rows, cols, k, m0, n0):  # noqa: F811
    rng = np.random.default_rng(rows + cols)
    lhs, rhs = lhs_of_the_whole_range(rng, rows, k), rhs_of_ones(rng, 160, k)
    times = -(-cols // 160)
    d = [on_device(ref.tiled(lhs[0], m0, 128)), on_device(ref.tiled(lhs[1], m0, 4)),
         on_device(ref.to_bytes(ref.tiled(rhs[0], n0, 128), "e2m1")).view(-1).repeat(times),
         on_device(ref.tiled(rhs[1], n0, 4)).view(-1).repeat(times)]
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[out]
    result = torch.full((rows // m0, cols // n0, m0, n0), 3.0, dtype=dtype, device="cuda")
    p = ref.mmt4d_params(*(x.data_ptr() for x in d), result.data_ptr(), (rows // m0, cols // n0, k // 128), (m0, n0, 128), "e4m3", out)
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == b"mx_mmt4d_resident"
    want = torch.from_numpy(wanted(lhs, rhs, out)).to(dtype).cuda().repeat(1, times)[:, :cols]
    assert torch.equal(result.permute(0, 2, 1, 3).reshape(rows, cols), want)


@pytest.mark.parametrize("out_type", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,tile", [(1, 64, 512, (1, 16, 128)), (16, 64, 1024, (16, 16, 128)), (70, 200, 640, (1, 16, 128)),
                                        (300, 300, 512, (16, 16, 128)), (300, 700, 512, (1, 16, 128)), (6, 8, 96, (2, 4, 96))])
def test_codes_that_are_nan(gpu_lib, m, n, k, tile, out_type):  # noqa: F811
    # A row with a NaN code is NaN, whatever it is multiplied by; the other rows are what they are.
    rng = np.random.default_rng(m)
    rows, cols, depth = (ref.up(v, t) for v, t in zip((m, n, k), tile))
    lhs, rhs = exact_codes(rng, rows, depth, "e4m3"), exact_codes(rng, cols, depth, "e2m1")
    rhs[0][cols // 2] = 0
    bad = np.zeros(rows, bool)
    if rows > 1:
        bad[[rows // 3, rows - 1]] = True
        lhs[0][rows // 3, depth // 2] = 0xFF
    bad[rows - 1] = True
    lhs[0][rows - 1, 5] = 0x7F
    got = ref.from_raw(product(gpu_lib, lhs, rhs, tile, "e4m3", out_type)[0], out_type)
    assert np.isnan(got[bad]).all()
    want = ref.to_type(in_64_bits(lhs, rhs, "e4m3")[~bad].astype(np.float32), out_type)
    np.testing.assert_array_equal(got[~bad], want)

"""Products of microscaled operands on the GPU.

Most inputs here are drawn so that every product and every partial sum is a multiple of one power
of two and below 2^24 of it: their sums are exact in f32 in any order, and the result is compared
bit for bit with 64 bits, rounded once where it is f16 or bf16. Where scales span a wide range a
result may be off by its summation: at most K additions, each off by at most one unit in the last
place of a partial sum, which the sum of the magnitudes bounds: K * 2^-23 * sum |a| |b|.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_pack import GUARD, guarded, host, on_device

pytestmark = pytest.mark.gpu


def exact_codes(rng, rows, cols, format):
    """Operands whose sums are exact: E2M1 of any kind (multiples of 2^-1 up to 6), E4M3 between 2^-3 and 7.5 (multiples of
    2^-6), zeros too, scales 2^0 and 2^1: products are multiples of 2^-7 up to 180, and their sums stay below 2^17."""
    codes, _ = ref.random_codes(rng, rows, cols, format)
    if format == "e4m3":
        codes = (codes & 0x87) | (rng.integers(4, 10, codes.shape) << 3).astype(np.uint8)
        codes[rng.random(codes.shape) < 0.1] = 0
    return codes, rng.integers(127, 129, (rows, cols // 32)).astype(np.uint8)


def product(lib, lhs, rhs, tile, lhs_format, out_type, init=None, m=None, n=None):
    """lhs, rhs: (codes, scales) of matrices padded to whole tiles -> the result as a matrix, raw, and the kernel."""
    m0, n0, k0 = tile
    rows, cols, k = lhs[0].shape[0], rhs[0].shape[0], lhs[0].shape[1]
    d = [on_device(ref.to_bytes(ref.tiled(lhs[0], m0, k0), lhs_format)), on_device(ref.tiled(lhs[1], m0, k0 // 32)),
         on_device(ref.to_bytes(ref.tiled(rhs[0], n0, k0), "e2m1")), on_device(ref.tiled(rhs[1], n0, k0 // 32))]
    dtype = np.float32 if out_type == "f32" else np.uint16
    nbytes = rows * cols * np.dtype(dtype).itemsize
    out = guarded(nbytes)
    if init is not None:
        out[:nbytes] = on_device(ref.tiled(ref.raw(init, out_type).reshape(rows, cols), m0, n0))
    p = ref.mmt4d_params(*(x.data_ptr() for x in d), out.data_ptr(), (rows // m0, cols // n0, k // k0), tile, lhs_format,
                         out_type, init is not None)
    lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    got = host(out)
    assert (got[nbytes:] == GUARD).all()
    return ref.untiled(got[:nbytes].view(dtype).reshape(rows // m0, cols // n0, m0, n0)), lib.iree_uk_mi355x_last_kernel()


def in_64_bits(lhs, rhs, lhs_format):
    return ref.widen(*lhs, lhs_format) @ ref.widen(*rhs, "e2m1").T


def check_exact(lib, rng, m, n, k, tile, lhs_format, out_type, accumulate=False):
    rows, cols, depth = ref.up(m, tile[0]), ref.up(n, tile[1]), ref.up(k, tile[2])
    lhs, rhs = exact_codes(rng, rows, depth, lhs_format), exact_codes(rng, cols, depth, "e2m1")
    init = ref.to_type(rng.integers(-64, 64, (rows, cols)), out_type) if accumulate else None
    got, kernel = product(lib, lhs, rhs, tile, lhs_format, out_type, init)
    want = in_64_bits(lhs, rhs, lhs_format) + (init if accumulate else 0)
    assert np.abs(want).max() < 2.0 ** 17
    np.testing.assert_array_equal(got, ref.raw(ref.to_type(want.astype(np.float32), out_type), out_type))
    return kernel


# Rows (one token to a small prompt), columns and depths of every kernel, odd ones among them; tiles that the fast kernels
# take (one row tall, or 128 deep) and tiles that only the general one does.
PROBLEMS = [
    (1, 16, 32, (1, 16, 32)), (1, 16, 128, (1, 16, 128)), (1, 100, 300, (1, 16, 128)), (1, 1000, 4096, (1, 16, 128)),
    (2, 512, 1024, (1, 16, 128)), (3, 200, 640, (1, 1, 128)), (5, 77, 1000, (1, 16, 128)), (8, 300, 2048, (8, 16, 128)),
    (16, 1040, 3000, (16, 16, 128)), (16, 64, 14336, (1, 16, 128)), (17, 333, 257, (1, 16, 128)), (31, 96, 96, (1, 1, 32)),
    (33, 500, 640, (16, 16, 128)), (64, 640, 1152, (1, 16, 128)), (65, 129, 2000, (1, 16, 128)), (100, 1000, 384, (4, 8, 128)),
    (128, 128, 512, (16, 16, 128)), (130, 700, 1000, (1, 16, 128)), (200, 264, 4096, (1, 1, 128)),
    (257, 513, 896, (1, 16, 128)), (300, 300, 130, (16, 16, 128)), (512, 1000, 640, (16, 16, 128)), (777, 1040, 544, (1, 16, 32)),
    (40, 50, 70, (5, 7, 64)), (9, 30, 500, (3, 5, 96)), (20, 20, 1030, (2, 4, 256)),
]


@pytest.mark.parametrize("out_type", ["f32", "bf16"])
@pytest.mark.parametrize("lhs_format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("m,n,k,tile", PROBLEMS)
def test_exact_sums(gpu_lib, m, n, k, tile, lhs_format, out_type):
    check_exact(gpu_lib, np.random.default_rng(m + n + k), m, n, k, tile, lhs_format, out_type)


@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lhs_format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (0, 3, 8, 12, 17, 20, 21, 23)])
def test_accumulate(gpu_lib, m, n, k, tile, lhs_format, out_type):
    check_exact(gpu_lib, np.random.default_rng(m), m, n, k, tile, lhs_format, out_type, accumulate=True)


@pytest.mark.parametrize("lhs_format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("m,n,k,tile", [PROBLEMS[i] for i in (1, 3, 8, 11, 13, 17, 19, 21, 23)])
def test_scales_of_a_wide_range(gpu_lib, m, n, k, tile, lhs_format):
    rng = np.random.default_rng(k)
    rows, cols, depth = ref.up(m, tile[0]), ref.up(n, tile[1]), ref.up(k, tile[2])
    lhs = ref.random_codes(rng, rows, depth, lhs_format, (97, 157))
    rhs = ref.random_codes(rng, cols, depth, "e2m1", (97, 157))
    got, _ = product(gpu_lib, lhs, rhs, tile, lhs_format, "f32")
    a, b = ref.widen(*lhs, lhs_format), ref.widen(*rhs, "e2m1")
    bound = depth * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)
    assert (np.abs(got - a @ b.T) <= bound).all()


@pytest.mark.parametrize("lhs_format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("m,n,k,tile", [(1, 64, 512, (1, 16, 128)), (16, 64, 1024, (16, 16, 128)), (70, 200, 640, (1, 16, 128)),
                                        (300, 300, 512, (16, 16, 128)), (6, 8, 96, (2, 4, 96))])
def test_scales_that_are_nan_and_scales_at_the_ends(gpu_lib, m, n, k, tile, lhs_format):
    rng = np.random.default_rng(m)
    rows, cols, depth = ref.up(m, tile[0]), ref.up(n, tile[1]), ref.up(k, tile[2])
    lhs, rhs = exact_codes(rng, rows, depth, lhs_format), exact_codes(rng, cols, depth, "e2m1")
    lhs[1][m // 2, -1] = 255                 # a NaN block makes its row NaN, zero codes or not
    lhs[0][m // 2, -32:] = 0
    rhs[1][n - 1, 0] = 255
    if m > 2:
        lhs[1][0, :], lhs[1][1, :] = 254, 0  # the largest scale times the least
        rhs[1][0, :], rhs[1][1, :] = 0, 254
    got, _ = product(gpu_lib, lhs, rhs, tile, lhs_format, "f32")
    with np.errstate(over="ignore", invalid="ignore"):
        want = in_64_bits(lhs, rhs, lhs_format).astype(np.float32)
    assert np.isnan(got[m // 2]).all() and np.isnan(got[:, n - 1]).all()
    rest = ~np.isnan(want)
    tiny = np.abs(want) < 2.0 ** -126        # (may come out as zero)
    # Rows and columns with scales 0 and 254 only, all the same: exact. But a sum of both signs whose magnitudes add up to
    # 2^128 or more may pass f32's range on its way, in one order or another, whatever its end is: infinities, and NaN
    # where two of them meet. Below that no partial sum, of any part of the products, reaches 2^128.
    with np.errstate(invalid="ignore"):
        within = np.abs(ref.widen(*lhs, lhs_format)) @ np.abs(ref.widen(*rhs, "e2m1")).T < 2.0 ** 128
    same = rest & ~tiny & within
    np.testing.assert_array_equal(got[same], want[same])
    assert (np.abs(got[rest & tiny]) <= 2.0 ** -126).all()
    assert not np.isfinite(got[rest & ~np.isfinite(want)]).any()


@pytest.mark.parametrize("accumulate", [False, True])
def test_no_depth(gpu_lib, accumulate):
    out = torch.full((4 * 32,), 3.0, device="cuda")
    some = torch.zeros(64, dtype=torch.uint8, device="cuda")
    p = ref.mmt4d_params(*[some.data_ptr()] * 4, out.data_ptr(), (4, 2, 0), (1, 16, 128), "e4m3", "f32", accumulate)
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    assert bool((out == (3.0 if accumulate else 0.0)).all())


@pytest.mark.parametrize("m,n,k,tile,lhs_gap,rhs_gap,out_gap,offset", [
    (40, 100, 384, (1, 16, 128), 32, 32, 4, 32), (40, 100, 384, (1, 16, 128), 2, 6, 3, 2),
    (48, 80, 384, (16, 16, 128), 64, 128, 16, 64), (300, 200, 512, (1, 1, 128), 64, 32, 1, 64),
    (2, 64, 640, (1, 16, 128), 10, 34, 5, 6), (700, 300, 256, (4, 4, 128), 32, 64, 7, 0)])
@pytest.mark.parametrize("lhs_format", ["e2m1", "e4m3"])
def test_strides_and_offsets(gpu_lib, lhs_format, m, n, k, tile, lhs_gap, rhs_gap, out_gap, offset):
    rng = np.random.default_rng(n)
    m0, n0, k0 = tile
    rows, cols = ref.up(m, m0), ref.up(n, n0)
    lhs, rhs = exact_codes(rng, rows, k, lhs_format), exact_codes(rng, cols, k, "e2m1")

    def spread(x, gap_bytes, first_bytes):
        x = np.ascontiguousarray(x).view(np.uint8)
        x = x.reshape(x.shape[0], -1)
        buf = np.full(first_bytes + x.shape[0] * (x.shape[1] + gap_bytes), GUARD, np.uint8)
        buf[first_bytes:].reshape(x.shape[0], -1)[:, :x.shape[1]] = x
        return on_device(buf)

    lb = ref.BITS[lhs_format]
    d_l = spread(ref.to_bytes(ref.tiled(lhs[0], m0, k0), lhs_format), lhs_gap * lb // 8, offset * lb // 8)
    d_ls = spread(ref.tiled(lhs[1], m0, k0 // 32), lhs_gap, offset)
    d_r = spread(ref.to_bytes(ref.tiled(rhs[0], n0, k0), "e2m1"), rhs_gap // 2, offset // 2)
    d_rs = spread(ref.tiled(rhs[1], n0, k0 // 32), rhs_gap, offset)
    row = cols * m0 + out_gap
    out = torch.full((offset + (rows // m0) * row,), -7.0, device="cuda")
    p = ref.mmt4d_params(d_l.data_ptr(), d_ls.data_ptr(), d_r.data_ptr(), d_rs.data_ptr(), out.data_ptr(),
                         (rows // m0, cols // n0, k // k0), tile, lhs_format, "f32")
    p.lhs_offset = p.lhs_scales_offset = p.rhs_offset = p.rhs_scales_offset = p.out_offset = offset
    p.lhs_stride0 += lhs_gap
    p.lhs_scales_stride0 += lhs_gap
    p.rhs_stride0 += rhs_gap
    p.rhs_scales_stride0 += rhs_gap
    p.out_stride0 = row
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    want = np.full(out.numel(), -7.0, np.float32)
    want[offset:].reshape(rows // m0, row)[:, :cols * m0] = \
        ref.tiled(in_64_bits(lhs, rhs, lhs_format), m0, n0).reshape(rows // m0, -1)
    np.testing.assert_array_equal(host(out), want)


def test_panels_that_coincide(gpu_lib):
    # A stride of zero broadcasts one panel: every row of tiles is the same product.
    rng = np.random.default_rng(1)
    lhs, rhs = exact_codes(rng, 1, 512, "e4m3"), exact_codes(rng, 64, 512, "e2m1")
    d = [on_device(lhs[0]), on_device(lhs[1]), on_device(ref.to_bytes(ref.tiled(rhs[0], 16, 128), "e2m1")),
         on_device(ref.tiled(rhs[1], 16, 4))]
    out = torch.zeros(70, 64, device="cuda")
    p = ref.mmt4d_params(*(x.data_ptr() for x in d), out.data_ptr(), (70, 4, 4), (1, 16, 128), "e4m3", "f32")
    p.lhs_stride0 = p.lhs_scales_stride0 = 0
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    want = np.repeat(in_64_bits(lhs, rhs, "e4m3"), 70, 0).astype(np.float32)
    np.testing.assert_array_equal(host(out), want)


def test_host_operands(gpu_lib):
    rng = np.random.default_rng(3)
    lhs, rhs = exact_codes(rng, 20, 256, "e4m3"), exact_codes(rng, 48, 256, "e2m1")
    a, s, b, t = lhs[0], lhs[1], ref.to_bytes(ref.tiled(rhs[0], 16, 128), "e2m1"), ref.tiled(rhs[1], 16, 4)
    out = np.full((20, 50), 9, np.float32)
    p = ref.mmt4d_params(a.ctypes.data, s.ctypes.data, b.ctypes.data, t.ctypes.data, out.ctypes.data, (20, 3, 2),
                         (1, 16, 128), "e4m3", "f32")
    p.out_stride0 = 50
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    np.testing.assert_array_equal(out[:, :48], in_64_bits(lhs, rhs, "e4m3"))
    assert (out[:, 48:] == 9).all()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (64, 1024, 4096), (512, 1024, 2048)])
def test_the_same_call_gives_the_same_bits(gpu_lib, m, n, k):
    rng = np.random.default_rng(7)
    lhs, rhs = ref.random_codes(rng, m, k, "e4m3"), ref.random_codes(rng, n, k, "e2m1")
    first, _ = product(gpu_lib, lhs, rhs, (1, 16, 128), "e4m3", "f32")
    for _ in range(3):
        np.testing.assert_array_equal(product(gpu_lib, lhs, rhs, (1, 16, 128), "e4m3", "f32")[0], first)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_rhs_beyond_32_bits(gpu_lib, m):
    # 4.5 GiB of weights in tiles of 16 x 128: ones, but for the last 64 columns. All values are multiples of 1/2 below 16: sums of
    # 131072 products with random signs are multiples of 1/4 below 2^22.
    cols, k = 73728, 131072
    rng = np.random.default_rng(m)
    lhs, last = exact_codes(rng, m, k, "e2m1"), exact_codes(rng, 64, k, "e2m1")
    codes = torch.full((cols * k // 2,), 0x22, dtype=torch.uint8, device="cuda")
    scales = torch.full((cols * k // 32,), 127, dtype=torch.uint8, device="cuda")
    codes[-32 * k:] = on_device(ref.to_bytes(ref.tiled(last[0], 16, 128), "e2m1"))
    scales[-2 * k:] = on_device(ref.tiled(last[1], 16, 4))
    out = torch.zeros(m, cols, device="cuda")
    a, s = on_device(ref.to_bytes(lhs[0], "e2m1")), on_device(lhs[1])
    p = ref.mmt4d_params(a.data_ptr(), s.data_ptr(), codes.data_ptr(), scales.data_ptr(), out.data_ptr(),
                         (m, cols // 16, k // 128), (1, 16, 128), "e2m1", "f32")
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    want = torch.from_numpy(ref.widen(*lhs, "e2m1").sum(1)).float().cuda()
    assert float(want.abs().max()) < 2.0 ** 22
    assert bool((out[:, :-64] == want[:, None]).all())
    np.testing.assert_array_equal(host(out[:, -64:].contiguous()).reshape(m, 64), in_64_bits(lhs, last, "e2m1"))


@pytest.mark.parametrize("m0", [1, 16])
def test_a_result_beyond_32_bits(gpu_lib, m0):
    # 4.5 GiB of bf16: ones times the weights, but for the last 48 rows.
    rows, cols = 73728, 32768
    rng = np.random.default_rng(m0)
    last, rhs = exact_codes(rng, 48, 128, "e4m3"), exact_codes(rng, cols, 128, "e2m1")
    lhs = torch.full((rows * 128,), 0x38, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows * 4,), 127, dtype=torch.uint8, device="cuda")
    lhs[-48 * 128:], scales[-48 * 4:] = on_device(ref.tiled(last[0], m0, 128)), on_device(ref.tiled(last[1], m0, 4))
    b, t = on_device(ref.to_bytes(ref.tiled(rhs[0], 16, 128), "e2m1")), on_device(ref.tiled(rhs[1], 16, 4))
    out = torch.zeros(rows // m0, cols // 16, m0, 16, dtype=torch.int16, device="cuda")
    p = ref.mmt4d_params(lhs.data_ptr(), scales.data_ptr(), b.data_ptr(), t.data_ptr(), out.data_ptr(),
                         (rows // m0, cols // 16, 1), (m0, 16, 128), "e4m3", "bf16")
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    ones = ref.raw(ref.to_type(ref.widen(*rhs, "e2m1").sum(1).astype(np.float32), "bf16"), "bf16").view(np.int16)
    ones = torch.from_numpy(ones.reshape(cols // 16, 1, 16)).cuda()
    for first in range(0, rows - 48, 8192):
        end = min(first + 8192, rows - 48)
        assert bool((out[first // m0:end // m0] == ones).all())
    got = ref.untiled(host(out[-48 // m0:].contiguous()).view(np.uint16).reshape(48 // m0, cols // 16, m0, 16))
    want = in_64_bits(last, rhs, "e4m3").astype(np.float32)
    np.testing.assert_array_equal(got, ref.raw(ref.to_type(want, "bf16"), "bf16"))


def test_accumulation_into_a_host_result_with_gaps(gpu_lib):
    rng = np.random.default_rng(4)
    lhs, rhs = exact_codes(rng, 20, 256, "e4m3"), exact_codes(rng, 48, 256, "e2m1")
    a, s, b, t = lhs[0], lhs[1], ref.to_bytes(ref.tiled(rhs[0], 16, 128), "e2m1"), ref.tiled(rhs[1], 16, 4)
    out = np.full((20, 50), 9, np.float32)
    p = ref.mmt4d_params(a.ctypes.data, s.ctypes.data, b.ctypes.data, t.ctypes.data, out.ctypes.data, (20, 3, 2),
                         (1, 16, 128), "e4m3", "f32", True)
    p.out_stride0 = 50
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    np.testing.assert_array_equal(out[:, :48], in_64_bits(lhs, rhs, "e4m3") + 9)
    assert (out[:, 48:] == 9).all()

"""Which kernel the host picks for a product of microscaled operands, on the CPU (host_launches.py): every kernel for every pair
of types is picked for some problem, and for problems that were timed with every kernel the one picked is within 8 % of the
best."""
import pytest

import mx_reference as ref
from host_launches import recorder  # noqa: F401

# lhs, result, rows, columns, K, rows of a lhs tile and of a rhs tile -> the kernel. K of one chunk of 128, then K long enough
# for a kernel to go round its loop.
KERNELS = [
    ("e2m1", "f32", 1302, 1551, 128, 1, 1, "block_128x128"),
    ("e2m1", "bf16", 1957, 2127, 128, 1, 1, "block_128x192"),
    ("e2m1", "bf16", 2667, 2351, 640, 1, 1, "block_128x256"),
    ("e2m1", "bf16", 1232, 785, 128, 16, 1, "block_128x64"),
    ("e2m1", "f32", 3856, 3292, 384, 16, 1, "block_256x256"),
    ("e2m1", "f32", 1424, 1369, 128, 16, 1, "block_64x128"),
    ("e2m1", "f32", 592, 434, 128, 1, 1, "block_64x64"),
    ("e2m1", "f32", 1, 16, 128, 1, 16, "few_16x16"),
    ("e2m1", "f32", 15, 16, 128, 1, 1, "few_16x16_staged"),
    ("e2m1", "f32", 1, 4106, 128, 1, 1, "few_16x32"),
    ("e2m1", "f32", 304, 401, 128, 1, 1, "few_16x32_staged"),
    ("e2m1", "bf16", 1, 8224, 128, 1, 16, "few_16x64"),
    ("e2m1", "bf16", 357, 688, 128, 1, 16, "few_16x64_staged"),
    ("e2m1", "f32", 202, 310, 128, 1, 1, "few_32x16_staged"),
    ("e2m1", "f32", 394, 331, 128, 1, 1, "few_32x32_staged"),
    ("e2m1", "bf16", 459, 640, 1280, 1, 16, "few_32x64_staged"),
    ("e4m3", "bf16", 1584, 1312, 128, 16, 16, "block_128x128"),
    ("e4m3", "bf16", 1824, 2221, 128, 16, 1, "block_128x192"),
    ("e4m3", "bf16", 2206, 2880, 1152, 1, 16, "block_128x256"),
    ("e4m3", "bf16", 1920, 1040, 128, 16, 16, "block_128x64"),
    ("e4m3", "bf16", 2768, 5191, 128, 16, 1, "block_256x256"),
    ("e4m3", "bf16", 795, 1248, 128, 1, 16, "block_64x128"),
    ("e4m3", "bf16", 432, 592, 128, 16, 16, "block_64x64"),
    ("e4m3", "bf16", 1, 16, 128, 1, 16, "few_16x16"),
    ("e4m3", "bf16", 10, 16, 128, 1, 16, "few_16x16_staged"),
    ("e4m3", "bf16", 3, 4192, 128, 1, 16, "few_16x32"),
    ("e4m3", "bf16", 256, 288, 128, 16, 16, "few_16x32_staged"),
    ("e4m3", "bf16", 1, 8313, 128, 1, 1, "few_16x64"),
    ("e4m3", "bf16", 226, 1078, 128, 1, 1, "few_16x64_staged"),
    ("e4m3", "bf16", 214, 302, 128, 1, 1, "few_32x16_staged"),
    ("e4m3", "bf16", 336, 389, 128, 16, 1, "few_32x32_staged"),
    ("e4m3", "bf16", 470, 560, 1024, 1, 16, "few_32x64_staged"),
    ("e4m3", "f32", 2732, 2182, 128, 1, 1, "block_128x128"),
    ("e4m3", "f32", 2582, 1584, 128, 1, 16, "block_128x192"),
    ("e4m3", "f32", 3081, 1968, 1664, 1, 16, "block_128x256"),
    ("e4m3", "f32", 1663, 1153, 128, 1, 1, "block_128x64"),
    ("e4m3", "f32", 3102, 4498, 640, 1, 1, "block_256x256"),
    ("e4m3", "f32", 658, 1551, 128, 1, 1, "block_64x128"),
    ("e4m3", "f32", 558, 464, 128, 1, 1, "block_64x64"),
    ("e4m3", "f32", 2, 16, 128, 1, 1, "few_16x16"),
    ("e4m3", "f32", 9, 16, 128, 1, 16, "few_16x16_staged"),
    ("e4m3", "f32", 1, 4144, 128, 1, 16, "few_16x32"),
    ("e4m3", "f32", 288, 240, 128, 16, 16, "few_16x32_staged"),
    ("e4m3", "f32", 1, 8232, 128, 1, 1, "few_16x64"),
    ("e4m3", "f32", 304, 816, 128, 16, 16, "few_16x64_staged"),
    ("e4m3", "f32", 288, 253, 128, 16, 1, "few_32x16_staged"),
    ("e4m3", "f32", 414, 309, 128, 1, 1, "few_32x32_staged"),
    ("e4m3", "f32", 565, 523, 512, 1, 1, "few_32x64_staged"),
    ("e2m1", "bf16", 1699, 1254, 896, 1, 1, "block_128x128"),
    ("e2m1", "f32", 2576, 1551, 896, 16, 1, "block_128x192"),
    ("e2m1", "f32", 2744, 2504, 896, 8, 8, "block_128x256"),
    ("e2m1", "bf16", 772, 1292, 896, 1, 1, "block_128x64"),
    ("e2m1", "bf16", 2640, 4800, 896, 8, 16, "block_256x256"),
    ("e2m1", "bf16", 795, 2360, 896, 1, 8, "block_64x128"),
    ("e2m1", "bf16", 584, 442, 896, 8, 1, "block_64x64"),
    ("e2m1", "bf16", 1, 16, 4736, 1, 16, "few_16x16"),
    ("e2m1", "f32", 16, 16, 4608, 16, 8, "few_16x16_staged"),
    ("e2m1", "bf16", 8, 4160, 4608, 8, 16, "few_16x32"),
    ("e2m1", "f32", 232, 544, 4608, 1, 16, "few_16x32_staged"),
    ("e2m1", "bf16", 272, 912, 4736, 8, 16, "few_16x64_staged"),
    ("e2m1", "bf16", 248, 276, 4480, 1, 1, "few_32x16_staged"),
    ("e2m1", "f32", 366, 372, 4480, 1, 1, "few_32x32_staged"),
    ("e2m1", "f32", 592, 424, 4480, 16, 8, "few_32x64_staged"),
    ("e4m3", "bf16", 1444, 1440, 896, 1, 16, "block_128x128"),
    ("e4m3", "bf16", 1744, 2413, 896, 16, 1, "block_128x192"),
    ("e4m3", "bf16", 2440, 2464, 1152, 8, 8, "block_128x256"),
    ("e4m3", "bf16", 1840, 1062, 896, 8, 1, "block_128x64"),
    ("e4m3", "bf16", 2352, 5840, 896, 16, 16, "block_256x256"),
    ("e4m3", "bf16", 833, 1176, 896, 1, 8, "block_64x128"),
    ("e4m3", "bf16", 528, 512, 896, 8, 1, "block_64x64"),
    ("e4m3", "bf16", 1, 16, 5120, 1, 16, "few_16x16"),
    ("e4m3", "bf16", 8, 19, 4736, 8, 1, "few_16x16_staged"),
    ("e4m3", "bf16", 1, 4176, 4608, 1, 16, "few_16x32"),
    ("e4m3", "bf16", 260, 272, 4608, 1, 16, "few_16x32_staged"),
    ("e4m3", "bf16", 330, 767, 5376, 1, 1, "few_16x64_staged"),
    ("e4m3", "bf16", 200, 312, 4480, 8, 8, "few_32x16_staged"),
    ("e4m3", "bf16", 299, 536, 4480, 1, 8, "few_32x32_staged"),
    ("e4m3", "bf16", 673, 384, 4480, 1, 16, "few_32x64_staged"),
    ("e4m3", "f32", 2316, 2672, 896, 1, 8, "block_128x128"),
    ("e4m3", "f32", 1904, 2224, 896, 16, 16, "block_128x192"),
    ("e4m3", "f32", 2072, 3208, 1408, 8, 1, "block_128x256"),
    ("e4m3", "f32", 1632, 2464, 896, 16, 8, "block_128x64"),
    ("e4m3", "f32", 2704, 4832, 896, 8, 16, "block_256x256"),
    ("e4m3", "f32", 1232, 800, 896, 8, 1, "block_64x128"),
    ("e4m3", "f32", 715, 761, 896, 1, 1, "block_64x64"),
    ("e4m3", "f32", 1, 19, 4608, 1, 1, "few_16x16"),
    ("e4m3", "f32", 8, 16, 4608, 8, 1, "few_16x16_staged"),
    ("e4m3", "f32", 1, 4128, 4608, 1, 8, "few_16x32"),
    ("e4m3", "f32", 177, 384, 4480, 1, 16, "few_16x32_staged"),
    ("e4m3", "f32", 805, 312, 5120, 1, 8, "few_16x64_staged"),
    ("e4m3", "f32", 301, 264, 4480, 1, 8, "few_32x16_staged"),
    ("e4m3", "f32", 344, 389, 4480, 8, 1, "few_32x32_staged"),
    ("e4m3", "f32", 464, 616, 4480, 16, 8, "few_32x64_staged"),
    ("e4m3", "bf16", 1, 8232, 4608, 1, 1, "few_16x64"),
    ("e4m3", "f32", 3, 8240, 4608, 1, 1, "few_16x64"),
]

# The same for the kernel that keeps the lhs in registers: whole and partial shares of K, rows and columns, matrices and tiles.
RESIDENT = [
    ("e2m1", "f32", 16, 28672, 8192, 1, 16), ("e2m1", "f16", 9, 33008, 4096, 1, 16), ("e2m1", "bf16", 13, 28672, 8064, 1, 16),
    ("e2m1", "f32", 16, 57000, 4096, 16, 1), ("e2m1", "bf16", 5, 40001, 3200, 1, 1), ("e2m1", "f16", 4, 33001, 4096, 1, 1),
    ("e4m3", "bf16", 16, 28672, 8192, 1, 16), ("e4m3", "f16", 16, 57008, 4096, 16, 16), ("e4m3", "bf16", 1, 28672, 8064, 1, 1),
    ("e4m3", "f32", 16, 28672, 8192, 16, 16), ("e4m3", "f32", 9, 40000, 3200, 1, 16), ("e4m3", "f32", 3, 28675, 8192, 1, 1),
    ("e4m3", "f32", 8, 33008, 4096, 1, 8),
]

# The same as above, and microseconds of the four best kernels.
TIMES = [
    ("e2m1", "f16", 352, 8653, 3584, 16, 1, {"block_128x128": 20.17, "block_128x64": 21.10, "block_64x128": 25.58, "block_128x192": 26.14}),
    ("e2m1", "f16", 723, 6288, 6912, 1, 16, {"block_128x192": 27.07, "block_128x256": 29.82, "block_128x128": 34.54, "block_64x128": 39.86}),
    ("e2m1", "f16", 94, 10432, 256, 1, 16, {"block_128x64": 4.21, "block_64x64": 4.56, "block_64x128": 4.75, "block_128x128": 5.23}),
    ("e2m1", "bf16", 905, 13328, 1792, 1, 16, {"block_256x256": 22.40, "block_128x256": 24.93, "block_128x128": 26.07, "block_128x192": 28.29}),
    ("e2m1", "f32", 34, 17504, 512, 1, 16, {"block_64x128": 4.64, "block_64x64": 5.06, "block_128x64": 6.02, "block_128x128": 6.18}),
    ("e2m1", "f16", 198, 3654, 256, 1, 1, {"block_64x64": 4.06, "block_128x64": 4.81, "block_64x128": 4.90, "block_128x128": 6.35}),
    ("e2m1", "bf16", 2, 256, 11136, 1, 16, {"few_16x16": 4.23, "few_16x16_staged": 4.42, "few_32x16_staged": 5.29, "few_16x32": 5.33}),
    ("e2m1", "bf16", 17, 79, 12800, 1, 1, {"few_16x16_staged": 6.70, "few_32x16_staged": 7.69, "few_16x16": 8.59, "few_16x32_staged": 9.94}),
    ("e2m1", "f32", 8, 6208, 4736, 1, 16, {"few_16x32": 3.98, "few_16x32_staged": 4.44, "few_16x16": 4.61, "few_16x16_staged": 4.77}),
    ("e2m1", "f16", 562, 400, 9856, 1, 16, {"few_16x64": 9.34, "few_32x32_staged": 9.66, "few_16x64_staged": 9.83, "few_16x32": 10.94}),
    ("e2m1", "f32", 31, 4624, 3712, 1, 16, {"few_32x32_staged": 4.51, "few_32x16_staged": 4.97, "few_16x64": 5.21, "few_16x64_staged": 5.44}),
    ("e2m1", "f16", 59, 4752, 13056, 1, 16, {"few_32x64_staged": 14.37, "few_32x32_staged": 18.31, "few_32x16_staged": 19.53, "few_16x16_staged": 22.40}),
    ("e4m3", "bf16", 2960, 762, 7552, 16, 1, {"block_128x128": 36.54, "block_64x128": 42.33, "block_128x64": 45.73, "block_64x64": 48.59}),
    ("e4m3", "f16", 416, 11360, 8960, 16, 16, {"block_128x192": 38.88, "block_128x256": 43.66, "block_128x128": 47.99, "block_64x128": 50.25}),
    ("e4m3", "f16", 384, 20059, 7168, 1, 1, {"block_128x256": 55.22, "block_128x128": 63.93, "block_256x256": 79.45, "block_128x192": 83.30}),
    ("e4m3", "bf16", 1477, 992, 128, 1, 16, {"block_128x64": 4.15, "block_64x128": 4.18, "block_64x64": 4.31, "block_128x128": 5.01}),
    ("e4m3", "f16", 544, 7088, 256, 16, 16, {"block_64x128": 5.91, "block_128x128": 7.05, "block_64x64": 7.41, "block_128x64": 7.74}),
    ("e4m3", "f16", 208, 2470, 4864, 16, 1, {"block_64x64": 11.46, "block_128x64": 15.85, "few_16x32_staged": 16.96, "block_64x128": 16.97}),
    ("e4m3", "f16", 2, 288, 8576, 1, 16, {"few_16x16": 4.27, "few_16x16_staged": 4.49, "few_16x32": 5.36, "few_16x32_staged": 5.57}),
    ("e4m3", "bf16", 19, 170, 7680, 1, 1, {"few_16x16_staged": 5.69, "few_32x16_staged": 6.93, "few_16x16": 7.77, "few_16x32_staged": 7.77}),
    ("e4m3", "bf16", 2, 24347, 1536, 1, 1, {"few_16x32": 7.11, "block_64x128": 7.26, "few_16x32_staged": 8.20, "few_16x16": 8.68}),
    ("e4m3", "bf16", 774, 96, 8704, 1, 16, {"few_16x32_staged": 6.69, "few_16x64_staged": 8.19, "few_16x32": 8.25, "few_32x32_staged": 8.48}),
    ("e4m3", "bf16", 32, 3225, 11776, 16, 1, {"few_32x16_staged": 9.93, "few_16x32_staged": 11.52, "few_32x32_staged": 12.43, "few_16x16_staged": 12.59}),
    ("e4m3", "f16", 135, 2448, 10496, 1, 16, {"few_32x64_staged": 15.31, "few_32x32_staged": 19.42, "few_16x32_staged": 21.61, "few_16x16_staged": 22.76}),
    ("e4m3", "f32", 3569, 11472, 256, 1, 16, {"block_128x128": 42.44, "block_64x128": 46.09, "block_128x64": 51.76, "block_128x256": 52.42}),
    ("e4m3", "f32", 523, 8352, 1408, 1, 16, {"block_128x192": 19.90, "block_64x128": 20.82, "block_128x128": 21.89, "block_128x256": 23.07}),
    ("e4m3", "f32", 2304, 608, 8448, 16, 16, {"block_64x128": 38.80, "block_64x64": 40.05, "block_128x64": 48.91, "block_128x128": 64.99}),
    ("e4m3", "f32", 3431, 144, 1024, 1, 16, {"block_64x64": 7.48, "block_64x128": 7.94, "block_128x64": 10.16, "block_128x128": 11.89}),
    ("e4m3", "f32", 62, 352, 8320, 1, 16, {"few_16x16_staged": 5.11, "few_16x32_staged": 6.18, "few_16x16": 7.23, "few_32x16_staged": 7.33}),
    ("e4m3", "f32", 522, 128, 12672, 1, 16, {"few_16x32_staged": 8.72, "few_16x32": 11.37, "few_16x64_staged": 11.60, "few_32x32_staged": 12.48}),
    ("e4m3", "f32", 57, 2672, 9088, 1, 16, {"few_32x32_staged": 10.45, "few_16x32_staged": 10.99, "few_16x64_staged": 11.93, "few_16x16_staged": 12.57}),
    ("e4m3", "f32", 524, 688, 12160, 1, 16, {"few_32x64_staged": 18.86, "few_16x32_staged": 20.25, "few_32x32_staged": 24.09, "few_16x64_staged": 24.75}),
]


def picked(recorder, lhs, out, rows, cols, k, m0, n0):  # noqa: F811
    p = ref.mmt4d_params(1 << 39, 2 << 39, 3 << 39, 4 << 39, 5 << 39, (rows // m0, cols // n0, k // 128), (m0, n0, 128), lhs, out)
    _, name = recorder.call("iree_uk_mi355x_mx_mmt4d_p", p)
    assert name.startswith("mx_mmt4d_")
    return name[len("mx_mmt4d_"):]


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,kernel", KERNELS)
def test_every_kernel_is_picked(recorder, lhs, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    assert picked(recorder, lhs, out, rows, cols, k, m0, n0) == kernel


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0", RESIDENT)
def test_the_lhs_stays_in_registers(recorder, lhs, out, rows, cols, k, m0, n0):  # noqa: F811
    assert picked(recorder, lhs, out, rows, cols, k, m0, n0) == "resident"


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,times", TIMES, ids=lambda v: "times" if isinstance(v, dict) else str(v))
def test_the_kernel_picked_is_among_the_best(recorder, lhs, out, rows, cols, k, m0, n0, times):  # noqa: F811
    name = picked(recorder, lhs, out, rows, cols, k, m0, n0)
    assert name in times
    assert times[name] <= 1.08 * min(times.values())


@pytest.mark.parametrize("change,kernel", [
    (lambda p: None, "block_64x128"),
    # What the fast kernels do not take: K that is not whole chunks, a tile's K other than a chunk, pieces off 16 bytes, scales
    # off 4.
    (lambda p: setattr(p, "K0", 96), "generic"),
    (lambda p: (setattr(p, "N0", 8), setattr(p, "K0", 64)), "generic"),
    (lambda p: setattr(p, "lhs_offset", 8), "generic"),
    (lambda p: setattr(p, "rhs_offset", 8), "generic"),
    (lambda p: setattr(p, "lhs_scales_offset", 2), "generic"),
    (lambda p: setattr(p, "rhs_scales_stride0", p.rhs_scales_stride0 + 2), "generic"),
    # What the block kernels do not take: tiles of the lhs of four rows, and rows or results farther apart than 32 bits reach.
    (lambda p: (setattr(p, "M0", 4), setattr(p, "M", p.M // 4), setattr(p, "lhs_stride0", 4 * p.lhs_stride0),
                setattr(p, "lhs_scales_stride0", 4 * p.lhs_scales_stride0), setattr(p, "out_stride0", 4 * p.out_stride0)), "few"),
    (lambda p: setattr(p, "rhs_stride0", 1 << 28), "few"),
    (lambda p: setattr(p, "out_stride0", 1 << 26), "few"),
    (lambda p: setattr(p, "lhs_stride0", 1 << 24), "few"),  # (nor does the lhs go through LDS)
])
def test_what_the_fast_kernels_do_not_take(recorder, change, kernel):  # noqa: F811
    p = ref.mmt4d_params(1 << 39, 2 << 39, 3 << 39, 4 << 39, 5 << 39, (1024, 128, 8), (1, 16, 128), "e4m3", "bf16")
    change(p)
    _, name = recorder.call("iree_uk_mi355x_mx_mmt4d_p", p)
    assert name.startswith("mx_mmt4d_" + kernel), name
    if p.lhs_stride0 == 1 << 24:
        assert not name.endswith("staged")


@pytest.mark.parametrize("tiles,tile,kernel", [
    # More rows of 16 or 32 than a grid has, in tiles that no block kernel takes; more columns than it has threads for.
    ((1 << 20, 1, 1), (4, 16, 128), "generic"), ((1 << 16, 1, 1), (4, 16, 128), "few"),
    ((10, 1 << 30, 1), (2, 1, 128), "generic"), ((10, 1 << 24, 1), (2, 1, 128), "few"),
    ((10, 1 << 30, 1), (1, 1, 128), "resident"), ((1 << 22, 1, 1), (1, 16, 128), "block")])
def test_grids_of_any_size(recorder, tiles, tile, kernel):  # noqa: F811
    p = ref.mmt4d_params(1 << 36, 2 << 39, 3 << 39, 4 << 39, 5 << 39, tiles, tile, "e4m3", "f32")
    _, name = recorder.call("iree_uk_mi355x_mx_mmt4d_p", p)
    assert name.startswith("mx_mmt4d_" + kernel), name

"""Quantisation into microscaled tiles and back on the GPU, bit for bit against a search in the
table of elements in 64 bits: both are exact up to one rounding, so nothing is left to tolerate.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu

GUARD = 0xA5


def on_device(x):
    return torch.from_numpy(np.ascontiguousarray(x).view(np.uint8).reshape(-1)).cuda()


def guarded(nbytes):
    return torch.full((nbytes + 64,), GUARD, dtype=torch.uint8, device="cuda")


def host(t):
    return t.cpu().numpy()


def quantised_by_gpu(lib, x, type, format, t0, t1):
    """x: f32 [rows][cols] that `type` holds."""
    rows, cols = x.shape
    src = on_device(ref.raw(x, type))
    n = ref.up(rows, t0) * ref.up(cols, t1)
    codes, scales = guarded(n * ref.BITS[format] // 8), guarded(n // 32)
    p = ref.pack_params(src.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), t0, t1, type, format)
    lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    codes, scales = host(codes), host(scales)
    assert (codes[-64:] == GUARD).all() and (scales[-64:] == GUARD).all()
    return codes[:-64], scales[:-64]


def wanted(x, format, t0, t1):
    codes, scales = ref.quantise(ref.padded(x, t0, t1), format)
    return ref.to_bytes(ref.tiled(codes, t0, t1), format).reshape(-1), ref.tiled(scales, t0, t1 // 32).reshape(-1)


SHAPES = [(1, 1, 1, 32), (1, 32, 1, 32), (3, 33, 16, 128), (17, 300, 16, 128), (5, 4095, 1, 128), (64, 256, 32, 64),
          (33, 100, 7, 96), (40, 31, 1, 32), (2, 8200, 3, 8224)]


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,t0,t1", SHAPES)
def test_pack(gpu_lib, type, format, rows, cols, t0, t1):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, cols))
    x = ref.to_type(x, type)
    got, want = quantised_by_gpu(gpu_lib, x, type, format, t0, t1), wanted(x, format, t0, t1)
    assert gpu_lib.iree_uk_mi355x_last_kernel() == b"mx_pack_rows"
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_pack_every_pattern(gpu_lib, type, format):
    # All 65536 patterns: in order (neighbours of a like size share a block, subnormals, infinities and NaNs among them),
    # and beside a value of the block's top binade, where they are rounded and saturate.
    bits = np.arange(65536, dtype=np.uint16)
    x = ref.from_raw(bits, type).reshape(-1, 32)
    with np.errstate(all="ignore"):
        by = np.where(np.isfinite(x), x, 0)
        y = np.repeat(by.reshape(-1, 1), 32, 1)[:, :32].copy()
        y *= np.linspace(-2, 2, 32, dtype=np.float32)  # multiples of every pattern, some beyond its type
    for m in (x, ref.to_type(y, type)):
        got, want = quantised_by_gpu(gpu_lib, m, type, format, 1, 32), wanted(m, format, 1, 32)
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[0], want[0])


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
def test_pack_f32_ends_of_the_range(gpu_lib, format):
    rows = []
    for top in (0.0, 2.0 ** -149, 2.0 ** -127, 2.0 ** -126, 2.0 ** -118, 1.99 * 2.0 ** -119, 6.5, 464.0, 480.0, 511.99,
                1.75 * 2.0 ** 127, 3.4028234e38, np.inf, -np.inf, np.nan):
        r = np.linspace(-1, 1, 32) * (top if np.isfinite(top) else 1.0)
        r[5] = top
        rows.append(r)
    # Ties between neighbouring elements, both signs, and zeros of both signs.
    table = ref.TABLE[format]
    middles = (table[1:] + table[:-1]) / 2
    ties = np.concatenate([middles, -middles, [0.0, -0.0]])
    ties = np.pad(ties, (0, -len(ties) % 31)).reshape(-1, 31)
    rows += [np.concatenate([[table[-1]], t]) for t in ties]
    x = np.array(rows).astype(np.float32)
    got, want = quantised_by_gpu(gpu_lib, x, "f32", format, 1, 32), wanted(x, format, 1, 32)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,t0,t1,strides", [
    (33, 70, 16, 128, (1, 40)), (300, 257, 16, 128, (1, 300)), (64, 128, 16, 128, (1, 64)), (5, 40, 1, 64, (200, 3)),
    (9, 64, 4, 32, (0, 1)), (9, 64, 4, 32, (1, 0)), (7, 96, 2, 96, (96, 1))])
def test_pack_strides(gpu_lib, type, format, rows, cols, t0, t1, strides):
    rng = np.random.default_rng(cols)
    flat = ref.to_type(rng.standard_normal((rows - 1) * strides[0] + (cols - 1) * strides[1] + 1), type)
    x = flat[np.arange(rows)[:, None] * strides[0] + np.arange(cols)[None] * strides[1]]
    src = on_device(ref.raw(flat, type))
    o0, o1 = -(-rows // t0), -(-cols // t1)
    # Panels with room between them, operands that begin behind the buffers' starts.
    row, gap, offset = o1 * t0 * t1, 6, 10
    codes = guarded((offset + o0 * (row + gap)) * ref.BITS[format] // 8)
    scales = guarded(3 + o0 * (row // 32 + 5))
    p = ref.pack_params(src.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), t0, t1, type, format, strides,
                        row + gap, row // 32 + 5)
    p.out_offset, p.scales_offset = offset, 3
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    want_codes, want_scales = wanted(x, format, t0, t1)
    expect = np.full(codes.numel(), GUARD, np.uint8)
    bits = ref.BITS[format]
    for i in range(o0):
        at = (offset + i * (row + gap)) * bits // 8
        expect[at:at + row * bits // 8] = want_codes.reshape(o0, -1)[i]
    np.testing.assert_array_equal(host(codes), expect)
    expect = np.full(scales.numel(), GUARD, np.uint8)
    for i in range(o0):
        at = 3 + i * (row // 32 + 5)
        expect[at:at + row // 32] = want_scales.reshape(o0, -1)[i]
    np.testing.assert_array_equal(host(scales), expect)


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,t0,t1,pitch,row_offset", [
    (8, 1, 16, 128, 8, 0), (64, 128, 16, 128, 64, 0), (200, 300, 16, 128, 200, 0), (136, 129, 1, 32, 144, 0),
    (512, 257, 7, 96, 520, 8), (72, 1000, 16, 64, 80, 0), (1032, 40, 32, 128, 1032, 0)])
def test_pack_transposed(gpu_lib, type, format, rows, cols, t0, t1, pitch, row_offset):
    # Columns of whole 16 bytes, as many as a workgroup takes, fewer and more; specials among the values.
    rng = np.random.default_rng(rows + cols)
    flat = ref.to_type(rng.standard_normal(row_offset + (cols - 1) * pitch + rows) * 2.0 ** rng.integers(-9, 9), type)
    flat[rng.integers(0, flat.size, 2)] = [np.nan, -np.inf]
    x = flat[row_offset + np.arange(rows)[:, None] + np.arange(cols)[None] * pitch]
    src = on_device(ref.raw(flat, type))
    n = ref.up(rows, t0) * ref.up(cols, t1)
    codes, scales = guarded(n * ref.BITS[format] // 8), guarded(n // 32)
    p = ref.pack_params(src.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), t0, t1, type, format, (1, pitch))
    p.in_offset = row_offset
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == b"mx_pack_transposed"
    want = wanted(x, format, t0, t1)
    np.testing.assert_array_equal(host(scales)[:-64], want[1])
    np.testing.assert_array_equal(host(codes)[:-64], want[0])
    assert (host(codes)[-64:] == GUARD).all() and (host(scales)[-64:] == GUARD).all()


def test_pack_without_input_is_all_padding(gpu_lib):
    codes, scales = guarded(2 * 64 // 2), guarded(2 * 2)
    src = torch.zeros(1, device="cuda")
    p = ref.pack_params(src.data_ptr(), 0, 0, codes.data_ptr(), scales.data_ptr(), 2, 64, "f32", "e2m1")
    p.out_size0 = p.out_size1 = 1
    p.out_stride0, p.scales_stride0 = 128, 4
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    assert (host(codes)[:64] == 0).all() and (host(scales)[:4] == 0).all()
    assert (host(codes)[64:] == GUARD).all() and (host(scales)[4:] == GUARD).all()


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_unpack_every_code_with_every_scale(gpu_lib, format, type):
    count = 16 if format == "e2m1" else 256
    codes = np.tile(np.arange(count, dtype=np.uint8), 256 * 32 // min(count, 32) if count < 32 else 256)
    codes = codes.reshape(256, -1)
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], codes.shape[1] // 32, 1)
    rows, cols = codes.shape
    out = torch.zeros(rows * cols * (4 if type == "f32" else 2), dtype=torch.uint8, device="cuda")
    d_codes, d_scales = on_device(ref.to_bytes(codes, format)), on_device(scales)
    p = ref.unpack_params(d_codes.data_ptr(), d_scales.data_ptr(), out.data_ptr(), rows, cols, 1, cols, format, type)
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    with np.errstate(over="ignore"):
        f32 = ref.widen(codes, scales, format).astype(np.float32)  # (4 significant bits: exact, or beyond the range)
    want = ref.to_type(f32, type)
    got = ref.from_raw(host(out).view(np.float32 if type == "f32" else np.uint16), type).reshape(rows, cols)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    np.testing.assert_array_equal(got[fine], want[fine])
    np.testing.assert_array_equal(np.signbit(got[fine]), np.signbit(want[fine]))


@pytest.mark.parametrize("format,type", [("e2m1", "bf16"), ("e2m1", "f32"), ("e4m3", "f16")])
@pytest.mark.parametrize("rows,cols,t0,t1,strides", [
    (1, 1, 1, 32, None), (3, 33, 16, 128, None), (17, 301, 16, 128, (310, 1)), (33, 70, 7, 96, (1, 40)),
    (5, 40, 1, 64, (200, 3)), (700, 4095, 16, 128, None), (130, 8200, 1, 8224, None)])
def test_unpack(gpu_lib, format, type, rows, cols, t0, t1, strides):
    rng = np.random.default_rng(rows)
    codes, scales = ref.random_codes(rng, ref.up(rows, t0), ref.up(cols, t1), format)
    s0, s1 = strides or (cols, 1)
    size = (rows - 1) * s0 + (cols - 1) * s1 + 1
    dtype = np.float32 if type == "f32" else np.uint16
    before = np.arange(size + 16).astype(dtype)
    out = on_device(before)
    d_codes = on_device(ref.to_bytes(ref.tiled(codes, t0, t1), format))
    d_scales = on_device(ref.tiled(scales, t0, t1 // 32))
    p = ref.unpack_params(d_codes.data_ptr(), d_scales.data_ptr(), out.data_ptr(), rows, cols, t0, t1, format, type, strides)
    if strides == (1, 40):  # (rows next to each other, so columns have to be: the call writes rows one after the other)
        with_failures(gpu_lib, p)
        return
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    want = before.copy()
    values = ref.raw(ref.to_type(ref.widen(codes, scales, format)[:rows, :cols].astype(np.float32), type), type)
    want[(np.arange(rows)[:, None] * s0 + np.arange(cols)[None] * s1).reshape(-1)] = values.reshape(-1)
    np.testing.assert_array_equal(host(out).view(dtype), want)


def with_failures(lib, p):
    from test_abi import Failures
    with Failures() as f:
        lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    assert len(f.seen) == 1 and "rows_apart" in f.seen[0]


def test_host_operands(gpu_lib):
    # In the library's default mode operands may be host memory: staged, computed, the touched rows copied back.
    rng = np.random.default_rng(5)
    rows, cols, t0, t1 = 37, 300, 16, 128
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    n = ref.up(rows, t0) * ref.up(cols, t1)
    codes, scales, out = np.zeros(n // 2, np.uint8), np.zeros(n // 32, np.uint8), np.full((rows, 310), 7, np.float32)
    p = ref.pack_params(x.ctypes.data, rows, cols, codes.ctypes.data, scales.ctypes.data, t0, t1, "f32", "e2m1")
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    want = wanted(x, "e2m1", t0, t1)
    np.testing.assert_array_equal(codes, want[0])
    np.testing.assert_array_equal(scales, want[1])
    p = ref.unpack_params(codes.ctypes.data, scales.ctypes.data, out.ctypes.data, rows, cols, t0, t1, "e2m1", "f32", (310, 1))
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    c, s = ref.quantise(ref.padded(x, t0, t1), "e2m1")
    np.testing.assert_array_equal(out[:, :cols], ref.widen(c, s, "e2m1")[:rows, :cols].astype(np.float32))
    assert (out[:, cols:] == 7).all()


def test_offsets_beyond_32_bits(gpu_lib):
    # 4.6 GiB of f16, the last rows of which lie past 2^32 bytes and 2^31 elements.
    rows, cols = 73728, 32768
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    x[:64] = torch.randn(64, cols, generator=gen, device="cuda").half()
    x[64:-64] = 1.0
    x[-64:] = torch.randn(64, cols, generator=gen, device="cuda").half()
    codes = torch.zeros(rows * cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows * cols // 32, dtype=torch.uint8, device="cuda")
    p = ref.pack_params(x.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), 16, 128, "f16", "e2m1")
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    for part in (slice(0, 64), slice(rows - 64, rows)):
        want = wanted(x[part].float().cpu().numpy(), "e2m1", 16, 128)
        np.testing.assert_array_equal(host(codes.view(rows, -1)[part]).reshape(-1), want[0])
        np.testing.assert_array_equal(host(scales.view(rows, -1)[part]).reshape(-1), want[1])
    back = torch.zeros_like(x)
    p = ref.unpack_params(codes.data_ptr(), scales.data_ptr(), back.data_ptr(), rows, cols, 16, 128, "e2m1", "f16")
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    assert bool((back[64:-64] == 1.0).all())
    c, s = ref.quantise(x[-64:].float().cpu().numpy(), "e2m1")
    np.testing.assert_array_equal(back[-64:].float().cpu().numpy(), ref.widen(c, s, "e2m1").astype(np.float32))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("type,format,rows", [("f32", "e2m1", 8192), ("bf16", "e4m3", 16384)])
def test_matrices_that_no_cache_holds(gpu_lib, type, format, rows, transposed):
    # 210 MB, which are read and written past the caches: one block of 512 x 640 over and over.
    cols = 6400
    rng = np.random.default_rng(rows)
    block = ref.to_type(rng.standard_normal((512, 640)) * np.exp2(rng.integers(-4, 5, (512, 1))), type)
    dtype = torch.float32 if type == "f32" else torch.bfloat16
    x = torch.from_numpy(block.astype(np.float32)).to(dtype).cuda().repeat(rows // 512, cols // 640)
    given = x.t().contiguous() if transposed else x
    codes = torch.zeros(rows * cols * ref.BITS[format] // 8, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows * cols // 32, dtype=torch.uint8, device="cuda")
    p = ref.pack_params(given.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), 16, 128, type, format)
    p.in_stride0, p.in_stride1 = (1, rows) if transposed else (cols, 1)
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == (b"mx_pack_transposed" if transposed else b"mx_pack_rows")
    want_codes, want_scales = wanted(block, format, 16, 128)
    for got, want in ((codes, want_codes), (scales, want_scales)):
        want = on_device(want).view(1, 32, 1, 5, -1)   # [.][panels of 16 rows][.][tiles of 128 columns][a tile]
        assert bool((got.view(rows // 512, 32, cols // 640, 5, -1) == want).all())
    back = torch.zeros_like(x)
    p = ref.unpack_params(codes.data_ptr(), scales.data_ptr(), back.data_ptr(), rows, cols, 16, 128, format, type)
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    values = torch.from_numpy(ref.widen(*ref.quantise(block, format), format).astype(np.float32)).cuda().to(dtype)
    assert bool((back.view(rows // 512, 512, cols // 640, 640) == values.view(1, 512, 1, 640)).all())

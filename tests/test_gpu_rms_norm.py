"""The root-mean-square norm on the GPU. The sum of squares is in 64 bits on both sides and
rounded to f32 once, everything behind it is elementwise with the same roundings: codes, scales
and sums agree bit for bit, unless r lies within 1e-15 of a border of f32 (one row in 10^8).
"""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_pack import GUARD, guarded, host, on_device

pytestmark = pytest.mark.gpu


def want_of(y, format, out_cols):
    y = np.pad(y, ((0, 0), (0, out_cols - y.shape[1])))
    if format == "s8":
        return ref.quantise_s8(y)
    codes, scales = ref.quantise(y, format)
    return ref.to_bytes(codes, format), scales


def run(lib, x, residual, weight, type, format, out_cols, epsilon=1e-5, weight_f32=False, in_place=None):
    rows, cols = x.shape
    d_x = on_device(ref.raw(x, type))
    d_r = on_device(ref.raw(residual, type)) if residual is not None else None
    d_w = on_device(ref.raw(weight, "f32" if weight_f32 else type)) if weight is not None else None
    total = {None: guarded(d_x.numel()), "in": d_x, "residual": d_r}[in_place] if residual is not None else None
    codes = guarded(rows * out_cols * (4 if format == "e2m1" else 8) // 8)
    scales = guarded(rows * 4 if format == "s8" else rows * out_cols // 32)
    p = ref.norm_params(d_x.data_ptr(), d_r.data_ptr() if d_r is not None else None,
                        total.data_ptr() if total is not None else None, d_w.data_ptr() if d_w is not None else None,
                        codes.data_ptr(), scales.data_ptr(), rows, cols, out_cols, type, format, epsilon)
    if weight_f32:
        p.flags |= ref.abi.RMS_NORM_WEIGHT_F32
    lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
    codes, scales = host(codes), host(scales)
    assert (codes[-64:] == GUARD).all() and (scales[-64:] == GUARD).all()
    codes = codes[:-64].view(np.int8 if format == "s8" else np.uint8).reshape(rows, -1)
    scales = scales[:-64].view(np.float32) if format == "s8" else scales[:-64].reshape(rows, -1)
    got_sum = None
    if total is not None:
        raw = host(total)
        if in_place is None:
            assert (raw[-64:] == GUARD).all()
            raw = raw[:-64]
        got_sum = raw.view(np.float32 if type == "f32" else np.uint16).reshape(rows, cols)
    return got_sum, codes, scales


def check(lib, x, residual, weight, type, format, out_cols, **kw):
    total, codes, scales = run(lib, x, residual, weight, type, format, out_cols, **kw)
    s, y = ref.norm(x, residual, weight, kw.get("epsilon", 1e-5), type)
    want_codes, want_scales = want_of(y, format, out_cols)
    if residual is not None:
        np.testing.assert_array_equal(ref.from_raw(total, type), s)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)


def inputs(rng, rows, cols, type, residual=True):
    x = ref.to_type(rng.standard_normal((rows, cols)) * np.where(rng.random(cols) < 0.03, 8, 1), type)
    r = ref.to_type(rng.standard_normal((rows, cols)), type) if residual else None
    return x, r, ref.to_type(1 + 0.1 * rng.standard_normal(cols), type)


# Each of the kernel's row lengths, one value and one short of a block or of a lane's eight among them.
COLS = [1, 31, 32, 100, 512, 513, 1000, 2048, 2049, 4095, 4096, 5000, 8192, 8200, 16384, 16392, 32768, 32769, 70001]


@pytest.mark.parametrize("format", ["s8", "e4m3", "e2m1"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", COLS)
def test_norm(gpu_lib, type, format, cols):
    rng = np.random.default_rng(cols)
    rows = 5
    x, r, w = inputs(rng, rows, cols, type)
    check(gpu_lib, x, r, w, type, format, cols if format == "s8" else ref.up(cols, 32))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == (b"rms_norm_row" if cols <= 32768 else b"rms_norm_long")


@pytest.mark.parametrize("format", ["s8", "e4m3", "e2m1"])
@pytest.mark.parametrize("rows,cols,out_cols", [(1, 8192, 8192), (300, 8192, 8192), (1, 4096, 4096), (777, 4095, 4096),
                                                (1029, 640, 640), (3, 33, 128), (2, 40000, 40064), (4, 0, 64)])
def test_rows_and_padding(gpu_lib, format, rows, cols, out_cols):
    rng = np.random.default_rng(rows)
    x, _, w = inputs(rng, rows, cols, "bf16", residual=False)
    if cols == 0:
        _, codes, scales = run(gpu_lib, x, None, w, "bf16", format, out_cols)
        assert (codes == 0).all() and (scales == (2.0 ** -126 if format == "s8" else 0)).all()
        return
    check(gpu_lib, x, None, w, "bf16", format, out_cols)


@pytest.mark.parametrize("in_place", ["in", "residual"])
@pytest.mark.parametrize("cols", [100, 4096, 40000])
@pytest.mark.parametrize("format", ["s8", "e4m3"])
def test_sum_in_place(gpu_lib, cols, format, in_place):
    rng = np.random.default_rng(cols)
    x, r, w = inputs(rng, 7, cols, "bf16")
    check(gpu_lib, x, r, w, "bf16", format, ref.up(cols, 32), in_place=in_place)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_weight_of_f32_and_no_weight(gpu_lib, type):
    rng = np.random.default_rng(9)
    x, r, _ = inputs(rng, 6, 1000, type)
    w = (1 + 0.1 * rng.standard_normal(1000)).astype(np.float32)
    check(gpu_lib, x, r, w, type, "e4m3", 1024, weight_f32=True)
    check(gpu_lib, x, r, None, type, "s8", 1000)


@pytest.mark.parametrize("format", ["s8", "e4m3", "e2m1"])
def test_values_that_are_not_finite_and_rows_of_zeros(gpu_lib, format):
    rng = np.random.default_rng(2)
    x, _, w = inputs(rng, 10, 500, "f32", residual=False)
    x[0] = 0
    x[1, 3] = np.nan
    x[2, 499] = np.inf
    x[3, 7] = -np.inf
    x[4] = 1e30                # squares beyond f32
    x[5] = 1e-30
    x[6] = 2.0 ** -149
    x[7] = 0
    x[7, 100] = 3e38
    x[8] = -0.0
    for epsilon in (1e-5, 0.0, 1e-30):
        check(gpu_lib, x, None, w, "f32", format, 512, epsilon=epsilon)
    w[17], w[40] = np.inf, 0
    check(gpu_lib, x, None, w, "f32", format, 512)


def test_strides_and_offsets(gpu_lib):
    # Rows inside wider matrices, codes and scales too; what lies between them stays.
    rng = np.random.default_rng(4)
    rows, cols, out_cols = 9, 333, 352
    x, r, w = inputs(rng, rows, cols, "f16")

    def wide(m, pitch, first):
        buf = np.full(first + rows * pitch, 1.5, np.float16)
        buf[first:].reshape(rows, pitch)[:, :cols] = m.astype(np.float16)
        return on_device(buf)

    d_x, d_r, d_s = wide(x, 350, 3), wide(r, 401, 1), wide(np.zeros_like(x), 339, 5)
    d_w = on_device(np.concatenate([[0, 0], w]).astype(np.float16))
    codes, scales = guarded(20 + rows * 400), guarded(2 + rows * 13)
    p = ref.norm_params(d_x.data_ptr(), d_r.data_ptr(), d_s.data_ptr(), d_w.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                        rows, cols, out_cols, "f16", "e4m3")
    p.in_offset, p.in_stride0 = 3, 350
    p.residual_offset, p.residual_stride0 = 1, 401
    p.sum_offset, p.sum_stride0 = 5, 339
    p.weight_offset = 2
    p.out_offset, p.out_stride0 = 20, 400
    p.scales_offset, p.scales_stride0 = 2, 13
    gpu_lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
    s, y = ref.norm(x, r, w, 1e-5, "f16")
    want_codes, want_scales = want_of(y, "e4m3", out_cols)
    expect = np.full(5 + rows * 339, 1.5, np.float16)
    expect[5:].reshape(rows, 339)[:, :cols] = s
    np.testing.assert_array_equal(host(d_s).view(np.float16), expect)
    expect = np.full(codes.numel(), GUARD, np.uint8)
    expect[20:20 + rows * 400].reshape(rows, 400)[:, :out_cols] = want_codes
    np.testing.assert_array_equal(host(codes), expect)
    expect = np.full(scales.numel(), GUARD, np.uint8)
    expect[2:2 + rows * 13].reshape(rows, 13)[:, :out_cols // 32] = want_scales
    np.testing.assert_array_equal(host(scales), expect)


def test_host_operands(gpu_lib):
    rng = np.random.default_rng(6)
    rows, cols = 11, 700
    x, r, w = inputs(rng, rows, cols, "f32")
    total, codes, scales = r.copy(), np.zeros((rows, 704), np.int8), np.zeros(rows, np.float32)
    p = ref.norm_params(x.ctypes.data, total.ctypes.data, total.ctypes.data, w.ctypes.data, codes.ctypes.data,
                        scales.ctypes.data, rows, cols, 704, "f32", "s8")
    gpu_lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
    s, y = ref.norm(x, r, w, 1e-5, "f32")
    want = want_of(y, "s8", 704)
    np.testing.assert_array_equal(total, s)
    np.testing.assert_array_equal(codes, want[0])
    np.testing.assert_array_equal(scales, want[1])


def test_a_row_does_not_depend_on_its_company(gpu_lib):
    # The same row alone and among 400 takes kernels with other numbers of lanes: the same codes.
    rng = np.random.default_rng(8)
    x, r, w = inputs(rng, 400, 8000, "bf16")
    many = run(gpu_lib, x, r, w, "bf16", "e2m1", 8000)
    for i in (0, 399):
        one = run(gpu_lib, x[i:i + 1], r[i:i + 1], w, "bf16", "e2m1", 8000)
        for a, b in zip(many, one):
            np.testing.assert_array_equal(a[i:i + 1], b)


@pytest.mark.parametrize("format", ["s8", "e4m3"])
def test_rows_beyond_32_bits(gpu_lib, format):
    # 4.5 GiB of bf16, sums in place of the residual: the last rows as a call of their own has them.
    rows, cols, few = 73728, 32768, 16
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    total = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    for t in (x, total):
        t[-few:] = torch.randn(few, cols, generator=gen, device="cuda").bfloat16()
    weight = torch.randn(cols, generator=gen, device="cuda").bfloat16()

    def call(x, total):
        n = x.shape[0]
        codes = torch.zeros(n, cols, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(n, 4 if format == "s8" else cols // 32, dtype=torch.uint8, device="cuda")
        p = ref.norm_params(x.data_ptr(), total.data_ptr(), total.data_ptr(), weight.data_ptr(), codes.data_ptr(),
                            scales.data_ptr(), n, cols, cols, "bf16", format)
        gpu_lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
        return total, codes, scales

    alone = call(x[-few:].clone(), total[-few:].clone())
    first = call(x[:1].clone(), total[:1].clone())
    everything = call(x, total)
    for all_rows, last, one in zip(everything, alone, first):
        assert torch.equal(all_rows[-few:], last)
        assert bool((all_rows[:-few] == one).all())


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("cols,pitch", [(4092, 4096), (4096, 4096), (4096, 4100)])
def test_sums_that_go_past_the_caches(gpu_lib, type, cols, pitch):
    # 28 MB in rows of whole or broken eights, aligned or not: the sum is torch's, codes are those of a few rows by themselves.
    rows, few, out_cols = 3400, 20, 4096
    dtype = torch.float16 if type == "f16" else torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, residual = (torch.randn(rows, pitch, generator=gen, device="cuda").to(dtype) for _ in range(2))

    def call(first, n):
        total = torch.full((n, pitch), 7.0, dtype=dtype, device="cuda")
        codes = torch.zeros(n, out_cols, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(n, out_cols // 32, dtype=torch.uint8, device="cuda")
        p = ref.norm_params(x[first].data_ptr(), residual[first].data_ptr(), total.data_ptr(), None, codes.data_ptr(),
                            scales.data_ptr(), n, cols, out_cols, type, "e4m3")
        p.in_stride0 = p.residual_stride0 = p.sum_stride0 = pitch
        gpu_lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
        return total, codes, scales

    total, codes, scales = call(0, rows)
    want = (x.float() + residual.float()).to(dtype)
    want[:, cols:] = 7.0
    assert torch.equal(total, want)
    for first in (0, rows - few):
        alone = call(first, few)
        assert torch.equal(codes[first:first + few], alone[1]) and torch.equal(scales[first:first + few], alone[2])

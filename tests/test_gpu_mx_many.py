"""The microscaled operators on more values than 32 bits number, and than a grid has lanes for, on the GPU: kernels that go round
again, with indices of 64 bits. Inputs overlap or coincide, which operands that are only read may."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_mmt4d import exact_codes
from test_gpu_mx_pack import on_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type,rows", [("f32", 8200), ("bf16", 16400)])
def test_unpack(gpu_lib, type, rows):  # noqa: F811
    # Tiles of one row of 2^20 values, each row 64 values behind the last; 40 columns of them.
    cols, tile = 40, 1 << 20
    rng = np.random.default_rng(1)
    codes, scales = ref.random_codes(rng, 1, 64 * rows + tile, "e2m1")
    d_codes, d_scales = on_device(ref.to_bytes(codes, "e2m1")), on_device(scales)
    out = torch.full((rows, 42), 7.0, dtype=torch.float32 if type == "f32" else torch.bfloat16, device="cuda")
    p = ref.unpack_params(d_codes.data_ptr(), d_scales.data_ptr(), out.data_ptr(), rows, cols, 1, tile, "e2m1", type, (42, 1), 64, 2)
    assert rows * (tile // 8) * (2 if type == "f32" else 1) > 1 << 31
    gpu_lib.iree_uk_mi355x_mx_unpack_p(C.byref(p))
    want = ref.to_type(ref.widen(codes, scales, "e2m1")[0, :64 * rows].reshape(rows, 64)[:, :cols], type)
    np.testing.assert_array_equal(out[:, :cols].float().cpu().numpy(), want)
    assert bool((out[:, cols:] == 7).all())


def test_pack(gpu_lib):  # noqa: F811
    # 33000 times the same row of 2^20 values: 17 GB of codes.
    rows, cols = 33000, 1 << 20
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, cols)).astype(np.float32)
    d_x = on_device(x)
    codes = torch.zeros(rows, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, cols // 32, dtype=torch.uint8, device="cuda")
    p = ref.pack_params(d_x.data_ptr(), rows, cols, codes.data_ptr(), scales.data_ptr(), 1, cols, "f32", "e2m1", (0, 1))
    gpu_lib.iree_uk_mi355x_mx_pack_p(C.byref(p))
    want = ref.quantise(x, "e2m1")
    for got, row in ((codes, ref.to_bytes(want[0], "e2m1")), (scales, want[1])):
        row = on_device(row)
        for first in range(0, rows, 3000):
            assert bool((got[first:first + 3000] == row).all())


def test_general_product(gpu_lib):  # noqa: F811
    # 33000 x 33000 results of K = 32: more than one for each thread.
    n = 33000
    rng = np.random.default_rng(3)
    lhs, rhs = exact_codes(rng, n, 32, "e4m3"), exact_codes(rng, n, 32, "e2m1")
    d = [on_device(lhs[0]), on_device(lhs[1]), on_device(ref.to_bytes(rhs[0], "e2m1")), on_device(rhs[1])]
    out = torch.zeros(n, n, device="cuda")
    p = ref.mmt4d_params(*(x.data_ptr() for x in d), out.data_ptr(), (n, n, 1), (1, 1, 32), "e4m3", "f32")
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == b"mx_mmt4d_generic"
    a = torch.from_numpy(ref.widen(*lhs, "e4m3").astype(np.float32)).cuda()
    b = torch.from_numpy(ref.widen(*rhs, "e2m1").astype(np.float32)).cuda()
    for first in range(0, n, 3000):  # (32 exact products: any order gives the same)
        assert torch.equal(out[first:first + 3000], a[first:first + 3000] @ b.t())

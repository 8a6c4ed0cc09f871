"""Every kernel of the products of microscaled operands on the GPU, with one chunk of K and with many: exact sums (see
test_gpu_mx_mmt4d.py), from the kernel that is meant."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_reference as ref
from test_gpu_configs import gpu_lib  # noqa: F401
from test_gpu_mx_mmt4d import check_exact, exact_codes, in_64_bits
from test_gpu_mx_pack import on_device
from test_mx_mmt4d_choice_on_host import KERNELS, RESIDENT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,kernel", KERNELS)
def test_exact_sums(gpu_lib, lhs, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    used = check_exact(gpu_lib, np.random.default_rng(rows + cols), rows, cols, k, (m0, n0, 128), lhs, out)
    assert used.decode() == "mx_mmt4d_" + kernel


@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0,kernel", [q for q in KERNELS if q[4] > 128 and q[2] * q[3] < 1 << 20])
def test_accumulate(gpu_lib, lhs, out, rows, cols, k, m0, n0, kernel):  # noqa: F811
    check_exact(gpu_lib, np.random.default_rng(rows + cols), rows, cols, k, (m0, n0, 128), lhs, out, accumulate=True)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("lhs,out,rows,cols,k,m0,n0", RESIDENT)
def test_a_rhs_that_no_cache_holds(gpu_lib, lhs, out, rows, cols, k, m0, n0, accumulate):  # noqa: F811
    # 160 rows of the rhs over and over, the last ones of them only in part.
    rng = np.random.default_rng(rows + cols)
    a, b = exact_codes(rng, rows, k, lhs), exact_codes(rng, 160, k, "e2m1")
    times = -(-cols // 160)
    d_a, d_as = on_device(ref.to_bytes(ref.tiled(a[0], m0, 128), lhs)), on_device(ref.tiled(a[1], m0, 4))
    d_b = on_device(ref.to_bytes(ref.tiled(b[0], n0, 128), "e2m1")).view(-1).repeat(times)
    d_bs = on_device(ref.tiled(b[1], n0, 4)).view(-1).repeat(times)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[out]
    result = torch.full((rows // m0, cols // n0, m0, n0), 3.0, dtype=dtype, device="cuda")
    p = ref.mmt4d_params(d_a.data_ptr(), d_as.data_ptr(), d_b.data_ptr(), d_bs.data_ptr(), result.data_ptr(),
                         (rows // m0, cols // n0, k // 128), (m0, n0, 128), lhs, out, accumulate)
    gpu_lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(p))
    assert gpu_lib.iree_uk_mi355x_last_kernel() == b"mx_mmt4d_resident"
    want = in_64_bits(a, b, lhs) + (3 if accumulate else 0)
    want = torch.from_numpy(ref.to_type(want.astype(np.float32), out).astype(np.float32)).to(dtype).cuda().repeat(1, times)[:, :cols]
    got = result.permute(0, 2, 1, 3).reshape(rows, cols)
    assert torch.equal(got, want)

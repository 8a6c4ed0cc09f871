"""The microscaled operators and the norm together, as a program uses them: weights quantised once, rows
normed into codes that the product reads as they are; the 8-bit form in front of the int8 product; a
captured step replayed; two threads on streams of their own.
"""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import mx_reference as ref
from iree_amd import abi
from test_gpu_configs import gpu_lib, mm_params  # noqa: F401
from test_gpu_mx_pack import host, on_device

pytestmark = pytest.mark.gpu


class Layer:
    """A residual, a norm and a projection: x, h [m][k] -> h + x, norm(h + x) @ weights^T."""

    def __init__(self, lib, seed, m, n, k, type, lhs_format, out_type):
        self.lib, self.m, self.n, self.k, self.type, self.lhs_format, self.out_type = lib, m, n, k, type, lhs_format, out_type
        rng = np.random.default_rng(seed)
        self.x = ref.to_type(rng.standard_normal((m, k)), type)
        self.h = ref.to_type(rng.standard_normal((m, k)), type)
        self.gain = ref.to_type(1 + 0.1 * rng.standard_normal(k), type)
        self.w = (rng.standard_normal((k, n)) * 0.05).astype(np.float32)
        self.kp, self.np = ref.up(k, 128), ref.up(n, 16)
        self.d_w = on_device(self.w)
        self.rhs = torch.zeros(self.np * self.kp // 2, dtype=torch.uint8, device="cuda")
        self.rhs_scales = torch.zeros(self.np * self.kp // 32, dtype=torch.uint8, device="cuda")
        self.d_x, self.d_h, self.d_gain = (on_device(ref.raw(v, type)) for v in (self.x, self.h, self.gain))
        self.total = torch.zeros_like(self.d_x)
        self.lhs = torch.zeros(m * self.kp * ref.BITS[lhs_format] // 8, dtype=torch.uint8, device="cuda")
        self.lhs_scales = torch.zeros(m * self.kp // 32, dtype=torch.uint8, device="cuda")
        self.out = torch.zeros(m * self.np * (4 if out_type == "f32" else 2), dtype=torch.uint8, device="cuda")
        # [k][n] read as [n][k].
        self.pack = ref.pack_params(self.d_w.data_ptr(), n, k, self.rhs.data_ptr(), self.rhs_scales.data_ptr(), 16, 128, "f32",
                                    "e2m1", (1, n))
        self.norm = ref.norm_params(self.d_x.data_ptr(), self.d_h.data_ptr(), self.total.data_ptr(), self.d_gain.data_ptr(),
                                    self.lhs.data_ptr(), self.lhs_scales.data_ptr(), m, k, self.kp, type, lhs_format)
        self.product = ref.mmt4d_params(self.lhs.data_ptr(), self.lhs_scales.data_ptr(), self.rhs.data_ptr(),
                                        self.rhs_scales.data_ptr(), self.out.data_ptr(), (m, self.np // 16, self.kp // 128),
                                        (1, 16, 128), lhs_format, out_type)

    def load(self):
        self.lib.iree_uk_mi355x_mx_pack_p(C.byref(self.pack))

    def step(self):
        self.lib.iree_uk_mi355x_rms_norm_p(C.byref(self.norm))
        self.lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(self.product))

    def check(self):
        s, y = ref.norm(self.x, self.h, self.gain, 1e-5, self.type)
        raw = np.float32 if self.type == "f32" else np.uint16
        np.testing.assert_array_equal(ref.from_raw(host(self.total).view(raw), self.type).reshape(self.m, self.k), s)
        lhs = ref.widen(*ref.quantise(ref.padded(y, 1, 128), self.lhs_format), self.lhs_format)
        rhs = ref.widen(*ref.quantise(ref.padded(self.w.T, 16, 128), "e2m1"), "e2m1")
        want = lhs @ rhs.T
        got = ref.from_raw(host(self.out).view(np.float32 if self.out_type == "f32" else np.uint16), self.out_type)
        got = got.reshape(self.m, self.np).astype(np.float64)
        # The summation (at most K additions, each off by a unit in the last place of a partial sum; 16-bit results of 8-bit
        # codes: of eight products, seven lose what lies 13 bits below the largest one's exponent) and half a step of the
        # result's type.
        loss = 7 * 2.0 ** -13 if self.lhs_format == "e4m3" and self.out_type != "f32" else 0
        bound = (self.kp * 2.0 ** -23 + loss) * (np.abs(lhs) @ np.abs(rhs).T)
        bound += {"f32": 0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[self.out_type] * (np.abs(want) + bound) + 2.0 ** -25
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("m,n,k,type,lhs_format,out_type", [
    (1, 1000, 2048, "bf16", "e4m3", "bf16"), (13, 300, 777, "f16", "e2m1", "f16"), (77, 4100, 4095, "bf16", "e4m3", "f16"),
    (300, 520, 1000, "f32", "e2m1", "f32")])
def test_layer(gpu_lib, m, n, k, type, lhs_format, out_type):
    layer = Layer(gpu_lib, m, m, n, k, type, lhs_format, out_type)
    layer.load()
    layer.step()
    layer.check()


def test_norm_in_front_of_the_int8_product(gpu_lib):
    # Codes row by row are the lhs of iree_uk_mmt4d with tiles one row tall; K padded to whole tiles by out_size1.
    m, n, k, k0 = 21, 64, 1000, 64
    kp = ref.up(k, k0)
    rng = np.random.default_rng(1)
    x = ref.to_type(rng.standard_normal((m, k)), "bf16")
    d_x = on_device(ref.raw(x, "bf16"))
    codes = torch.zeros(m, kp, dtype=torch.int8, device="cuda")
    scales = torch.zeros(m, device="cuda")
    p = ref.norm_params(d_x.data_ptr(), None, None, None, codes.data_ptr(), scales.data_ptr(), m, k, kp, "bf16", "s8")
    gpu_lib.iree_uk_mi355x_rms_norm_p(C.byref(p))
    w = rng.integers(-128, 128, (n, kp)).astype(np.int8)
    d_w = on_device(ref.tiled(w, 16, k0))
    out = torch.zeros(m, n, dtype=torch.int32, device="cuda")
    q = mm_params(codes.data_ptr(), d_w.data_ptr(), out.data_ptr(), m, n // 16, kp // k0, 1, 16, k0, abi.MMT4D_TYPE_S8S8S32)
    gpu_lib.iree_uk_mmt4d_p(C.byref(q))
    _, y = ref.norm(x, None, None, 1e-5, "bf16")
    want, scale = ref.quantise_s8(np.pad(y, ((0, 0), (0, kp - k))))
    np.testing.assert_array_equal(host(out), want.astype(np.int64) @ w.astype(np.int64).T)
    np.testing.assert_array_equal(host(scales), scale)


@pytest.mark.parametrize("m", [1, 16, 77, 300])
def test_a_captured_step_is_replayed(gpu_lib, m):
    # Every replay against the reference, with eager work and synchronisation between them; two graphs of two layers.
    layers = [Layer(gpu_lib, 10 + i, m, 520, 1000, "bf16", "e4m3", "f32") for i in range(2)]
    for layer in layers:
        layer.load()
        layer.step()  # (kernels are loaded before the capture)
    graphs, stream = [], torch.cuda.Stream()
    try:
        torch.cuda.synchronize()
        for layer in layers:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                gpu_lib.iree_uk_mi355x_set_stream(torch.cuda.current_stream().cuda_stream, 1)
                layer.step()
            graphs.append(graph)
        for i in range(3):
            for layer in layers:
                layer.out.fill_(255)
                layer.lhs.fill_(i)
                layer.lhs_scales.fill_(255)
            torch.cuda.synchronize()
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for layer in layers:
                layer.check()
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)


def test_two_threads_on_streams_of_their_own(gpu_lib):
    layers = [Layer(gpu_lib, 20 + i, 40 + i, 300, 900, "bf16", "e4m3", "bf16") for i in range(2)]
    torch.cuda.synchronize()

    def work(layer):
        stream = torch.cuda.Stream()
        gpu_lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
        layer.load()
        for _ in range(20):
            layer.step()
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(layer,)) for layer in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for layer in layers:
        layer.check()


@pytest.mark.parametrize("entry", ["pack", "norm", "product"])
def test_host_memory_is_refused_in_asynchronous_mode(gpu_lib, entry):
    from test_abi import Failures
    layer = Layer(gpu_lib, 1, 4, 32, 128, "f32", "e4m3", "f32")
    some = np.zeros(1 << 16, np.uint8)
    p, call = {"pack": (layer.pack, gpu_lib.iree_uk_mi355x_mx_pack_p), "norm": (layer.norm, gpu_lib.iree_uk_mi355x_rms_norm_p),
               "product": (layer.product, gpu_lib.iree_uk_mi355x_mx_mmt4d_p)}[entry]
    p.out_buffer = some.ctypes.data
    gpu_lib.iree_uk_mi355x_set_stream(None, 1)
    try:
        with Failures() as f:
            call(C.byref(p))
        assert len(f.seen) == 1 and "asynchronous mode" in f.seen[0]
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)

"""Feed-forward operators on several streams at once, and captured calls whose buffers change between replays."""
import ctypes as C

import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu
TILE = (1, 16, 16)


class Adapters:
    def __init__(self, lib, seed, m, n, k, rank, count):
        rng = np.random.default_rng(seed)
        self.lib, self.m, self.p = lib, m, abi.AdapterMmt4dParams()
        ref.tiles_into(self.p, m, n, k, TILE)
        self.p.rank, self.p.count, self.p.flags = rank, count, abi.ADAPTER_MMT4D_TYPE_BF16BF16F32
        self.lhs, self.out = ref.matrix(values(rng, m, k, "bf16"), 1, 16, "bf16"), ref.empty(m, n, 1, "f32")
        self.down = ref.Buffer(count, rank * k, "bf16", data=values(rng, count * rank, k, "bf16", 0.1))
        self.up = ref.Buffer(count, n * rank, "bf16", data=values(rng, count * n, rank, "bf16", 0.1))
        for name, cols in (("lhs", 0), ("out", 0), ("down", k), ("up", rank)):
            getattr(self, name).into(self.p, name)
            if cols:
                setattr(self.p, name + "_stride1", cols)
        self.index = torch.from_numpy(rng.integers(-1, count, m).astype(np.int32)).cuda()
        self.p.index_buffer = self.index.data_ptr()
        self.workspace = ref.workspace(lib, "adapter_mmt4d", self.p)

    def __call__(self):
        self.lib.iree_uk_mi355x_adapter_mmt4d_p(C.byref(self.p))

    def result(self):
        return ref.fetched(self.out, 1, 16)


class Backward:
    def __init__(self, lib, seed, m, n, k):
        rng = np.random.default_rng(seed)
        self.lib, self.p = lib, abi.GatedMmt4dBackwardParams()
        ref.tiles_into(self.p, m, n, k, TILE)
        self.p.flags = abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_SILU
        self.held = {"lhs": ref.matrix(values(rng, m, k, "bf16"), 1, 16, "bf16"), "lhs_grad": ref.empty(m, k, 1, "f32")}
        for name in ("gate", "up"):
            self.held[name] = ref.matrix(values(rng, n, k, "bf16", 0.1), 16, 16, "bf16")
            self.held[name + "_pre"] = ref.matrix(values(rng, m, n, "bf16"), 1, 16, "bf16")
            self.held[name + "_grad"] = ref.empty(n, k, 16, "f32")
        self.held["out_grad"] = ref.matrix(values(rng, m, n, "f32"), 1, 16, "f32")
        for name, buffer in self.held.items():
            buffer.into(self.p, name)
        self.workspace = ref.workspace(lib, "gated_mmt4d_backward", self.p)

    def __call__(self):
        self.lib.iree_uk_mi355x_gated_mmt4d_backward_p(C.byref(self.p))

    def result(self):
        return np.concatenate([ref.fetched(self.held[name], t0, 16) for name, t0 in (("lhs_grad", 1), ("gate_grad", 16), ("up_grad", 16))])


def on_stream(lib, stream, *calls):
    try:
        with torch.cuda.stream(stream):
            lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            for call in calls:
                call()
    finally:
        lib.iree_uk_mi355x_set_stream(None, 0)


def captured(lib, *calls):
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=stream):
            lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            for call in calls:
                call()
    finally:
        lib.iree_uk_mi355x_set_stream(None, 0)
    return graph


@pytest.mark.parametrize("m,rank,count", [(1, 16, 3), (50, 16, 7), (300, 64, 5), (2000, 64, 9)])
def test_a_captured_call_takes_the_adapters_that_rows_have_at_replay(gpu_lib, m, rank, count):  # noqa: F811
    a = Adapters(gpu_lib, m, m, 320, 2048, rank, count)
    graph = captured(gpu_lib, a)
    rng = np.random.default_rng(m + 1)
    for _ in range(4):
        a.index.copy_(torch.from_numpy(rng.integers(-1, count, m).astype(np.int32)))
        a()
        want = a.result()
        a.out.device[:-64].fill_(0x55)
        a.workspace[0][:a.workspace[1]].fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(a.result(), want)


# (few rows and a long K of lhs_grad, which is split)
@pytest.mark.parametrize("m,n,k", [(24, 2048, 256), (200, 4096, 128)])
def test_split_sums_replayed(gpu_lib, m, n, k):  # noqa: F811
    b = Backward(gpu_lib, m, m, n, k)
    b()
    want, other = b.result(), Backward(gpu_lib, m + 1, m, n, k)
    graph = captured(gpu_lib, b)
    for _ in range(3):
        b.held["lhs_grad"].device[:-64].fill_(0x55)
        b.workspace[0][:b.workspace[1]].fill_(0xFF)
        other()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(b.result(), want)


def test_calls_at_once(gpu_lib):  # noqa: F811
    calls = [Adapters(gpu_lib, 1, 64, 4096, 2048, 16, 20), Adapters(gpu_lib, 2, 500, 1024, 1024, 64, 5), Adapters(gpu_lib, 5, 2000, 1024, 1024, 64, 7), Backward(gpu_lib, 3, 100, 2048, 512),
             Backward(gpu_lib, 4, 700, 512, 512)]
    wants = []
    for call in calls:
        call()
        wants.append(call.result())
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for call, stream in zip(calls, streams):
            on_stream(gpu_lib, stream, call, call)
    torch.cuda.synchronize()
    for call, want in zip(calls, wants):
        np.testing.assert_array_equal(call.result(), want)

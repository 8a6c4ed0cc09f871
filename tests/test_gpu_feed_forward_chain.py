"""A serving step's feed-forward block as a program makes it: adapters beside gate and up, the gated product on top of
them, the product with the last weights, adapters beside that; eagerly and as a replayed graph."""
import ctypes as C

import numpy as np
import pytest
import torch

import feed_forward_reference as ref
from feed_forward_reference import check, values
from iree_amd import abi
from test_gpu_configs import gpu_lib  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (37, 640, 384), (300, 512, 256)])
def test_a_serving_step(gpu_lib, m, n, k, type):  # noqa: F811
    rng = np.random.default_rng(m)
    tile, rank, count = (1, 16, 16), 16, 5
    x = values(rng, m, k, type)
    gate, up_, last = (values(rng, r, c, type, 1 / np.sqrt(c)) for r, c in ((n, k), (n, k), (k, n)))
    index, scales = rng.integers(-1, count, m).astype(np.int32), (rng.random(count) + 0.5).astype(np.float32)
    pairs = {name: (values(rng, count * rank, c, type, 1 / np.sqrt(c)).reshape(count, rank, c),
                    values(rng, count * r, rank, type, 0.2).reshape(count, r, rank))
             for name, r, c in (("gate", n, k), ("up", n, k), ("last", k, n))}
    held = {"x": ref.matrix(x, 1, 16, type), "gate": ref.matrix(gate, 16, 16, type), "up": ref.matrix(up_, 16, 16, type),
            "last": ref.matrix(last, 16, 16, type), "gate_pre": ref.empty(m, n, 1, "f32"), "up_pre": ref.empty(m, n, 1, "f32"),
            "hidden": ref.empty(m, n, 1, type), "out": ref.empty(m, k, 1, type)}
    d_index, d_scales = torch.from_numpy(index).cuda(), torch.from_numpy(scales).cuda()
    keep, calls = [], []

    def adapter(name, lhs, out, out_type, rows, depth, accumulate):
        p = abi.AdapterMmt4dParams()
        ref.tiles_into(p, m, rows, depth, tile)
        p.rank, p.count = rank, count
        for part, v in zip(("down", "up"), pairs[name]):
            b = ref.Buffer(count, v[0].size, type, data=v)
            keep.append(b)
            b.into(p, part)
            setattr(p, part + "_stride1", v.shape[2])
        held[lhs].into(p, "lhs")
        held[out].into(p, "out")
        p.index_buffer, p.scales_buffer = d_index.data_ptr(), d_scales.data_ptr()
        p.flags = ref.type_flag("ADAPTER_MMT4D", type, out_type) | (abi.ADAPTER_MMT4D_ACCUMULATE if accumulate else 0)
        keep.append(ref.workspace(gpu_lib, "adapter_mmt4d", p))
        calls.append((gpu_lib.iree_uk_mi355x_adapter_mmt4d_p, p))

    adapter("gate", "x", "gate_pre", "f32", n, k, False)
    adapter("up", "x", "up_pre", "f32", n, k, False)
    p = abi.GatedMmt4dParams()
    ref.tiles_into(p, m, n, k, tile)
    for name, buffer in (("lhs", "x"), ("gate", "gate"), ("up", "up"), ("gate_pre", "gate_pre"), ("up_pre", "up_pre"), ("out", "hidden")):
        held[buffer].into(p, name)
    p.flags = ref.type_flag("GATED_MMT4D", type, type) | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_PRE_LOAD | abi.GATED_MMT4D_PRE_F32
    calls.append((gpu_lib.iree_uk_mi355x_gated_mmt4d_p, p))
    q = abi.Mmt4dParams()
    ref.tiles_into(q, m, k, n, tile)
    for name, buffer in (("lhs", "hidden"), ("rhs", "last"), ("out", "out")):
        held[buffer].into(q, name)
    q.flags = ref.type_flag("MMT4D", type, type) | abi.MMT4D_SKIP_INTERMEDIATE_ROUNDINGS
    calls.append((gpu_lib.iree_uk_mmt4d_p, q))
    adapter("last", "hidden", "out", type, k, n, True)

    g_part, g_off = ref.adapters(x, *pairs["gate"], index, scales)
    u_part, u_off = ref.adapters(x, *pairs["up"], index, scales)
    (h, g, u), (h_off, _, _) = ref.gated(x, gate, up_, "silu", (g_part, u_part))
    # (the adapters' parts are off by g_off and u_off, and rounded to f32)
    g_off, u_off = g_off + ref.U * np.abs(g_part), u_off + ref.U * np.abs(u_part)
    h_off = h_off + 1.13 * g_off * (np.abs(u) + u_off) + np.abs(ref.act(g, "silu")[0]) * u_off
    h_off = h_off + ref.rounded_off(np.abs(h) + h_off, type)
    y, y_off = h @ last.T, h_off @ np.abs(last).T + (n + 2) * ref.U * ((np.abs(h) + h_off) @ np.abs(last).T)
    y_off = y_off + ref.rounded_off(np.abs(y) + y_off, type)
    down, up_of = pairs["last"]
    part, part_off = ref.adapters(h, down, up_of, index, scales)
    for a in range(count):  # what the hidden values' own error does to the adapters' part
        rows = index == a
        part_off[rows] += np.abs(scales[a]) * (h_off[rows] @ np.abs(down[a]).T @ np.abs(up_of[a]).T) * (1 + 2.0 ** -10)
    want, off = y + part, y_off + part_off + ref.U * np.abs(y + part)

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def step():
        for function, params in calls:
            function(C.byref(params))

    try:
        with torch.cuda.stream(stream):
            gpu_lib.iree_uk_mi355x_set_stream(stream.cuda_stream, 1)
            step()
            stream.synchronize()
            eager = ref.fetched(held["out"], 1, 16)
            check(eager, want, off, type)
            with torch.cuda.graph(graph, stream=stream):
                step()
    finally:
        gpu_lib.iree_uk_mi355x_set_stream(None, 0)
    for _ in range(3):
        for name in ("gate_pre", "up_pre", "hidden", "out"):
            held[name].device[:-64].fill_(0x55)
        for buffer, size in (w for w in keep if isinstance(w, tuple)):
            buffer[:size].fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(ref.fetched(held["out"], 1, 16), eager)

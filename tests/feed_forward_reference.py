"""Plain implementations of the gated product, its backward pass and the adapters in 64 bits, how far a result in f32
arithmetic may be off them, and their calls on tiled buffers with gaps and guards.

Bounds. A sum of n products in f32, in any order, is off by at most n additions, each by at most one unit in the last
place of a partial sum, which the sum of the magnitudes bounds: n * 2^-23 * sum |a| |b| (products of two 16-bit floats are
exact in f32, or off by half a unit, which adds one to n). The activations' e^-z is off, relatively, by |z| times two
roundings of z's and by one unit of the instruction, 1 / (1 + e) by two more units: (3 |z| + 6) * 2^-23 in all, generously
taken; below 2^-100 results may come out as zero.
"""
import ctypes as C

import numpy as np
import torch

from iree_amd import abi
from mx_reference import from_raw, raw, tiled, to_type, untiled, up

U = 2.0 ** -23
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}  # half a step of subnormals, or more
GUARD = 0xA5
ROOT = np.sqrt(2 / np.pi)


def values(rng, rows, cols, type, scale=1.0):
    return to_type((rng.standard_normal((rows, cols)) * scale).astype(np.float32), type).astype(np.float64)


def rounded_off(x, type):
    """How far a value that was rounded to `type` may be off."""
    return HALF_STEP[type] * np.abs(x) + TINY[type]


# In 64 bits -------------------------------------------------------------------------------


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-x))


def act(x, activation):
    """-> (act(x), act'(x), |z|)"""
    if activation == "gelu":
        z, inner = 2 * ROOT * (x + 0.044715 * x ** 3), 2 * ROOT * (1 + 3 * 0.044715 * x ** 2)
    else:
        z, inner = x, 1.0
    s = sigmoid(z)
    bend = s * sigmoid(-z) * inner
    if activation == "sigmoid":
        return s, bend, np.abs(z)
    return x * s, s + x * bend, np.abs(z)


def slope_magnitude(x, activation):
    z, inner = (2 * ROOT * (x + 0.044715 * x ** 3), 2 * ROOT * (1 + 3 * 0.044715 * x ** 2)) if activation == "gelu" else (x, 1.0)
    bend = sigmoid(z) * sigmoid(-z) * inner
    return bend if activation == "sigmoid" else sigmoid(z) + np.abs(x) * bend


def act_off(x, x_off, activation):
    """How far act(x) may be off for an x that is off by x_off: the slope is at most 1.13 in magnitude."""
    value, _, z = act(x, activation)
    return 1.13 * x_off + (3 * np.minimum(z, 100) + 6) * U * np.abs(value) + 2.0 ** -100


def gated(x, gate, up_, activation, pre=None):
    """-> (out, g, u) and how far each may be off in f32, ahead of the last rounding."""
    k = x.shape[1]
    g, u = x @ gate.T, x @ up_.T
    g_off, u_off = (k + 2) * U * (np.abs(x) @ np.abs(gate).T), (k + 2) * U * (np.abs(x) @ np.abs(up_).T)
    if pre is not None:
        g, u = g + pre[0], u + pre[1]
        g_off, u_off = g_off + U * (np.abs(pre[0]) + np.abs(g)), u_off + U * (np.abs(pre[1]) + np.abs(u))
    value = act(g, activation)[0]
    a_off = act_off(g, g_off, activation)
    off = a_off * (np.abs(u) + u_off) + np.abs(value) * u_off + U * np.abs(value * u)
    return (value * u, g, u), (off, g_off, u_off)


def backward(x, gate, up_, g, u, grad, activation, type, g_off=0, u_off=0):
    """-> (lhs_grad, gate_grad, up_grad) and how far each may be off ahead of the last rounding: the gradients of g and u are
    rounded to `type`. Where g and u are off themselves: slopes are at most 1.13 and slopes of slopes at most 1 in magnitude."""
    value, slope, z = act(g, activation)
    dg, du = grad * u * slope, grad * value
    dg_off = np.abs(grad * u) * ((3 * np.minimum(z, 100) + 12) * U * slope_magnitude(g, activation) + 2.0 ** -100) + 2 * U * np.abs(dg)
    dg_off = dg_off + np.abs(grad) * (1.13 * u_off + (np.abs(u) + u_off) * g_off)
    du_off = np.abs(grad) * act_off(g, g_off, activation) + U * np.abs(du)
    dg_off, du_off = dg_off + rounded_off(np.abs(dg) + dg_off, type), du_off + rounded_off(np.abs(du) + du_off, type)
    m, n = g.shape

    def product(a, a_off, b, terms):
        return a_off @ np.abs(b) + (terms + 2) * U * ((np.abs(a) + a_off) @ np.abs(b))

    results = dg @ gate + du @ up_, dg.T @ x, du.T @ x
    offs = (product(dg, dg_off, gate, 2 * n) + product(du, du_off, up_, 2 * n), product(dg.T, dg_off.T, x, m),
            product(du.T, du_off.T, x, m))
    return results, offs


def adapters(x, down, up_, index, scales):
    """x [m][k], down [count][rank][k], up_ [count][n][rank] -> (the part that is added, how far it may be off)."""
    m, k = x.shape
    n, rank = up_.shape[1], up_.shape[2]
    part, off = np.zeros((m, n)), np.zeros((m, n))
    for a in range(down.shape[0]):
        rows = np.nonzero(index == a)[0]
        if not len(rows):
            continue
        s = 1.0 if scales is None else np.float64(scales[a])
        t, t_off = x[rows] @ down[a].T, (k + 2) * U * (np.abs(x[rows]) @ np.abs(down[a]).T)
        part[rows] = s * (t @ up_[a].T)
        off[rows] = np.abs(s) * (t_off @ np.abs(up_[a]).T + (rank + 4) * U * ((np.abs(t) + t_off) @ np.abs(up_[a]).T))
    return part, off


def check(got, want, off, type):
    """`got`: values of `type`; `off`: how far the value may be off ahead of its rounding."""
    bound = off + rounded_off(np.abs(want) + off, type)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], bound[bad][:5])


# Buffers ----------------------------------------------------------------------------------


class Buffer:
    """Panels of tiles in device memory (or the host's), `gap` elements between them and `offset` in front, guards all round."""

    def __init__(self, panels, elements, type, gap=0, offset=0, data=None, host=False):
        self.panels, self.elements, self.type, self.offset = panels, elements, type, offset
        self.size = 4 if type == "f32" else 2
        self.stride = elements + gap
        whole = np.full((offset + max(panels, 1) * self.stride) * self.size + 64, GUARD, np.uint8)
        if data is not None:
            rows = raw(data, type).reshape(panels, elements).view(np.uint8)
            self._inner(whole)[:, :elements * self.size] = rows
        self.start = whole.copy()
        self.host = whole if host else None
        self.device = None if host else torch.from_numpy(whole).cuda()

    def _inner(self, whole):
        first, step = self.offset * self.size, self.stride * self.size
        return whole[first:first + self.panels * step].reshape(self.panels, step)

    def into(self, p, name):
        setattr(p, name + "_buffer", self.host.ctypes.data if self.device is None else self.device.data_ptr())
        setattr(p, name + "_offset", self.offset)
        setattr(p, name + "_stride0", self.stride)

    def fetch(self):
        """The elements' bytes as values [panels][elements]; what lies between and around them is as it was."""
        whole = self.host.copy() if self.device is None else self.device.cpu().numpy()
        width = self.elements * self.size
        got = self._inner(whole)[:, :width].copy()
        self._inner(whole)[:, :width] = self._inner(self.start)[:, :width]
        np.testing.assert_array_equal(whole, self.start)
        return from_raw(got.reshape(-1).view(np.float32 if self.type == "f32" else np.uint16), self.type).reshape(self.panels, self.elements)


def matrix(x, t0, t1, type, **layout):
    """[rows][cols], whole tiles."""
    return Buffer(x.shape[0] // t0, x.shape[1] * t0, type, data=tiled(x, t0, t1), **layout)


def empty(rows, cols, t0, type, **layout):
    return Buffer(rows // t0, cols * t0, type, **layout)


def fetched(buffer, t0, t1):
    x = buffer.fetch()
    return untiled(x.reshape(x.shape[0], x.shape[1] // (t0 * t1), t0, t1)).astype(np.float64)


def type_flag(prefix, type, out):
    return getattr(abi, "%s_TYPE_%s%s%s" % (prefix, type.upper(), type.upper(), out.upper()))


def tiles_into(p, m, n, k, tile):
    p.M0, p.N0, p.K0 = tile
    p.M, p.N, p.K = m // p.M0, n // p.N0, k // p.K0


def workspace(lib, name, p):
    """A workspace of the size that the call asks for, full of NaN."""
    size = getattr(lib, "iree_uk_mi355x_%s_workspace" % name)(C.byref(p))
    w = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    p.workspace_buffer, p.workspace_size = w.data_ptr(), size
    return w, size


def call(lib, name, p):
    getattr(lib, "iree_uk_mi355x_%s_p" % name)(C.byref(p))


def run_gated(lib, x, gate, up_, activation, tile, type, out, pre=None, mode="none", pre_type="f32", layout={}, host=False):
    """-> (out, g, u as stored or None), the kernel"""
    (m, k), n = x.shape, gate.shape[0]
    m0, n0, k0 = tile
    p = abi.GatedMmt4dParams()
    tiles_into(p, m, n, k, tile)
    at = lambda name: dict(layout.get(name, {}), host=host)  # noqa: E731
    held = {"lhs": matrix(x, m0, k0, type, **at("lhs")), "gate": matrix(gate, n0, k0, type, **at("gate")),
            "up": matrix(up_, n0, k0, type, **at("up")), "out": empty(m, n, m0, out, **at("out"))}
    p.flags = type_flag("GATED_MMT4D", type, out) | getattr(abi, "GATED_MMT4D_" + activation.upper())
    if mode != "none":
        for name, v in zip(("gate_pre", "up_pre"), pre or (None, None)):
            held[name] = empty(m, n, m0, pre_type, **at(name)) if v is None else matrix(v, m0, n0, pre_type, **at(name))
        p.flags |= (abi.GATED_MMT4D_PRE_LOAD if "load" in mode else 0) | (abi.GATED_MMT4D_PRE_STORE if "store" in mode else 0)
        if pre_type == "f32":
            p.flags |= abi.GATED_MMT4D_PRE_F32
    for name, b in held.items():
        b.into(p, name)
    call(lib, "gated_mmt4d", p)
    kernel = lib.iree_uk_mi355x_last_kernel()
    stored = [fetched(held[name], m0, n0) for name in ("gate_pre", "up_pre")] if mode != "none" else [None, None]
    return (fetched(held["out"], m0, n0), *stored), kernel


def run_backward(lib, x, gate, up_, g, u, grad, activation, tile, type, out, pre_type, accumulate=None, which="lgu", layout={},
                 host=False):
    """-> (lhs_grad, gate_grad, up_grad; None where not asked for), the kernel"""
    (m, k), n = x.shape, gate.shape[0]
    m0, n0, k0 = tile
    p = abi.GatedMmt4dBackwardParams()
    tiles_into(p, m, n, k, tile)
    at = lambda name: dict(layout.get(name, {}), host=host)  # noqa: E731
    held = {"lhs": matrix(x, m0, k0, type, **at("lhs")), "gate": matrix(gate, n0, k0, type, **at("gate")),
            "up": matrix(up_, n0, k0, type, **at("up")), "gate_pre": matrix(g, m0, n0, pre_type, **at("gate_pre")),
            "up_pre": matrix(u, m0, n0, pre_type, **at("up_pre")), "out_grad": matrix(grad, m0, n0, out, **at("out_grad"))}
    if "l" in which:
        held["lhs_grad"] = empty(m, k, m0, out, **at("lhs_grad"))
    for i, name in enumerate(("gate_grad", "up_grad")):
        if name[0] in which:
            held[name] = empty(n, k, n0, out, **at(name)) if accumulate is None else matrix(accumulate[i], n0, k0, out, **at(name))
    p.flags = type_flag("GATED_MMT4D", type, out) | getattr(abi, "GATED_MMT4D_" + activation.upper())
    p.flags |= (abi.GATED_MMT4D_PRE_F32 if pre_type == "f32" else 0) | (abi.GATED_MMT4D_ACCUMULATE if accumulate is not None else 0)
    for name, b in held.items():
        b.into(p, name)
    w, size = workspace(lib, "gated_mmt4d_backward", p)
    call(lib, "gated_mmt4d_backward", p)
    kernel = lib.iree_uk_mi355x_last_kernel()
    assert bool((w[size:] == 0xFF).all())
    sides = {"lhs_grad": (m0, k0), "gate_grad": (n0, k0), "up_grad": (n0, k0)}
    return tuple(fetched(held[name], *sides[name]) if name in held else None for name in sides), kernel


def run_adapters(lib, x, down, up_, index, scales, tile, type, out, init=None, layout={}, down_gap=(0, 0), up_gap=(0, 0), host=False):
    """-> the result, the kernel"""
    (m, k), (count, n, rank) = x.shape, up_.shape
    m0, n0, k0 = tile
    p = abi.AdapterMmt4dParams()
    tiles_into(p, m, n, k, tile)
    p.rank, p.count = rank, count
    at = lambda name: dict(layout.get(name, {}), host=host)  # noqa: E731
    held = {"lhs": matrix(x, m0, k0, type, **at("lhs")),
            "out": empty(m, n, m0, out, **at("out")) if init is None else matrix(init, m0, n0, out, **at("out"))}
    keep = []
    for name, v, gap in (("down", down, down_gap), ("up", up_, up_gap)):
        rows, cols = v.shape[1:]
        wide = np.full((count, rows, cols + gap[1]), np.nan)
        wide[:, :, :cols] = v
        held[name] = Buffer(max(count, 1), rows * (cols + gap[1]), type, data=wide if count else np.zeros((1, rows, cols + gap[1])),
                            gap=gap[0], **at(name))
        setattr(p, name + "_stride1", cols + gap[1])
    for name, b in held.items():
        b.into(p, name)
    index = np.ascontiguousarray(index, np.int32)
    if scales is not None:
        scales = np.ascontiguousarray(scales, np.float32)
    for name, v in (("index", index), ("scales", scales)):
        if v is None:
            continue
        t = v if host else torch.from_numpy(v).cuda()
        keep.append(t)
        setattr(p, name + "_buffer", v.ctypes.data if host else t.data_ptr())
    p.flags = type_flag("ADAPTER_MMT4D", type, out) | (abi.ADAPTER_MMT4D_ACCUMULATE if init is not None else 0)
    w, size = workspace(lib, "adapter_mmt4d", p)
    call(lib, "adapter_mmt4d", p)
    kernel = lib.iree_uk_mi355x_last_kernel()
    assert bool((w[size:] == 0xFF).all())
    return fetched(held["out"], m0, n0), kernel

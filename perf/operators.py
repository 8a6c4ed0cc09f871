"""Performance cases of the microscaled operators and of the norm that feeds them.

Microscaled values are 4-bit (e2m1) or 8-bit (e4m3) floats with one power-of-two scale
(e8m0) for every 32 consecutive values along K. A case has a "kind":

  pack        a row-major or transposed matrix into codes and scales, tiled for a product
  unpack      tiled codes and scales back into a row-major matrix
  round_trip  one after the other: the matrix as the product will see it
  norm        root-mean-square norm of rows, with the residual's addition where "residual"
              is true, into 8-bit integers with a scale for each row ("s8") or microscaled
  product     lhs [m, k] times rhs [n, k] transposed, both microscaled and tiled
  chain       norm into microscaled rows, then the product that reads them

With `own` false, run() computes them from elementary torch operations; with `own` true it
makes the library's calls, enqueued on torch's current stream.

The scale of a block is 2 to the floor of log2 of its largest magnitude, less the largest
exponent of the element type, not below 2**-127; elements are rounded to nearest, ties to
even, and saturate. The norm is y = (s * r) * w in 32 bits, with s the sum of input and residual
rounded to their type and r = 1 / sqrt(mean(s * s) + epsilon) in 64 bits, rounded to 32; an
8-bit row's scale is its largest |y| / 127 and not below 2**-126, its values y times the
scale's reciprocal, rounded to nearest, ties to even.
"""
import ctypes as C
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Largest exponent and value of the element types.
_EMAX = {"e2m1": 2, "e4m3": 8}
_EPSILON = 1e-5

_MAX_FLOPS = 2 * 4096 ** 3
_MAX_BYTES = 600 << 20


def _pack(name, type, format, rows, cols, tile, transposed=False, kind="pack"):
    return {"name": name, "kind": kind, "type": type, "format": format, "rows": rows, "cols": cols,
            "t0": tile[0], "t1": tile[1], "transposed": transposed}


def _norm(name, type, format, rows, cols, residual=True):
    return {"name": name, "kind": "norm", "type": type, "format": format, "rows": rows, "cols": cols,
            "residual": residual}


def _product(name, lhs, out, m, n, k, m0=1, n0=16):
    return {"name": name, "kind": "product", "lhs": lhs, "out": out, "m": m, "n": n, "k": k, "m0": m0, "n0": n0}


def listed():
    return [
        # One token's activations on their way into a product: what a call costs.
        _pack("pack_e4m3_token", "bf16", "e4m3", 1, 8192, (1, 128)),
        # The activations of a prompt, odd in both directions.
        _pack("pack_e2m1_ragged", "f16", "e2m1", 777, 4095, (16, 128), kind="round_trip"),
        # An f32 master copy of weights, [k][n], into the tiles that the product reads, and back
        # into what the product will multiply by (a training step's simulated quantisation).
        _pack("round_trip_weights", "f32", "e2m1", 14336, 4096, (16, 128), transposed=True, kind="round_trip"),
        # Stored weights widened for a program that multiplies in bf16.
        _pack("unpack_weights", "bf16", "e2m1", 28672, 8192, (16, 128), kind="unpack"),
        # One token's norm in front of an 8-bit integer product.
        _norm("norm_s8_token", "bf16", "s8", 1, 8192),
        # A prompt's norm in front of a microscaled product.
        _norm("norm_e4m3_prompt", "bf16", "e4m3", 4096, 8192),
        # The first norm of a model in f32, nothing added, rows that no block divides.
        _norm("norm_e2m1_ragged", "f32", "e2m1", 777, 4095, residual=False),
        # One decoded token through a feed-forward projection: streams the weights once.
        _product("decode_1", "e4m3", "bf16", 1, 14336, 4096),
        # Sixteen sequences through a larger one, activations in four bits too.
        _product("decode_16", "e2m1", "f32", 16, 28672, 8192),
        # A prompt of 512 tokens through an up-projection.
        _product("prefill_512", "e4m3", "bf16", 512, 11008, 4096),
        # The large square product, both sides in four bits and tiled.
        _product("square_4096", "e2m1", "f32", 4096, 4096, 4096, m0=16),
        # A ragged batch: norm, then the projection, as a layer makes them.
        {"name": "chain_ragged", "kind": "chain", "type": "bf16", "lhs": "e4m3", "out": "f16", "m": 77, "n": 4100,
         "k": 4095},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw_once(rng):
    kind = rng.choice(["pack", "unpack", "round_trip", "norm", "norm", "product", "product", "product", "chain"])
    type = rng.choice(sorted(_DTYPES))
    if kind in ("pack", "unpack", "round_trip"):
        return _pack("", type, "e4m3" if kind == "pack" else rng.choice(["e2m1", "e4m3"]), _log(rng, 1, 32768),
                     _log(rng, 32, 16384), rng.choice([(1, 128), (16, 128)]),
                     kind != "unpack" and rng.random() < 0.3, kind)
    if kind == "norm":
        return _norm("", type, rng.choice(["s8", "e4m3", "e2m1"]), _log(rng, 1, 8192), _log(rng, 64, 16384),
                     rng.random() < 0.7)
    lhs, out = rng.choice(["e2m1", "e4m3"]), rng.choice(sorted(_DTYPES))
    m = rng.choice([_log(rng, 1, 16), _log(rng, 17, 256), _log(rng, 257, 4096)])
    n, k = _log(rng, 64, 28672), _log(rng, 64, 14336)
    if kind == "chain":
        return {"kind": "chain", "type": type, "lhs": lhs, "out": out, "m": m, "n": n, "k": k}
    return _product("", lhs, out, m, n, k, m0=1 if rng.random() < 0.7 else 16, n0=16 if rng.random() < 0.8 else 1)


def draw(rng):
    while True:
        case = _draw_once(rng)
        case.pop("name", None)
        w = work(case)
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES:
            return case


def _up(v, to):
    return -(-v // to) * to


def _code_bytes(count, format):
    return count // 2 if format == "e2m1" else count


def _mx_bytes(rows, cols, format, t0, t1=128):
    """Bytes of the codes and scales of a padded matrix."""
    count = _up(rows, t0) * _up(cols, t1)
    return _code_bytes(count, format) + count // 32


def _product_work(case, lhs_bytes):
    m, n, k = _up(case["m"], case.get("m0", 1)), _up(case["n"], case.get("n0", 16)), _up(case["k"], 128)
    out = m * n * _DTYPES[case["out"]].itemsize
    return lhs_bytes + _mx_bytes(case["n"], case["k"], "e2m1", case.get("n0", 16)) + out, 2 * m * n * k


def _norm_bytes(case, rows, cols, format, residual):
    size = _DTYPES[case["type"]].itemsize
    given = rows * cols * size * (3 if residual else 1) + cols * size  # (with a residual: it is read, the sum written)
    return given + (rows * cols + 4 * rows if format == "s8" else _mx_bytes(rows, cols, format, 1))


def work(case):
    kind = case["kind"]
    if kind in ("pack", "unpack", "round_trip"):
        plain = case["rows"] * case["cols"] * _DTYPES[case["type"]].itemsize
        tiled = _mx_bytes(case["rows"], case["cols"], case["format"], case["t0"], case["t1"])
        return {"bytes": (plain + tiled) * (2 if kind == "round_trip" else 1), "flops": 0}
    if kind == "norm":
        return {"bytes": _norm_bytes(case, case["rows"], case["cols"], case["format"], case["residual"]), "flops": 0}
    lhs = _mx_bytes(case["m"], case["k"], case["lhs"], case.get("m0", 1))
    total, flops = _product_work(case, lhs)
    if kind == "chain":
        total += _norm_bytes(case, case["m"], case["k"], case["lhs"], True)
    return {"bytes": total, "flops": flops}


# Inputs -----------------------------------------------------------------------------------


def _activations(gen, rows, cols):
    """Normal values; one channel in 64 is eight times as large, as in a trained model."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 1 / 64
    return x * torch.where(loud, 8.0, 1.0)


def _weights(gen, rows, cols):
    return torch.randn(rows, cols, generator=gen, device="cuda") * 0.02


def _quantised(x, format):
    """f32 [rows][cols], cols a multiple of 32 -> (element values in f32, scale bytes [rows][cols / 32])."""
    blocks = x.reshape(x.shape[0], -1, 32)
    largest = blocks.abs().amax(-1)
    exponent = (largest.view(torch.int32) >> 23) - _EMAX[format]
    scale = exponent.clamp(min=0)
    # 2**(127 - scale), which is a normal number for every scale up to 252
    v = (blocks * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)).reshape(x.shape)
    if format == "e4m3":
        return v.clamp(-448, 448).to(torch.float8_e4m3fn).float(), scale.to(torch.uint8)
    v = v.clamp(-6, 6)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(v / step) * step, scale.to(torch.uint8)


def _codes(values, format):
    """Element values -> bytes; two 4-bit codes a byte, the first in the low half."""
    if format == "e4m3":
        return values.to(torch.float8_e4m3fn).view(torch.uint8)
    a = values.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code + torch.signbit(values).to(torch.uint8) * 8
    return code[:, 0::2] | code[:, 1::2] << 4


def _values(codes, format):
    """Bytes -> element values in f32."""
    if format == "e4m3":
        return codes.view(torch.float8_e4m3fn).float()
    both = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    magnitude = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    return torch.cat([magnitude, -magnitude])[both.long()]


def _scale_values(scale):
    """Scale bytes -> 2**(scale - 127) in f32."""
    return scale.view(torch.float8_e8m0fnu).float()


def _padded(x, t0, t1):
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, _up(cols, t1) - cols, 0, _up(rows, t0) - rows))


def _tiled(x, t0, t1):
    """[rows][cols] -> [rows / t0][cols / t1][t0][t1], flat."""
    rows, cols = x.shape
    return x.reshape(rows // t0, t0, cols // t1, t1).transpose(1, 2).contiguous().reshape(-1)


def _untiled(x, rows, cols, t0, t1):
    return x.reshape(rows // t0, cols // t1, t0, t1).transpose(1, 2).reshape(rows, cols)


def _mx_operand(x, format, t0, t1):
    """A matrix -> tiled codes and tiled scales."""
    values, scale = _quantised(_padded(x, t0, t1), format)
    codes = _codes(values, format)
    return _tiled(codes, t0, _code_bytes(t1, format)), _tiled(scale, t0, t1 // 32)


def _mx_empty(rows, cols, format, t0, t1):
    count = _up(rows, t0) * _up(cols, t1)
    return (torch.zeros(_code_bytes(count, format), dtype=torch.uint8, device="cuda"),
            torch.zeros(count // 32, dtype=torch.uint8, device="cuda"))


def _widened(codes, scale, rows, cols, format, t0, t1):
    """Tiled codes and scales of a padded matrix -> its values in f32."""
    rows, cols = _up(rows, t0), _up(cols, t1)
    values = _values(_untiled(codes, rows, _code_bytes(cols, format), t0, _code_bytes(t1, format)), format)
    scale = _scale_values(_untiled(scale, rows, cols // 32, t0, t1 // 32))
    return (values.reshape(rows, -1, 32) * scale.unsqueeze(-1)).reshape(rows, cols)


def _norm_inputs(gen, case, rows, cols, residual):
    dtype = _DTYPES[case["type"]]
    x = _activations(gen, rows, cols).to(dtype)
    old = _activations(gen, rows, cols).to(dtype) if residual else None
    weight = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
    return x, old, weight


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"case": dict(case)}
    if kind in ("pack", "round_trip"):
        x = _weights(gen, case["rows"], case["cols"]) if case["transposed"] else _activations(gen, case["rows"], case["cols"])
        x = x.to(_DTYPES[case["type"]])
        state["x"] = x.t().contiguous() if case["transposed"] else x
    if kind == "unpack":
        state["codes"], state["scales"] = _mx_operand(_weights(gen, case["rows"], case["cols"]), case["format"],
                                                      case["t0"], case["t1"])
    if kind in ("pack", "round_trip"):
        state["codes"], state["scales"] = _mx_empty(case["rows"], case["cols"], case["format"], case["t0"], case["t1"])
    if kind in ("unpack", "round_trip"):
        state["out"] = torch.zeros(case["rows"], case["cols"], dtype=_DTYPES[case["type"]], device="cuda")
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        state["x"], state["residual"], state["weight"] = _norm_inputs(gen, case, rows, cols, case["residual"])
        state["sum"] = torch.zeros_like(state["x"]) if case["residual"] else None
        if case["format"] == "s8":
            state["codes"] = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
            state["scales"] = torch.zeros(rows, device="cuda")
        else:
            state["codes"], state["scales"] = _mx_empty(rows, cols, case["format"], 1, 128)
        if case["format"] == "e2m1":
            state["out"] = torch.zeros(rows, _up(cols, 128), device="cuda")
    if kind in ("product", "chain"):
        m, n, k, m0, n0 = case["m"], case["n"], case["k"], case.get("m0", 1), case.get("n0", 16)
        state["rhs"], state["rhs_scales"] = _mx_operand(_weights(gen, n, k), "e2m1", n0, 128)
        if kind == "product":
            state["lhs"], state["lhs_scales"] = _mx_operand(_activations(gen, m, k), case["lhs"], m0, 128)
        else:
            state["x"], state["residual"], state["weight"] = _norm_inputs(gen, case, m, k, True)
            state["sum"] = torch.zeros_like(state["x"])
            state["lhs"], state["lhs_scales"] = _mx_empty(m, k, case["lhs"], 1, 128)
        state["out"] = torch.zeros(_up(m, m0) * _up(n, n0), dtype=_DTYPES[case["out"]], device="cuda")
    state["returned"] = _returned(state)
    return state


def _returned(state):
    """The output buffers, as the types whose values they hold."""
    case = state["case"]
    kind = case["kind"]
    if kind in ("unpack", "round_trip", "product"):
        return state["out"]
    if kind == "chain":
        return {"sum": state["sum"], "out": state["out"]}
    got = {"sum": state["sum"]} if kind == "norm" and case["residual"] else {}
    if case["format"] == "s8":
        return dict(got, values=state["codes"], scales=state["scales"])
    scales = state["scales"].view(torch.float8_e8m0fnu)
    if case["format"] == "e2m1":
        return dict(got, values=state["out"], scales=scales)  # (codes of 4 bits, widened by an unpack)
    return dict(got, values=state["codes"].view(torch.float8_e4m3fn), scales=scales)


# Plain form -------------------------------------------------------------------------------


def _plain_norm(state, rows, cols):
    """-> (sum of input and residual, y in f32)"""
    total = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(state["x"].dtype)
    wide = total.double()
    r = torch.rsqrt((wide * wide).sum(-1) / cols + C.c_float(_EPSILON).value).float()
    return total, total.float() * r.unsqueeze(-1) * state["weight"].float()


def _plain_product(lhs, rhs, out):
    return (lhs @ rhs.t()).to(out)


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "pack":
        x = (state["x"].t() if case["transposed"] else state["x"]).float()
        values, scale = _quantised(_padded(x, case["t0"], case["t1"]), case["format"])
        return {"values": _tiled(values.to(torch.float8_e4m3fn), case["t0"], case["t1"]),
                "scales": _tiled(scale, case["t0"], case["t1"] // 32).view(torch.float8_e8m0fnu)}
    if kind == "round_trip":
        x = (state["x"].t() if case["transposed"] else state["x"]).float()
        values, scale = _quantised(_padded(x, 1, 32), case["format"])
        y = values.reshape(values.shape[0], -1, 32) * _scale_values(scale).unsqueeze(-1)
        return y.reshape(values.shape)[:, :case["cols"]].to(_DTYPES[case["type"]])
    if kind == "unpack":
        y = _widened(state["codes"], state["scales"], case["rows"], case["cols"], case["format"], case["t0"], case["t1"])
        return y[:case["rows"], :case["cols"]].to(_DTYPES[case["type"]])
    if kind == "norm":
        total, y = _plain_norm(state, case["rows"], case["cols"])
        got = {"sum": total} if case["residual"] else {}
        if case["format"] == "s8":
            scale = (y.abs().amax(-1) / 127).clamp(min=2.0 ** -126)
            return dict(got, values=torch.round(y * (1 / scale).unsqueeze(-1)).to(torch.int8), scales=scale)
        values, scale = _quantised(_padded(y, 1, 128), case["format"])
        if case["format"] == "e2m1":
            widened = (values.reshape(values.shape[0], -1, 32) * _scale_values(scale).unsqueeze(-1)).reshape(values.shape)
            return dict(got, values=widened, scales=scale.reshape(-1).view(torch.float8_e8m0fnu))
        return dict(got, values=values.to(torch.float8_e4m3fn).reshape(-1), scales=scale.reshape(-1).view(torch.float8_e8m0fnu))
    m, n, k, m0, n0 = case["m"], case["n"], case["k"], case.get("m0", 1), case.get("n0", 16)
    rhs = _widened(state["rhs"], state["rhs_scales"], n, k, "e2m1", n0, 128)
    if kind == "chain":
        total, y = _plain_norm(state, m, k)
        values, scale = _quantised(_padded(y, 1, 128), case["lhs"])
        lhs = (values.reshape(m, -1, 32) * _scale_values(scale).unsqueeze(-1)).reshape(m, -1)
        return {"sum": total, "out": _tiled(_plain_product(lhs, rhs, _DTYPES[case["out"]]), m0, n0)}
    lhs = _widened(state["lhs"], state["lhs_scales"], m, k, case["lhs"], m0, 128)
    return _tiled(_plain_product(lhs, rhs, _DTYPES[case["out"]]), m0, n0)


# The library's calls ------------------------------------------------------------------------


def _pack_call(lib, abi, state, format, x, rows, cols, t0, t1, transposed):
    p = abi.MxPackParams()
    p.in_buffer = x.data_ptr()
    p.in_stride0, p.in_stride1 = (1, rows) if transposed else (cols, 1)
    p.out_buffer, p.scales_buffer = state["codes"].data_ptr(), state["scales"].data_ptr()
    p.in_size0, p.in_size1 = rows, cols
    p.out_size0, p.out_size1, p.out_size2, p.out_size3 = -(-rows // t0), -(-cols // t1), t0, t1
    p.out_stride0, p.scales_stride0 = p.out_size1 * t0 * t1, p.out_size1 * t0 * t1 // 32
    p.flags = getattr(abi, "MX_PACK_TYPE_%s%s" % (state["case"]["type"].upper(), format.upper()))
    return lib.iree_uk_mi355x_mx_pack_p, p


def _unpack_call(lib, abi, state, format, type, rows, cols, t0, t1):
    p = abi.MxUnpackParams()
    p.in_buffer, p.scales_buffer = state["codes"].data_ptr(), state["scales"].data_ptr()
    p.in_size0, p.in_size1, p.in_size2, p.in_size3 = -(-rows // t0), -(-cols // t1), t0, t1
    p.in_stride0, p.scales_stride0 = p.in_size1 * t0 * t1, p.in_size1 * t0 * t1 // 32
    p.out_buffer, p.out_stride0, p.out_stride1 = state["out"].data_ptr(), cols, 1
    p.out_size0, p.out_size1 = rows, cols
    p.flags = getattr(abi, "MX_UNPACK_TYPE_%s%s" % (format.upper(), type.upper()))
    return lib.iree_uk_mi355x_mx_unpack_p, p


def _norm_call(lib, abi, state, format, rows, cols, out_cols, codes, scales):
    p = abi.RmsNormParams()
    p.in_buffer, p.in_stride0 = state["x"].data_ptr(), cols
    if state["residual"] is not None:
        p.residual_buffer, p.residual_stride0 = state["residual"].data_ptr(), cols
        p.sum_buffer, p.sum_stride0 = state["sum"].data_ptr(), cols
    p.weight_buffer = state["weight"].data_ptr()
    p.out_buffer, p.out_stride0 = codes.data_ptr(), out_cols
    p.scales_buffer, p.scales_stride0 = scales.data_ptr(), 1 if format == "s8" else out_cols // 32
    p.size0, p.size1, p.out_size1 = rows, cols, out_cols
    p.epsilon = _EPSILON
    p.flags = getattr(abi, "RMS_NORM_TYPE_%s%s" % (state["case"]["type"].upper(), format.upper()))
    return lib.iree_uk_mi355x_rms_norm_p, p


def _product_call(lib, abi, state):
    case = state["case"]
    m0, n0, k0 = case.get("m0", 1), case.get("n0", 16), 128
    p = abi.MxMmt4dParams()
    p.M, p.N, p.K = -(-case["m"] // m0), -(-case["n"] // n0), -(-case["k"] // k0)
    p.M0, p.N0, p.K0 = m0, n0, k0
    p.lhs_buffer, p.lhs_scales_buffer = state["lhs"].data_ptr(), state["lhs_scales"].data_ptr()
    p.rhs_buffer, p.rhs_scales_buffer = state["rhs"].data_ptr(), state["rhs_scales"].data_ptr()
    p.out_buffer = state["out"].data_ptr()
    p.lhs_stride0, p.rhs_stride0, p.out_stride0 = p.K * m0 * k0, p.K * n0 * k0, p.N * m0 * n0
    p.lhs_scales_stride0, p.rhs_scales_stride0 = p.lhs_stride0 // 32, p.rhs_stride0 // 32
    p.flags = getattr(abi, "MX_MMT4D_TYPE_%sE2M1%s" % (case["lhs"].upper(), case["out"].upper()))
    return lib.iree_uk_mi355x_mx_mmt4d_p, p


def _calls(state):
    """The calls of one pass, their parameters filled in as a program does once for its buffers."""
    from iree_amd import abi, library
    lib = library.load()
    lib.iree_uk_mi355x_set_stream(torch.cuda.current_stream().cuda_stream, 1)
    case = state["case"]
    kind = case["kind"]
    calls = []
    if kind in ("pack", "round_trip"):
        calls.append(_pack_call(lib, abi, state, case["format"], state["x"], case["rows"], case["cols"], case["t0"],
                                case["t1"], case["transposed"]))
    if kind in ("unpack", "round_trip"):
        calls.append(_unpack_call(lib, abi, state, case["format"], case["type"], case["rows"], case["cols"], case["t0"],
                                  case["t1"]))
    if kind == "norm":
        cols = case["cols"] if case["format"] == "s8" else _up(case["cols"], 128)
        calls.append(_norm_call(lib, abi, state, case["format"], case["rows"], case["cols"], cols, state["codes"],
                                state["scales"]))
        if case["format"] == "e2m1":
            calls.append(_unpack_call(lib, abi, state, "e2m1", "f32", case["rows"], cols, 1, 128))
    if kind == "chain":
        calls.append(_norm_call(lib, abi, state, case["lhs"], case["m"], case["k"], _up(case["k"], 128), state["lhs"],
                                state["lhs_scales"]))
    if kind in ("product", "chain"):
        calls.append(_product_call(lib, abi, state))
    return [(function, C.byref(p)) for function, p in calls]


def run(state):
    if not own:
        return _run_plain(state)
    if "calls" not in state:
        state["calls"] = _calls(state)
    for function, params in state["calls"]:
        function(params)
    return state["returned"]


# In 64 bits -------------------------------------------------------------------------------


def _exact_quantised(x, format):
    """f64 [rows][cols] -> (element values, scales [rows][cols / 32]), both in f64."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32))
    blocks = x.reshape(x.shape[0], -1, 32)
    largest = blocks.abs().amax(-1)
    e = torch.frexp(largest).exponent - 1 - _EMAX[format]  # largest = 2**(e + emax) * [1, 2)
    e = torch.where(largest > 0, e, -127).clamp(min=-127)
    v = torch.ldexp(blocks, -e.unsqueeze(-1))
    mantissa_bits, lowest, top = (1, 0, 6.0) if format == "e2m1" else (3, -6, 448.0)
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 1).clamp(min=lowest) - mantissa_bits)
    q = torch.minimum(torch.round(v.abs() / step) * step, torch.full_like(v, top)) * torch.sign(v)
    return q.reshape(x.shape), torch.ldexp(torch.ones_like(largest), e)


def _exact_times(values, scale):
    return (values.reshape(values.shape[0], -1, 32) * scale.unsqueeze(-1)).reshape(values.shape)


def _exact_norm(x, old, weight):
    total = x if old is None else (x.double() + old.double()).to(x.dtype)
    s = total.double()
    return total.double(), s / torch.sqrt((s * s).mean(-1, keepdim=True) + _EPSILON) * weight.double()


def _to_tiles(x, t0, t1, pad):
    rows, cols = x.shape
    whole = torch.full((_up(rows, t0), _up(cols, t1)), pad, dtype=x.dtype, device=x.device)
    whole[:rows, :cols] = x
    return whole.unfold(0, t0, t0).unfold(1, t1, t1).reshape(-1)


def _exact_product(lhs, rhs):
    return lhs @ rhs.t()


def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind in ("pack", "round_trip"):
        x = _weights(gen, case["rows"], case["cols"]) if case["transposed"] else _activations(gen, case["rows"], case["cols"])
        q, scale = _exact_quantised(x.to(_DTYPES[case["type"]]).double(), case["format"])
        if kind == "round_trip":
            return _exact_times(q, scale)[:, :case["cols"]]
        return {"values": _to_tiles(q, case["t0"], case["t1"], 0.0),
                "scales": _to_tiles(scale, case["t0"], case["t1"] // 32, 2.0 ** -127)}
    if kind == "unpack":
        q, scale = _exact_quantised(_weights(gen, case["rows"], case["cols"]).double(), case["format"])
        return _exact_times(q, scale)[:, :case["cols"]]
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        total, y = _exact_norm(*_norm_inputs(gen, case, rows, cols, case["residual"]))
        got = {"sum": total} if case["residual"] else {}
        if case["format"] == "s8":
            return dict(got, values=None, scales=y.abs().amax(-1) / 127)
        q, scale = _exact_quantised(y, case["format"])
        scales = _to_tiles(scale, 1, 4, 2.0 ** -127)
        if case["format"] == "e4m3":
            return dict(got, values=_to_tiles(q, 1, 128, 0.0), scales=scales)
        return dict(got, values=_to_tiles(_exact_times(q, scale), 1, 128, 0.0).reshape(rows, -1), scales=scales)
    m, n, k, m0, n0 = case["m"], case["n"], case["k"], case.get("m0", 1), case.get("n0", 16)
    rhs = _exact_times(*_exact_quantised(_weights(gen, n, k).double(), "e2m1"))
    if kind == "product":
        lhs = _exact_times(*_exact_quantised(_activations(gen, m, k).double(), case["lhs"]))
        return _to_tiles(_exact_product(lhs, rhs), m0, n0, 0.0)
    total, y = _exact_norm(*_norm_inputs(gen, case, m, k, True))
    lhs = _exact_times(*_exact_quantised(y, case["lhs"]))
    return {"sum": total, "out": _to_tiles(_exact_product(lhs, rhs), m0, n0, 0.0)}

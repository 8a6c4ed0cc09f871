"""Plain implementations of the microscaled operators and of the norm, in 64 bits, and
the parameter structs of their calls on numpy arrays or device addresses.

A quantised matrix is (codes, scales): uint8 codes one a value, not yet two a byte, and one
scale byte for 32 values.
"""
import numpy as np

from iree_amd import abi

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([(8 + c % 8) * 2.0 ** (c // 8 - 10) if c >= 8 else c * 2.0 ** -9 for c in range(127)])
TABLE = {"e2m1": E2M1, "e4m3": E4M3}
SIGN = {"e2m1": 8, "e4m3": 128}
EMAX = {"e2m1": 2, "e4m3": 8}
BITS = {"e2m1": 4, "e4m3": 8}


def up(v, to):
    return -(-v // to) * to


def bf16_round(x):
    """f64 or f32 values that f32 holds -> the nearest bf16, in f32 (ties to even)."""
    x = np.asarray(x, dtype=np.float32)
    bits = x.view(np.uint32).astype(np.uint64)
    r = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float32)


def to_type(x, type):
    """f32 values rounded to `type`, in f32."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(over="ignore"):
        return {"f32": x, "f16": x.astype(np.float16).astype(np.float32), "bf16": bf16_round(x)}[type]


def raw(x, type):
    """Values that `type` holds, as they lie in memory."""
    x = np.asarray(x, dtype=np.float32)
    if type == "f32":
        return x.copy()
    if type == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    return (x.view(np.uint32) >> 16).astype(np.uint16)


def from_raw(x, type):
    if type == "f32":
        return x.view(np.float32)
    if type == "f16":
        return x.view(np.float16).astype(np.float32)
    return (x.view(np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantise(x, format):
    """f64 [rows][cols], cols a multiple of 32 -> codes, scales, by search in the table of elements."""
    with np.errstate(invalid="ignore"):  # (signalling NaNs)
        x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(x.shape[0], -1, 32)
    bad = ~np.isfinite(blocks).all(-1)
    blocks = np.where(bad[..., None], 0.0, blocks)
    largest = np.abs(blocks).max(-1)
    exponent = np.frexp(largest)[1] - 1
    scale = np.where(largest > 0, np.maximum(exponent + 127 - EMAX[format], 0), 0)
    v = np.ldexp(np.abs(blocks), 127 - scale[..., None])
    table = TABLE[format]
    above = np.clip(np.searchsorted(table, v), 1, len(table) - 1)  # table[above - 1] < v <= table[above], or the end
    low, high = table[above - 1], table[above]
    take_high = (v - low > high - v) | ((v - low == high - v) & (above % 2 == 0))
    codes = np.where(take_high, above, above - 1)
    codes = codes + np.where(np.signbit(blocks), SIGN[format], 0)
    codes[bad] = 0
    scale[bad] = 255
    return codes.astype(np.uint8).reshape(x.shape), scale.astype(np.uint8)


def widen(codes, scales, format):
    """The values of codes and scales in f64."""
    magnitude = np.concatenate([TABLE[format], [np.nan]]) if format == "e4m3" else TABLE[format]
    v = np.concatenate([magnitude, -magnitude])[codes].reshape(codes.shape[0], -1, 32)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * s[..., None]).reshape(codes.shape)


def tiled(x, t0, t1):
    rows, cols = x.shape
    return np.ascontiguousarray(x.reshape(rows // t0, t0, cols // t1, t1).transpose(0, 2, 1, 3))


def untiled(x):
    o0, o1, t0, t1 = x.shape
    return np.ascontiguousarray(x.transpose(0, 2, 1, 3)).reshape(o0 * t0, o1 * t1)


def to_bytes(codes, format):
    """Codes one a value -> as they lie in memory, along the last axis."""
    return codes if format == "e4m3" else (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def from_bytes(x, format):
    if format == "e4m3":
        return x
    return np.stack([x & 15, x >> 4], -1).reshape(*x.shape[:-1], -1)


def padded(x, t0, t1):
    return np.pad(x, ((0, up(x.shape[0], t0) - x.shape[0]), (0, up(x.shape[1], t1) - x.shape[1])))


def random_codes(rng, rows, cols, format, scales=(117, 137)):
    codes = rng.integers(0, 16 if format == "e2m1" else 256, (rows, cols)).astype(np.uint8)
    if format == "e4m3":
        codes = np.where(codes % 128 == 127, codes - 1, codes).astype(np.uint8)
    return codes, rng.integers(scales[0], scales[1] + 1, (rows, cols // 32)).astype(np.uint8)


def norm(x, residual, weight, epsilon, type):
    """-> (sum as `type` holds it, y as the operator defines it: in f32, from r rounded to f32)."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(all="ignore"):
        s = x if residual is None else to_type(x + residual, type)
        wide = s.astype(np.float64)
        r = (1 / np.sqrt((wide * wide).sum(-1) / s.shape[1] + np.float64(np.float32(epsilon)))).astype(np.float32)
        y = s * r[:, None]
        return s, (y if weight is None else y * np.asarray(weight, dtype=np.float32)).astype(np.float32)


def quantise_s8(y):
    with np.errstate(all="ignore"):
        largest = np.abs(y).max(-1).astype(np.float32)
        scale = np.maximum(largest / np.float32(127), np.float32(2.0 ** -126)).astype(np.float32)
        bad = ~np.isfinite(y).all(-1)
        q = np.rint(y * (np.float32(1) / scale)[:, None])
    q[bad] = 0
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


# Parameters -------------------------------------------------------------------------------


def pack_params(src, rows, cols, codes, scales, t0, t1, type, format, in_strides=None, codes_stride0=None,
                scales_stride0=None):
    p = abi.MxPackParams()
    p.in_buffer, (p.in_stride0, p.in_stride1) = src, in_strides or (cols, 1)
    p.out_buffer, p.scales_buffer = codes, scales
    p.in_size0, p.in_size1 = rows, cols
    p.out_size0, p.out_size1, p.out_size2, p.out_size3 = -(-rows // t0), -(-cols // t1), t0, t1
    row = p.out_size1 * t0 * t1
    p.out_stride0 = codes_stride0 if codes_stride0 is not None else row
    p.scales_stride0 = scales_stride0 if scales_stride0 is not None else row // 32
    p.flags = getattr(abi, "MX_PACK_TYPE_%s%s" % (type.upper(), format.upper()))
    return p


def unpack_params(codes, scales, dst, rows, cols, t0, t1, format, type, out_strides=None, codes_stride0=None,
                  scales_stride0=None):
    p = abi.MxUnpackParams()
    p.in_buffer, p.scales_buffer, p.out_buffer = codes, scales, dst
    p.in_size0, p.in_size1, p.in_size2, p.in_size3 = -(-rows // t0), -(-cols // t1), t0, t1
    row = p.in_size1 * t0 * t1
    p.in_stride0 = codes_stride0 if codes_stride0 is not None else row
    p.scales_stride0 = scales_stride0 if scales_stride0 is not None else row // 32
    p.out_stride0, p.out_stride1 = out_strides or (cols, 1)
    p.out_size0, p.out_size1 = rows, cols
    p.flags = getattr(abi, "MX_UNPACK_TYPE_%s%s" % (format.upper(), type.upper()))
    return p


def mmt4d_params(lhs, lhs_scales, rhs, rhs_scales, out, tiles, tile, lhs_format, out_type, accumulate=False):
    p = abi.MxMmt4dParams()
    p.lhs_buffer, p.lhs_scales_buffer, p.rhs_buffer, p.rhs_scales_buffer = lhs, lhs_scales, rhs, rhs_scales
    p.out_buffer = out
    p.M, p.N, p.K = tiles
    p.M0, p.N0, p.K0 = tile
    p.lhs_stride0, p.rhs_stride0, p.out_stride0 = p.K * p.M0 * p.K0, p.K * p.N0 * p.K0, p.N * p.M0 * p.N0
    p.lhs_scales_stride0, p.rhs_scales_stride0 = p.lhs_stride0 // 32, p.rhs_stride0 // 32
    p.flags = getattr(abi, "MX_MMT4D_TYPE_%sE2M1%s" % (lhs_format.upper(), out_type.upper()))
    if accumulate:
        p.flags |= abi.MX_MMT4D_ACCUMULATE
    return p


def norm_params(x, residual, total, weight, out, scales, rows, cols, out_cols, type, format, epsilon=1e-5):
    p = abi.RmsNormParams()
    p.in_buffer, p.in_stride0 = x, cols
    p.residual_buffer, p.residual_stride0 = residual, cols
    p.sum_buffer, p.sum_stride0 = total, cols
    p.weight_buffer = weight
    p.out_buffer, p.out_stride0 = out, out_cols
    p.scales_buffer, p.scales_stride0 = scales, 1 if format == "s8" else out_cols // 32
    p.size0, p.size1, p.out_size1 = rows, cols, out_cols
    p.epsilon = epsilon
    p.flags = getattr(abi, "RMS_NORM_TYPE_%s%s" % (type.upper(), format.upper()))
    return p

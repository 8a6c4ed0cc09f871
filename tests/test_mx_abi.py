"""What the microscaled operators and the norm refuse, and what they return from early: no GPU needed."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import mx_reference as ref
from iree_amd import abi, library
from test_abi import Failures

BUF = np.zeros(1 << 16, np.uint8)
AT = BUF.ctypes.data


def refused(entry, p, what=None):
    lib = library.load()
    with Failures() as f:
        getattr(lib, "iree_uk_mi355x_%s_p" % entry)(C.byref(p) if p is not None else None)
    assert len(f.seen) == 1, f.seen
    assert lib.iree_uk_mi355x_last_kernel() == b""
    if what:
        assert what in f.seen[0], f.seen


def changed(p, kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def pack(**kw):
    p = ref.pack_params(AT, 16, 128, AT + 16384, AT + 32768, 16, 128, "f32", "e2m1")
    return changed(p, kw)


def unpack(**kw):
    return changed(ref.unpack_params(AT, AT + 16384, AT + 32768, 16, 128, 16, 128, "e2m1", "f32"), kw)


def mmt4d(**kw):
    p = ref.mmt4d_params(AT, AT + 8192, AT + 16384, AT + 24576, AT + 32768, (2, 2, 1), (16, 16, 128), "e2m1", "f32")
    return changed(p, kw)


def norm(**kw):
    p = ref.norm_params(AT, AT + 8192, AT + 16384, AT + 24576, AT + 32768, AT + 40960, 4, 64, 64, "f32", "e4m3")
    return changed(p, kw)


@pytest.mark.parametrize("entry", ["mx_pack", "mx_unpack", "mx_mmt4d", "rms_norm"])
def test_null_parameters(entry):
    refused(entry, None)


@pytest.mark.parametrize("kw", [
    dict(flags=0), dict(flags=7), dict(flags=0x101), dict(in_size0=-1), dict(in_size1=-1), dict(out_size0=-1),
    dict(out_size3=100), dict(out_size3=-32), dict(in_stride0=-1), dict(in_stride1=-1), dict(out_stride0=-2),
    dict(scales_stride0=-1), dict(out_offset=1), dict(out_stride0=2049), dict(in_size0=17), dict(in_size1=129),
    dict(out_size0=2, in_size0=32, out_stride0=2046), dict(out_size0=2, in_size0=32, out_stride0=2048, scales_stride0=63),
    dict(scales_buffer=AT + 16384 + 1000), dict(scales_buffer=AT), dict(out_buffer=AT + 8000),
    dict(in_buffer=None), dict(out_buffer=None), dict(scales_buffer=None), dict(in_buffer=None, in_offset=4),
    dict(out_size1=1 << 62), dict(out_size0=1 << 40, out_size1=1 << 40)])
def test_pack(kw):
    refused("mx_pack", pack(**kw))


@pytest.mark.parametrize("kw", [
    dict(flags=0), dict(flags=7), dict(flags=0x201), dict(out_size0=-1), dict(in_size2=-1), dict(in_size3=48),
    dict(in_stride0=-2), dict(in_offset=3), dict(in_stride0=1001), dict(scales_stride0=-1), dict(out_stride0=-1),
    dict(out_stride1=-1), dict(out_stride0=127), dict(out_stride1=0), dict(out_size0=17), dict(out_size1=129),
    dict(out_buffer=AT + 512), dict(out_buffer=AT + 16384 + 8), dict(out_buffer=None), dict(in_buffer=None),
    dict(scales_buffer=None), dict(scales_buffer=None, scales_offset=16)])
def test_unpack(kw):
    refused("mx_unpack", unpack(**kw))


@pytest.mark.parametrize("kw", [
    dict(flags=0), dict(flags=7), dict(flags=0x201), dict(M=-1), dict(N=1 << 31), dict(K=-1), dict(M0=1 << 15),
    dict(N0=-1), dict(K0=100), dict(K0=-32), dict(lhs_offset=1), dict(rhs_offset=1), dict(lhs_stride0=2047),
    dict(rhs_stride0=2047), dict(lhs_stride0=-2048), dict(rhs_scales_stride0=-64), dict(out_stride0=511),
    dict(out_buffer=AT), dict(out_buffer=AT + 8192), dict(out_buffer=AT + 16384), dict(out_buffer=AT + 24576 - 4),
    dict(lhs_buffer=None), dict(lhs_scales_buffer=None), dict(rhs_buffer=None), dict(rhs_scales_buffer=None),
    dict(out_buffer=None), dict(out_buffer=None, out_offset=4)])
def test_mmt4d(kw):
    refused("mx_mmt4d", mmt4d(**kw))


@pytest.mark.parametrize("kw", [
    dict(flags=0), dict(flags=10), dict(flags=0x204), dict(size0=-1), dict(size1=-1), dict(out_size1=63),
    dict(out_size1=72), dict(in_stride0=-1), dict(residual_stride0=-1), dict(sum_stride0=-1), dict(out_stride0=-1),
    dict(scales_stride0=-1), dict(epsilon=-1.0), dict(epsilon=float("nan")), dict(residual_buffer=None),
    dict(sum_stride0=63), dict(out_stride0=63), dict(scales_stride0=1), dict(flags=abi.RMS_NORM_TYPE_F32E2M1, out_offset=1),
    dict(sum_buffer=AT + 4), dict(sum_buffer=AT + 8192, sum_stride0=65), dict(sum_buffer=AT + 24576),
    dict(out_buffer=AT + 24576), dict(out_buffer=AT), dict(scales_buffer=AT + 16384), dict(scales_buffer=AT + 32768 + 8),
    dict(in_buffer=None), dict(out_buffer=None), dict(scales_buffer=None), dict(out_buffer=None, out_offset=32)])
def test_norm(kw):
    refused("rms_norm", norm(**kw))


def test_early_returns_look_at_no_buffer():
    lib = library.load()
    none = dict.fromkeys(("in_buffer", "out_buffer", "scales_buffer"))
    with Failures() as f:
        lib.iree_uk_mi355x_mx_pack_p(C.byref(pack(out_size0=0, in_size0=0, **none)))
        lib.iree_uk_mi355x_mx_unpack_p(C.byref(unpack(out_size0=0, **none)))
        products = dict.fromkeys(("lhs_buffer", "lhs_scales_buffer", "rhs_buffer", "rhs_scales_buffer", "out_buffer"))
        lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(mmt4d(M=0, **products)))
        lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(mmt4d(N0=0, **products)))
        lib.iree_uk_mi355x_mx_mmt4d_p(C.byref(mmt4d(K=0, flags=abi.MX_MMT4D_TYPE_E2M1E2M1F32 | abi.MX_MMT4D_ACCUMULATE,
                                                    **products)))
        lib.iree_uk_mi355x_rms_norm_p(C.byref(norm(size0=0, residual_buffer=None, sum_buffer=None, **none)))
    assert f.seen == []
    assert lib.iree_uk_mi355x_last_kernel() == b""


def test_column_ranges_of_one_matrix_do_not_overlap():
    # Input and sum side by side in the rows of one buffer: no byte in common, though the spans cross. Without a GPU the
    # call fails later, in the HIP runtime; with one it runs.
    p = norm(in_stride0=128, sum_buffer=AT + 256, sum_stride0=128, residual_buffer=AT + 32768 + 16384, residual_stride0=64)
    p.out_buffer, p.scales_buffer = AT + 32768, AT + 40960
    with Failures() as f:
        library.load().iree_uk_mi355x_rms_norm_p(C.byref(p))
    assert not any("overlap" in m for m in f.seen), f.seen


def test_reference_quantiser_rounds_to_nearest_even():
    # The tests' own search, on values whose codes are known.
    x = np.zeros((1, 32))
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.76]
    codes, scales = ref.quantise(x, "e2m1")
    assert scales[0, 0] == 127 and codes[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8 + 2]
    x[0, :3] = [448, 464, -500]
    codes, scales = ref.quantise(x, "e4m3")
    assert scales[0, 0] == 127 and codes[0, :3].tolist() == [126, 126, 254]


def test_structs_and_flags_match_the_header(tmp_path):
    structs = {"mx_pack": abi.MxPackParams, "mx_unpack": abi.MxUnpackParams, "mx_mmt4d": abi.MxMmt4dParams,
               "rms_norm": abi.RmsNormParams}
    flags = [n for n in vars(abi) if re.match(r"(MX_PACK|MX_UNPACK|MX_MMT4D|RMS_NORM)_", n)]
    lines, want = [], []
    for name, struct in structs.items():
        c = "iree_uk_mi355x_%s_params_t" % name
        lines.append('printf("%%zu\\n", sizeof(%s));' % c)
        want.append(C.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (c, field))
            want.append(getattr(struct, field).offset)
    for flag in flags:
        lines.append('printf("%%d\\n", (int)IREE_UK_MI355X_FLAG_%s);' % flag)
        want.append(getattr(abi, flag))
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "iree_uk_mi355x.h"\nint main(void) {\n%s\nreturn 0;\n}\n' %
                      "\n".join(lines))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I" + include, str(source), "-o", str(program)], check=True)
    got = subprocess.run([str(program)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    assert [int(x) for x in got] == want and len(flags) == 29

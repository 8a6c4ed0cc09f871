"""What the gated product, its backward pass and the adapters refuse, and what they return from early: no GPU needed."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from iree_amd import abi, library
from test_abi import Failures

BUF = np.zeros((1 << 20) + 256, np.uint8)
AT = -(-BUF.ctypes.data // 256) * 256
NONE = None


def refused(entry, p):
    """By a check of its own, not by the HIP runtime."""
    lib = library.load()
    with Failures() as f:
        getattr(lib, "iree_uk_mi355x_%s_p" % entry)(C.byref(p) if p is not None else None)
    assert len(f.seen) == 1 and "hip" not in f.seen[0] and "launch" not in f.seen[0], f.seen
    assert lib.iree_uk_mi355x_last_kernel() == b""


def filled(p, operands, **kw):
    p.M, p.N, p.K, p.M0, p.N0, p.K0 = 2, 3, 4, 4, 16, 8
    rows = {"lhs": 128, "lhs_grad": 128, "gate": 512, "up": 512, "gate_grad": 512, "up_grad": 512}
    for i, name in enumerate(operands):
        setattr(p, name + "_buffer", AT + 32768 * i)
        setattr(p, name + "_stride0", rows.get(name, 192))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def gated(**kw):
    return filled(abi.GatedMmt4dParams(), ("lhs", "gate", "up", "gate_pre", "up_pre", "out"), **dict(
        dict(flags=abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_PRE_STORE), **kw))


def backward(**kw):
    p = filled(abi.GatedMmt4dBackwardParams(), ("lhs", "gate", "up", "gate_pre", "up_pre", "out_grad", "lhs_grad", "gate_grad", "up_grad"),
               flags=abi.GATED_MMT4D_TYPE_BF16BF16F32 | abi.GATED_MMT4D_GELU)
    p.workspace_buffer, p.workspace_size = AT + 32768 * 10, 65536
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def adapter(**kw):
    p = filled(abi.AdapterMmt4dParams(), ("lhs", "down", "up", "out"), flags=abi.ADAPTER_MMT4D_TYPE_F16F16F32)
    p.rank, p.count = 8, 2
    p.down_stride0, p.down_stride1, p.up_stride0, p.up_stride1 = 8 * 32, 32, 48 * 8, 8
    p.index_buffer, p.scales_buffer = AT + 32768 * 4, AT + 32768 * 5
    p.workspace_buffer, p.workspace_size = AT + 32768 * 6, 65536
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("entry", ["gated_mmt4d", "gated_mmt4d_backward", "adapter_mmt4d"])
def test_null_parameters(entry):
    refused(entry, None)


SIZES = [dict(M=-1), dict(N=1 << 31), dict(K=-1), dict(M0=1 << 15), dict(N0=-1), dict(K0=-8)]
F32 = abi.GATED_MMT4D_TYPE_F16F16F32
PRE_LOAD, PRE_STORE, PRE_F32 = abi.GATED_MMT4D_PRE_LOAD, abi.GATED_MMT4D_PRE_STORE, abi.GATED_MMT4D_PRE_F32


@pytest.mark.parametrize("kw", SIZES + [
    dict(flags=abi.GATED_MMT4D_SILU), dict(flags=F32), dict(flags=F32 | 0x400), dict(flags=5 | abi.GATED_MMT4D_SILU),
    dict(flags=F32 | abi.GATED_MMT4D_SILU | PRE_F32), dict(flags=F32 | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_ACCUMULATE),
    dict(flags=F32 | abi.GATED_MMT4D_SILU | 0x10000), dict(lhs_stride0=-128), dict(gate_stride0=-1), dict(up_stride0=-512),
    dict(gate_pre_stride0=191), dict(up_pre_stride0=-192), dict(out_stride0=191), dict(lhs_buffer=NONE), dict(gate_buffer=NONE),
    dict(up_buffer=NONE), dict(gate_pre_buffer=NONE), dict(up_pre_buffer=NONE, up_pre_offset=4), dict(out_buffer=NONE),
    dict(out_buffer=AT), dict(out_buffer=AT + 32768 + 64), dict(out_buffer=AT + 65536 - 4), dict(out_buffer=AT + 3 * 32768),
    dict(gate_pre_buffer=AT), dict(up_pre_buffer=AT + 2 * 32768), dict(up_pre_buffer=AT + 3 * 32768 + 2),
    dict(M=(1 << 31) - 1, lhs_stride0=1 << 60), dict(lhs_offset=1 << 62)])
def test_gated(kw):
    refused("gated_mmt4d", gated(**kw))


def test_gated_terms_that_are_only_loaded_may_coincide():
    p = gated(flags=F32 | abi.GATED_MMT4D_SILU | PRE_LOAD, gate_pre_stride0=0, up_pre_stride0=0, up_pre_buffer=AT + 3 * 32768)
    with Failures() as f:  # (without a GPU the call fails later, in the HIP runtime; with one it runs)
        library.load().iree_uk_mi355x_gated_mmt4d_p(C.byref(p))
    assert not any("overlap" in m or "apart" in m or "stride" in m for m in f.seen), f.seen


@pytest.mark.parametrize("kw", SIZES + [
    dict(flags=abi.GATED_MMT4D_SILU), dict(flags=F32), dict(flags=F32 | abi.GATED_MMT4D_SILU | PRE_LOAD),
    dict(flags=F32 | abi.GATED_MMT4D_SILU | PRE_STORE), dict(lhs_stride0=-128), dict(gate_stride0=-1), dict(out_grad_stride0=-192),
    dict(gate_pre_stride0=-192), dict(lhs_grad_stride0=127), dict(gate_grad_stride0=511), dict(up_grad_stride0=0), dict(lhs_buffer=NONE),
    dict(gate_buffer=NONE), dict(up_buffer=NONE), dict(gate_pre_buffer=NONE), dict(up_pre_buffer=NONE), dict(out_grad_buffer=NONE),
    dict(workspace_buffer=NONE), dict(workspace_size=0), dict(workspace_size=-1), dict(workspace_buffer=AT + 32768 * 10 + 8),
    dict(lhs_grad_buffer=AT), dict(gate_grad_buffer=AT + 32768), dict(up_grad_buffer=AT + 7 * 32768 + 32), dict(workspace_buffer=AT),
    dict(lhs_grad_buffer=AT + 5 * 32768), dict(workspace_buffer=AT + 8 * 32768), dict(out_grad_offset=1 << 62)])
def test_backward(kw):
    refused("gated_mmt4d_backward", backward(**kw))


@pytest.mark.parametrize("kw", SIZES + [
    dict(flags=0), dict(flags=5), dict(flags=0x201), dict(rank=-1), dict(rank=1 << 15), dict(count=-1), dict(count=1 << 31),
    dict(M=(1 << 31) - 1, M0=2), dict(lhs_stride0=-128), dict(down_stride0=-1), dict(down_stride1=-32), dict(up_stride0=-8),
    dict(up_stride1=-8), dict(out_stride0=191), dict(lhs_buffer=NONE), dict(down_buffer=NONE), dict(up_buffer=NONE),
    dict(index_buffer=NONE), dict(out_buffer=NONE), dict(workspace_buffer=NONE), dict(workspace_size=0),
    dict(workspace_buffer=AT + 32768 * 6 + 16), dict(index_buffer=AT + 32768 * 4 + 2), dict(scales_buffer=AT + 1), dict(out_buffer=AT),
    dict(out_buffer=AT + 32768), dict(out_buffer=AT + 2 * 32768), dict(out_buffer=AT + 4 * 32768), dict(out_buffer=AT + 5 * 32768),
    dict(workspace_buffer=AT + 32768), dict(workspace_buffer=AT + 3 * 32768), dict(down_stride1=1 << 61)])
def test_adapter(kw):
    refused("adapter_mmt4d", adapter(**kw))


def test_the_workspaces_of_calls_that_are_refused():
    lib = library.load()
    for size, p in ((lib.iree_uk_mi355x_gated_mmt4d_backward_workspace, backward(flags=0)),
                    (lib.iree_uk_mi355x_adapter_mmt4d_workspace, adapter(rank=-1)),
                    (lib.iree_uk_mi355x_gated_mmt4d_backward_workspace, backward(M=(1 << 31) - 1, N=(1 << 31) - 1, M0=16384, N0=16384))):
        with Failures() as f:
            assert size(C.byref(p)) == 0
        assert len(f.seen) == 1


def test_workspaces_look_at_no_buffer():
    lib = library.load()
    with Failures() as f:
        p = backward(lhs_buffer=NONE, gate_buffer=NONE, up_buffer=NONE, workspace_buffer=NONE)
        assert lib.iree_uk_mi355x_gated_mmt4d_backward_workspace(C.byref(p)) > 0
        p = adapter(lhs_buffer=NONE, down_buffer=NONE, out_buffer=NONE, index_buffer=NONE, workspace_buffer=NONE)
        assert lib.iree_uk_mi355x_adapter_mmt4d_workspace(C.byref(p)) > 0
    assert f.seen == []


def test_early_returns_look_at_no_buffer():
    lib = library.load()
    none = dict.fromkeys(("lhs_buffer", "gate_buffer", "up_buffer", "gate_pre_buffer", "up_pre_buffer", "out_buffer"))
    grads = dict.fromkeys(("lhs_grad_buffer", "gate_grad_buffer", "up_grad_buffer"))
    inputs = dict.fromkeys(("lhs_buffer", "gate_buffer", "up_buffer", "gate_pre_buffer", "up_pre_buffer", "out_grad_buffer"))
    pools = dict.fromkeys(("lhs_buffer", "down_buffer", "up_buffer", "index_buffer", "out_buffer", "workspace_buffer"))
    accumulate = abi.ADAPTER_MMT4D_TYPE_F16F16F32 | abi.ADAPTER_MMT4D_ACCUMULATE
    with Failures() as f:
        for kw in (dict(M=0), dict(N=0), dict(M0=0), dict(N0=0)):
            lib.iree_uk_mi355x_gated_mmt4d_p(C.byref(gated(**kw, **none)))
            lib.iree_uk_mi355x_adapter_mmt4d_p(C.byref(adapter(**kw, **pools)))
        for kw in (dict(K=0), dict(K0=0), dict(M=0, N=0), grads, dict(N=0, lhs_grad_buffer=NONE),
                   dict(M=0, flags=F32 | abi.GATED_MMT4D_SILU | abi.GATED_MMT4D_ACCUMULATE), dict(M=0, gate_grad_buffer=NONE, up_grad_buffer=NONE)):
            lib.iree_uk_mi355x_gated_mmt4d_backward_p(C.byref(backward(workspace_buffer=NONE, **{**inputs, **kw})))
        for kw in (dict(K=0), dict(rank=0), dict(count=0)):
            lib.iree_uk_mi355x_adapter_mmt4d_p(C.byref(adapter(flags=accumulate, **kw, **pools)))
    assert f.seen == []
    assert lib.iree_uk_mi355x_last_kernel() == b""


def test_structs_and_flags_match_the_header(tmp_path):
    structs = {"gated_mmt4d": abi.GatedMmt4dParams, "gated_mmt4d_backward": abi.GatedMmt4dBackwardParams,
               "adapter_mmt4d": abi.AdapterMmt4dParams}
    flags = [n for n in vars(abi) if re.match(r"(GATED_MMT4D|ADAPTER_MMT4D)_", n)]
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
    assert [int(x) for x in got] == want and len(flags) == 16

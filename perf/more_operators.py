"""Performance cases of the gated feed-forward product, its backward pass, and low-rank adapters.

A case has a "kind":

  gated     out = act(lhs gate^T) * (lhs up^T) from one call; "pre" says whether terms are added to
            the two products first ("load") or the products are stored as well ("store")
  backward  from out's gradient and the stored products: the gradients of lhs, gate and up
  train     a gated product that stores, then its backward pass
  adapters  out = lhs rhs^T, plus for each row scale (lhs down^T) up^T of the adapter that its index
            names, where it names one
  block     a serving step's feed-forward block: adapters beside gate and up, the gated product, the
            product with the last weights, and the adapters beside that

lhs is [m, k], weights are [n, k], in tiles of 16 x 16; "m0" is the height of the tiles of lhs and
out, of which 1 makes them row-major. Sizes are filled up with zeros to whole tiles. An adapter's
down is [rank, k] and its up [n, rank], row-major. act is x s(x) (silu), x s(1.595769 x + 0.0713548 x^3)
(gelu in its tanh form) or s(x) (sigmoid), with s the logistic function.

With `own` false, run() computes them from elementary torch operations; with `own` true it makes the
library's calls, enqueued on torch's current stream.
"""
import ctypes as C
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_N0 = _K0 = 16
_CUBIC = 0.044715
_ROOT = math.sqrt(2 / math.pi)

_MAX_FLOPS = 8 * 4096 * 11008 * 4096
_MAX_BYTES = 960 << 20


def _gated(name, type, out, activation, m, n, k, m0=1, pre="none", pre_type="f32", kind="gated"):
    return {"name": name, "kind": kind, "type": type, "out": out, "activation": activation, "m": m, "n": n, "k": k,
            "m0": m0, "pre": pre, "pre_type": pre_type}


def _adapters(name, type, out, m, n, k, rank, count, rows, kind="adapters"):
    return {"name": name, "kind": kind, "type": type, "out": out, "m": m, "n": n, "k": k, "m0": 1, "rank": rank,
            "count": count, "rows": rows}


def listed():
    return [
        # One decoded token: streams both weights once.
        _gated("gated_token", "bf16", "bf16", "silu", 1, 14336, 4096),
        # Sixteen sequences decoded together through a larger layer.
        _gated("gated_decode_16", "f16", "f16", "gelu", 16, 28672, 8192),
        # A ragged batch on top of terms from elsewhere (adapters, biases of a row).
        _gated("gated_ragged", "bf16", "f32", "sigmoid", 77, 4100, 4095, pre="load"),
        # A prompt of 512 tokens.
        _gated("gated_prompt_512", "bf16", "bf16", "silu", 512, 11008, 4096),
        # A long prompt, operands and result in tiles.
        _gated("gated_prompt_4096", "f16", "f16", "silu", 4096, 11008, 4096, m0=16),
        # A training step of a small layer with odd sizes.
        _gated("train_small", "f16", "f16", "gelu", 130, 1000, 500, pre="store", pre_type="f16", kind="train"),
        # A training step of a micro-batch of 2048 tokens.
        _gated("train_2048", "bf16", "bf16", "silu", 2048, 8192, 4096, pre="store", pre_type="bf16", kind="train"),
        # The backward pass of a large micro-batch, from products that the forward pass has stored.
        _gated("backward_4096", "bf16", "bf16", "silu", 4096, 11008, 4096, pre_type="bf16", kind="backward"),
        # One token of one request beside the shared projection: what the calls cost.
        _adapters("adapters_token", "bf16", "bf16", 1, 4096, 4096, 16, 8, "mixed"),
        # 64 requests decoded together, of 64 adapters, in the order in which they came.
        _adapters("adapters_decode_64", "bf16", "f32", 64, 14336, 4096, 16, 64, "mixed"),
        # Prompts of several requests, each its rows in a run, some without an adapter.
        _adapters("adapters_prompts", "f16", "f32", 2000, 4096, 4096, 64, 12, "runs"),
        # A serving step's whole feed-forward block.
        dict(_adapters("block_decode_40", "bf16", "bf16", 40, 11008, 4096, 16, 16, "mixed", kind="block"), activation="silu"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw_once(rng):
    kind = rng.choice(["gated", "gated", "gated", "train", "backward", "adapters", "adapters", "adapters", "block"])
    type = rng.choice(["f16", "bf16"])
    out = rng.choice([type, "f32"])
    m = rng.choice([_log(rng, 1, 16), _log(rng, 17, 256), _log(rng, 257, 4096)])
    n, k = _log(rng, 64, 28672), _log(rng, 64, 14336)
    if kind in ("adapters", "block"):
        case = _adapters("", type, type if kind == "block" else out, m, n, k, rng.choice([4, 8, 16, 32, 64, 128, rng.randint(1, 64)]),
                         _log(rng, 1, 64), rng.choice(["mixed", "runs"]), kind)
        return dict(case, activation=rng.choice(["silu", "gelu", "sigmoid"])) if kind == "block" else case
    m0 = rng.choice([1, 1, 16])
    activation = rng.choice(["silu", "gelu", "sigmoid"])
    if kind == "gated":
        pre = rng.choice(["none", "none", "load", "store"])
        return _gated("", type, out, activation, m, n, k, m0, pre, rng.choice([type, "f32"]) if pre == "load" else out)
    return _gated("", type, type, activation, m, n, k, m0, "store" if kind == "train" else "none", type, kind)


def draw(rng):
    while True:
        case = _draw_once(rng)
        case.pop("name", None)
        if case.get("pre") == "store" and case["pre_type"] not in (case["type"], "f32"):
            continue
        w = work(case)
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES:
            return case


def _up(v, to):
    return -(-v // to) * to


def _padded_sizes(case):
    return _up(case["m"], case["m0"]), _up(case["n"], _N0), _up(case["k"], _K0)


def _adapter_work(case, m, n, k):
    """Of the adapters beside one product: bytes of the weights of those that rows can name, and operations."""
    rank, named = case["rank"], min(case["count"], case["m"])
    return 2 * named * rank * (k + n) + 4 * m, 2 * m * rank * (k + n)


def work(case):
    m, n, k = _padded_sizes(case)
    kind = case["kind"]
    out = _DTYPES[case["out"]].itemsize
    product = 2 * m * n * k
    if kind == "adapters":
        b, f = _adapter_work(case, m, n, k)
        return {"bytes": 2 * (m * k + n * k) + out * m * n + b, "flops": product + f}
    if kind == "block":
        b1, f1 = _adapter_work(case, m, n, k)
        b2, f2 = _adapter_work(case, m, k, n)
        return {"bytes": 2 * (m * k + 3 * n * k) + out * m * k + 2 * b1 + b2, "flops": 3 * product + 2 * f1 + f2}
    weights = 2 * 2 * n * k
    pre = 2 * m * n * _DTYPES[case["pre_type"]].itemsize
    forward = 2 * m * k + weights + out * m * n + (pre if case["pre"] != "none" else 0)
    # read: the products, out's gradient, lhs and the weights; written: their gradients
    backward = pre + out * m * n + 2 * m * k + weights + out * (m * k + 2 * n * k)
    if kind == "gated":
        return {"bytes": forward, "flops": 2 * product}
    if kind == "backward":
        return {"bytes": backward, "flops": 4 * product}
    return {"bytes": forward + backward, "flops": 6 * product}


# Inputs -----------------------------------------------------------------------------------


def _filled(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _tiled(x, t0, t1):
    """[rows][cols] -> [rows / t0][cols / t1][t0][t1], flat."""
    rows, cols = x.shape
    if t0 == 1:
        return x.contiguous().reshape(-1)
    return x.reshape(rows // t0, t0, cols // t1, t1).transpose(1, 2).contiguous().reshape(-1)


def _untiled(x, rows, cols, t0, t1):
    if t0 == 1:
        return x.reshape(rows, cols)
    return x.reshape(rows // t0, cols // t1, t0, t1).transpose(1, 2).reshape(rows, cols)


def _activations(gen, rows, cols):
    """Normal values; one channel in 64 is eight times as large, as in a trained model."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 1 / 64
    return x * torch.where(loud, 8.0, 1.0)


def _weights(gen, rows, cols):
    """Such that products of normed activations are of the order of one."""
    return torch.randn(rows, cols, generator=gen, device="cuda") / math.sqrt(cols)


def _row_indices(gen, case):
    m, count = case["m"], case["count"]
    if case["rows"] == "mixed":
        # Every request has an adapter of its own while there are enough.
        return torch.randperm(max(m, count), generator=gen, device="cuda")[:m].remainder(count).to(torch.int32)
    # Runs of rows, of random lengths; one in eight or so has no adapter.
    runs = max(1, min(m, case["count"]))
    ends = torch.sort(torch.randint(0, m + 1, (runs - 1,), generator=gen, device="cuda")).values
    of = torch.randint(0, count, (runs,), generator=gen, device="cuda")
    of = torch.where(torch.rand(runs, generator=gen, device="cuda") < 1 / 8, -1, of)
    return of[torch.searchsorted(ends, torch.arange(m, device="cuda"), right=True)].to(torch.int32)


def _adapter_inputs(gen, case, n, k, dtype):
    """Of one product of [.., k] with [n, k]: down [count][rank][k], up [count][n][rank]."""
    count, rank = case["count"], case["rank"]
    down = torch.randn(count, rank, k, generator=gen, device="cuda") / math.sqrt(k)
    up = torch.randn(count, n, rank, generator=gen, device="cuda") * 0.1
    return down.to(dtype), up.to(dtype)


def _inputs(case, seed):
    """Row-major inputs, filled up to whole tiles, by name."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, n, k = _padded_sizes(case)
    dtype, kind = _DTYPES[case["type"]], case["kind"]
    made = {}

    def put(name, x, rows, cols, type=dtype):
        made[name] = _filled(x, rows, cols).to(type)

    put("lhs", _activations(gen, case["m"], case["k"]), m, k)
    if kind == "adapters":
        put("rhs", _weights(gen, case["n"], case["k"]), n, k)
    else:
        put("gate", _weights(gen, case["n"], case["k"]), n, k)
        put("up", _weights(gen, case["n"], case["k"]), n, k)
    if kind == "block":
        put("last", _weights(gen, case["k"], case["n"]), k, n)
    if kind in ("adapters", "block"):
        made["index"] = _row_indices(gen, case)
        made["scales"] = torch.rand(case["count"], generator=gen, device="cuda") + 0.5
        pairs = [("", n, k)] if kind == "adapters" else [("gate_", n, k), ("up_", n, k), ("last_", k, n)]
        for name, to, of in pairs:
            made[name + "down"], made[name + "to"] = _adapter_inputs(gen, case, to, of, dtype)
        return made
    if case["pre"] == "load" or kind == "backward":
        for name in ("gate_pre", "up_pre"):
            x = 1.4 * torch.randn(case["m"], case["n"], generator=gen, device="cuda")
            put(name, x, m, n, _DTYPES[case["pre_type"]])
    if kind in ("backward", "train"):
        put("out_grad", torch.randn(case["m"], case["n"], generator=gen, device="cuda"), m, n, _DTYPES[case["out"]])
    return made


def prepare(case, seed):
    m, n, k = _padded_sizes(case)
    m0, made = case["m0"], _inputs(case, seed)
    state = {"case": dict(case), "sizes": (m, n, k)}
    for name, x in made.items():
        if name in ("lhs",):
            x = _tiled(x, m0, _K0)
        elif name in ("rhs", "gate", "up", "last"):
            x = _tiled(x, _N0, _K0)
        elif name in ("gate_pre", "up_pre", "out_grad"):
            x = _tiled(x, m0, _N0)
        state[name] = x

    def empty(name, count, type):
        state[name] = torch.zeros(count, dtype=_DTYPES[type], device="cuda")

    kind = case["kind"]
    if kind in ("gated", "train"):
        empty("out", m * n, case["out"])
        if case["pre"] == "store":
            empty("gate_pre", m * n, case["pre_type"])
            empty("up_pre", m * n, case["pre_type"])
    if kind in ("backward", "train"):
        empty("lhs_grad", m * k, case["out"])
        empty("gate_grad", n * k, case["out"])
        empty("up_grad", n * k, case["out"])
    if kind == "adapters":
        empty("out", m * n, case["out"])
    if kind == "block":
        empty("gate_pre", m * n, "f32")
        empty("up_pre", m * n, "f32")
        empty("hidden", m * n, case["type"])
        empty("out", m * k, case["out"])
    return state


def _returned(state):
    case = state["case"]
    names = ["out"] if case["kind"] != "backward" else []
    if case.get("pre") == "store":
        names += ["gate_pre", "up_pre"]
    if case["kind"] in ("backward", "train"):
        names += ["lhs_grad", "gate_grad", "up_grad"]
    return {name: state[name] for name in names}


# Plain form -------------------------------------------------------------------------------


def _logistic(x):
    return 1 / (1 + torch.exp(-x))


def _plain_act(x, activation):
    if activation == "silu":
        return x * _logistic(x)
    if activation == "gelu":
        return x * _logistic(2 * _ROOT * (x + _CUBIC * x * x * x))
    return _logistic(x)


def _plain_act_and_slope(x, activation):
    if activation == "gelu":
        s, inner = _logistic(2 * _ROOT * (x + _CUBIC * x * x * x)), 2 * _ROOT * (1 + 3 * _CUBIC * x * x)
    else:
        s, inner = _logistic(x), 1.0
    if activation == "sigmoid":
        return s, s * (1 - s)
    return x * s, s + x * s * (1 - s) * inner


def _plain_adapters(y, x, index, down, up, scales):
    """y + the adapters' part, in f32."""
    for a in range(down.shape[0]):
        rows = torch.nonzero(index == a).reshape(-1)
        part = scales[a] * ((x[rows] @ down[a].float().t()) @ up[a].float().t())
        y = y.index_add(0, rows, part)
    return y


def _run_plain(state):
    case = state["case"]
    m, n, k = state["sizes"]
    m0, kind = case["m0"], case["kind"]
    out_type = _DTYPES[case["out"]]
    x = _untiled(state["lhs"], m, k, m0, _K0).float()
    if kind == "adapters":
        y = x @ _untiled(state["rhs"], n, k, _N0, _K0).float().t()
        return {"out": _plain_adapters(y, x, state["index"], state["down"], state["to"], state["scales"]).to(out_type).reshape(-1)}
    gate, up = (_untiled(state[name], n, k, _N0, _K0).float() for name in ("gate", "up"))
    if kind == "block":
        index, scales = state["index"], state["scales"]
        g = _plain_adapters(x @ gate.t(), x, index, state["gate_down"], state["gate_to"], scales)
        u = _plain_adapters(x @ up.t(), x, index, state["up_down"], state["up_to"], scales)
        h = _plain_act(g, case["activation"]) * u
        y = h @ _untiled(state["last"], k, n, _N0, _K0).float().t()
        return {"out": _plain_adapters(y, h, index, state["last_down"], state["last_to"], scales).to(out_type).reshape(-1)}
    got = {}
    if kind == "backward" or case["pre"] == "load":
        g, u = (_untiled(state[name], m, n, m0, _N0).float() for name in ("gate_pre", "up_pre"))
    if kind != "backward":
        if case["pre"] == "load":
            g, u = g + x @ gate.t(), u + x @ up.t()
        else:
            g, u = x @ gate.t(), x @ up.t()
        got["out"] = _tiled((_plain_act(g, case["activation"]) * u).to(out_type), m0, _N0)
        if case["pre"] == "store":
            got["gate_pre"], got["up_pre"] = (_tiled(v.to(_DTYPES[case["pre_type"]]), m0, _N0) for v in (g, u))
    if kind in ("backward", "train"):
        grad = _untiled(state["out_grad"], m, n, m0, _N0).float()
        value, slope = _plain_act_and_slope(g, case["activation"])
        dg, du = grad * u * slope, grad * value
        got["lhs_grad"] = _tiled((dg @ gate + du @ up).to(out_type), m0, _K0)
        got["gate_grad"] = _tiled((dg.t() @ x).to(out_type), _N0, _K0)
        got["up_grad"] = _tiled((du.t() @ x).to(out_type), _N0, _K0)
    return got


# The library's calls ------------------------------------------------------------------------


def _operand(p, name, tensor, stride0):
    setattr(p, name + "_buffer", tensor.data_ptr())
    setattr(p, name + "_stride0", stride0)


def _tiles(p, m, n, k, m0):
    p.M, p.N, p.K, p.M0, p.N0, p.K0 = m // m0, n // _N0, k // _K0, m0, _N0, _K0


def _type_name(case, out=None):
    type = case["type"].upper()
    return type + type + (out or case["out"]).upper()


def _mmt4d_call(lib, abi, state, lhs, rhs, out, m, n, k):
    case = state["case"]
    p = abi.Mmt4dParams()
    _tiles(p, m, n, k, case["m0"])
    _operand(p, "lhs", state[lhs], p.K * p.M0 * p.K0)
    _operand(p, "rhs", state[rhs], p.K * p.N0 * p.K0)
    _operand(p, "out", state[out], p.N * p.M0 * p.N0)
    p.flags = getattr(abi, "MMT4D_TYPE_" + _type_name(case)) | abi.MMT4D_SKIP_INTERMEDIATE_ROUNDINGS
    return lib.iree_uk_mmt4d_p, p


def _gated_call(lib, abi, state, out):
    case = state["case"]
    m, n, k = state["sizes"]
    pre = "load" if case["kind"] == "block" else case["pre"]
    p = abi.GatedMmt4dParams()
    _tiles(p, m, n, k, case["m0"])
    _operand(p, "lhs", state["lhs"], p.K * p.M0 * p.K0)
    _operand(p, "gate", state["gate"], p.K * p.N0 * p.K0)
    _operand(p, "up", state["up"], p.K * p.N0 * p.K0)
    _operand(p, "out", state[out], p.N * p.M0 * p.N0)
    p.flags = getattr(abi, "GATED_MMT4D_TYPE_" + _type_name(case)) | getattr(abi, "GATED_MMT4D_" + case["activation"].upper())
    if pre != "none":
        _operand(p, "gate_pre", state["gate_pre"], p.out_stride0)
        _operand(p, "up_pre", state["up_pre"], p.out_stride0)
        p.flags |= abi.GATED_MMT4D_PRE_LOAD if pre == "load" else abi.GATED_MMT4D_PRE_STORE
        if state["gate_pre"].dtype == torch.float32:
            p.flags |= abi.GATED_MMT4D_PRE_F32
    return lib.iree_uk_mi355x_gated_mmt4d_p, p


def _workspace(state, name, p, size):
    state[name] = torch.empty(max(1, size(C.byref(p))), dtype=torch.uint8, device="cuda")
    p.workspace_buffer, p.workspace_size = state[name].data_ptr(), state[name].numel()


def _backward_call(lib, abi, state):
    case = state["case"]
    m, n, k = state["sizes"]
    p = abi.GatedMmt4dBackwardParams()
    _tiles(p, m, n, k, case["m0"])
    for name in ("gate_pre", "up_pre", "out_grad"):
        _operand(p, name, state[name], p.N * p.M0 * p.N0)
    for name in ("lhs", "lhs_grad"):
        _operand(p, name, state[name], p.K * p.M0 * p.K0)
    for name in ("gate", "up", "gate_grad", "up_grad"):
        _operand(p, name, state[name], p.K * p.N0 * p.K0)
    p.flags = getattr(abi, "GATED_MMT4D_TYPE_" + _type_name(case)) | getattr(abi, "GATED_MMT4D_" + case["activation"].upper())
    if state["gate_pre"].dtype == torch.float32:
        p.flags |= abi.GATED_MMT4D_PRE_F32
    _workspace(state, "workspace", p, lib.iree_uk_mi355x_gated_mmt4d_backward_workspace)
    return lib.iree_uk_mi355x_gated_mmt4d_backward_p, p


def _adapter_call(lib, abi, state, prefix, lhs, out, m, n, k, out_type, accumulate):
    case = state["case"]
    p = abi.AdapterMmt4dParams()
    _tiles(p, m, n, k, case["m0"])
    _operand(p, "lhs", state[lhs], p.K * p.M0 * p.K0)
    _operand(p, "out", state[out], p.N * p.M0 * p.N0)
    p.rank, p.count = case["rank"], case["count"]
    _operand(p, "down", state[prefix + "down"], p.rank * k)
    _operand(p, "up", state[prefix + "to"], n * p.rank)
    p.down_stride1, p.up_stride1 = k, p.rank
    p.index_buffer, p.scales_buffer = state["index"].data_ptr(), state["scales"].data_ptr()
    p.flags = getattr(abi, "ADAPTER_MMT4D_TYPE_" + _type_name(case, out_type))
    if accumulate:
        p.flags |= abi.ADAPTER_MMT4D_ACCUMULATE
    _workspace(state, prefix + "workspace", p, lib.iree_uk_mi355x_adapter_mmt4d_workspace)
    return lib.iree_uk_mi355x_adapter_mmt4d_p, p


def _calls(lib, state):
    """The calls of one pass, their parameters filled in as a program does once for its buffers."""
    from iree_amd import abi
    case = state["case"]
    kind = case["kind"]
    m, n, k = state["sizes"]
    if kind == "adapters":
        calls = [_mmt4d_call(lib, abi, state, "lhs", "rhs", "out", m, n, k),
                 _adapter_call(lib, abi, state, "", "lhs", "out", m, n, k, case["out"], True)]
    elif kind == "block":
        calls = [_adapter_call(lib, abi, state, "gate_", "lhs", "gate_pre", m, n, k, "f32", False),
                 _adapter_call(lib, abi, state, "up_", "lhs", "up_pre", m, n, k, "f32", False),
                 _gated_call(lib, abi, state, "hidden"),
                 _mmt4d_call(lib, abi, state, "hidden", "last", "out", m, k, n),
                 _adapter_call(lib, abi, state, "last_", "hidden", "out", m, k, n, case["out"], True)]
    else:
        calls = [_gated_call(lib, abi, state, "out")] if kind != "backward" else []
        if kind != "gated":
            calls.append(_backward_call(lib, abi, state))
    return [(function, C.byref(p)) for function, p in calls]


def run(state):
    if not own:
        return _run_plain(state)
    from iree_amd import library
    lib = library.load()
    lib.iree_uk_mi355x_set_stream(torch.cuda.current_stream().cuda_stream, 1)
    if "calls" not in state:
        state["calls"] = _calls(lib, state)
    for function, params in state["calls"]:
        function(params)
    return _returned(state)


# In 64 bits -------------------------------------------------------------------------------


def _to_tiles(x, t0, t1):
    rows, cols = x.shape
    return x.reshape(rows, cols // t1, t1).unfold(0, t0, t0).permute(0, 1, 3, 2).reshape(-1) if t0 > 1 else x.reshape(-1)


def _exact_act(x, activation):
    """-> (act(x), its derivative)"""
    if activation == "gelu":  # 0.5 x (1 + tanh(..)), and its derivative by the product rule
        t = torch.tanh(_ROOT * (x + _CUBIC * x ** 3))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * _ROOT * (1 + 3 * _CUBIC * x ** 2)
    s, r = torch.sigmoid(x), torch.sigmoid(-x)
    if activation == "sigmoid":
        return s, s * r
    return x * s, s * (1 + x * r)


def _exact_adapters(x, index, down, up, scales):
    part = torch.zeros(x.shape[0], up.shape[1], dtype=torch.float64, device=x.device)
    for a in sorted(set(index.tolist()) - {-1}):
        rows = index == a
        part[rows] = scales[a].double() * (x[rows] @ down[a].double().t() @ up[a].double().t())
    return part


def exact(case, seed):
    made = _inputs(case, seed)
    kind, m0 = case["kind"], case["m0"]
    made = {name: v if name == "index" or v.dim() == 3 else v.double() for name, v in made.items()}
    x = made["lhs"]

    def adapters(prefix, of):
        return _exact_adapters(of, made["index"], made[prefix + "down"], made[prefix + "to"], made["scales"])

    if kind == "adapters":
        return {"out": (x @ made["rhs"].t() + adapters("", x)).reshape(-1)}
    gate, up = made["gate"], made["up"]
    if kind == "block":
        h = _exact_act(x @ gate.t() + adapters("gate_", x), case["activation"])[0] * (x @ up.t() + adapters("up_", x))
        return {"out": (h @ made["last"].t() + adapters("last_", h)).reshape(-1)}
    g, u = made.get("gate_pre", 0), made.get("up_pre", 0)
    if kind != "backward":
        g, u = g + x @ gate.t(), u + x @ up.t()
    value, slope = _exact_act(g, case["activation"])
    got = {}
    if kind != "backward":
        got["out"] = _to_tiles(value * u, m0, _N0)
        if case["pre"] == "store":
            got["gate_pre"], got["up_pre"] = _to_tiles(g, m0, _N0), _to_tiles(u, m0, _N0)
    if kind in ("backward", "train"):
        dg, du = made["out_grad"] * u * slope, made["out_grad"] * value
        got["lhs_grad"] = _to_tiles(dg @ gate + du @ up, m0, _K0)
        got["gate_grad"] = _to_tiles(dg.t() @ x, _N0, _K0)
        got["up_grad"] = _to_tiles(du.t() @ x, _N0, _K0)
    return got

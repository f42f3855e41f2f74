"""The measured work of the 8-bit operators: quantising rows, the norm that feeds a projection, the projection.

An 8-bit row is stored as e4m3 codes with one power-of-two scale per 32 of them (a byte, the exponent plus
127): the smallest scale that leaves every value of the block within the codes' largest, 448.  Rows are padded
with zero codes to a multiple of 128.  Sizes are those of the repository's encoders (768 and 1,024 wide, requests
of one to 1,024 tokens, batches of 65,536 rows) and generic odd ones between them.
"""
import math
import os
import sys

import torch

own = False

LARGEST = 448.0  # of the e4m3 codes
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}  # the library's element types
ACTIVATIONS = {"none": 0, "gelu": 1, "relu": 2, "geglu": 3, "swiglu": 4}
KINDS = {"layer": 0, "rms": 1}
EPS = 1e-5


def listed():
    return [
        # The norm in front of a projection, one token: latency alone.
        {"name": "norm_1", "op": "norm", "kind": "layer", "rows": 1, "width": 768, "branch": "f32", "splits": 2,
         "bias": True, "out32": False},
        # One 512-token request: the branch comes as the projection's two split-K partials.
        {"name": "norm_512_rms", "op": "norm", "kind": "rms", "rows": 512, "width": 1024, "branch": "f32", "splits": 2,
         "bias": False, "out32": False},
        # A ragged batch's rows in a post-norm encoder, where the normalised row is also the next residual.
        {"name": "norm_15088_post", "op": "norm", "kind": "layer", "rows": 15088, "width": 768, "branch": "f16",
         "splits": 1, "bias": True, "out32": True},
        # The largest batch, 64 x 1,024 tokens, with a 16-bit branch.
        {"name": "norm_65536_rms", "op": "norm", "kind": "rms", "rows": 65536, "width": 1024, "branch": "bf16",
         "splits": 1, "bias": False, "out32": False},
        # Rows of an odd width and number, quantised and read back.
        {"name": "quantize_5003x1000", "op": "quantize", "dtype": "f32", "rows": 5003, "width": 1000},
        # Attention rows of the largest batch on their way into the output projection.
        {"name": "quantize_65536x1024", "op": "quantize", "dtype": "f16", "rows": 65536, "width": 1024},
        # A single token's up projection: its time is the weights' way to the compute units.
        {"name": "linear_1_gelu", "op": "linear", "M": 1, "N": 4096, "K": 1024, "act": "gelu", "bias": True,
         "residual": "", "out": "f16"},
        # QKV projection of one short request (96 packed rows).
        {"name": "linear_96", "op": "linear", "M": 96, "N": 2304, "K": 768, "act": "none", "bias": True,
         "residual": "", "out": "bf16"},
        # Down projection of one 512-token request, added to its residual stream.
        {"name": "linear_512_add", "op": "linear", "M": 512, "N": 1024, "K": 4096, "act": "none", "bias": True,
         "residual": "f32", "out": "f32"},
        # A gated up projection over an odd number of rows.
        {"name": "linear_1571_swiglu", "op": "linear", "M": 1571, "N": 4352, "K": 1088, "act": "swiglu", "bias": False,
         "residual": "", "out": "bf16"},
        # FFN of the largest batch: up with its output in 8 bits, then down onto the residual stream.
        {"name": "linear_65536_up", "op": "linear", "M": 65536, "N": 4096, "K": 1024, "act": "gelu", "bias": True,
         "residual": "", "out": "e4m3"},
        {"name": "linear_65536_down", "op": "linear", "M": 65536, "N": 1024, "K": 4096, "act": "none", "bias": True,
         "residual": "f32", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear"])
    if op == "norm":
        width = rng.choice([768, 1024, rng.randint(64, 2048)])
        branch = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "kind": rng.choice(["layer", "rms"]), "rows": _log(rng, 1, (1 << 26) // width), "width": width,
                "branch": branch, "splits": rng.randint(1, 4) if branch == "f32" else 1,
                "bias": rng.random() < 0.5, "out32": rng.random() < 0.3}
    if op == "quantize":
        width = rng.choice([768, 1024, rng.randint(64, 4096)])
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": _log(rng, 1, (1 << 26) // width),
                "width": width}
    act = rng.choice(["none", "gelu", "relu", "geglu", "swiglu"])
    N, K = (rng.choice([768, 1024, 2304, 4096, _log(rng, 64, 4096)]) for _ in range(2))
    if act in ("geglu", "swiglu"):
        N = -(-N // 32) * 32
    return {"op": op, "M": _log(rng, 1, min((1 << 38) // (N * K), (1 << 28) // max(N, K))), "N": N, "K": K, "act": act,
            "bias": rng.random() < 0.5, "residual": rng.choice(["", "", "f32", "bf16"]),
            "out": rng.choice(["f32", "f16", "bf16", "e4m3"])}


def _padded(width):
    return -(-width // 128) * 128


def _scale_exponent(blocks):
    """Per block of the last axis: the smallest e with every magnitude at most 448 * 2^e, and at least -127."""
    part, power = torch.frexp(blocks.abs().amax(-1))  # amax = part * 2^power, part in [0.5, 1); 448 = 0.875 * 2^9
    e = power - 9 + (part > 0.875)
    return torch.where(part == 0, torch.full_like(e, -127), e.clamp(min=-127))


def _power(e):
    """2^e in fp32 from its bits (exp2 need not be exact); 0 for e = -127, the scale of blocks of zeros."""
    return ((e + 127) << 23).view(torch.float32)


def _quantized(x):
    """Rows of fp32 values as padded e4m3 codes [rows][padded] and scale bytes [rows][padded / 32]."""
    rows, width = x.shape
    blocks = torch.nn.functional.pad(x, (0, _padded(width) - width)).view(rows, -1, 32)
    e = _scale_exponent(blocks)
    codes = (blocks * _power(-e).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.view(rows, -1), (e + 127).to(torch.uint8)


def _values(codes, scales, width):
    """What 8-bit rows stand for, fp32."""
    rows = codes.shape[0]
    step = _power(scales.to(torch.int32) - 127)
    return (codes.float().view(rows, -1, 32) * step.unsqueeze(-1)).view(rows, -1)[:, :width]


def _features(case):
    return case["N"] // 2 if case["act"] in ("geglu", "swiglu") else case["N"]


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * std

    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if case["op"] == "linear":
        M, N, K, features = case["M"], case["N"], case["K"], _features(case)
        # Activations with a few large channels, as norms leave them.
        spread = torch.exp(normal(K, std=0.5))
        s["x"], s["xs"] = _quantized(normal(M, K) * spread)
        s["w"], s["ws"] = _quantized(normal(N, K, std=0.7 / math.sqrt(K)))
        s["bias"] = normal(N, std=0.1) if case["bias"] else None
        s["residual"] = normal(M, features).to(TYPES[case["residual"]]) if case["residual"] else None
        rows, width = M, features
        if case["out"] != "e4m3":
            s["out"] = torch.empty(M, features, dtype=TYPES[case["out"]], device=dev)
    elif case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["residual"] = normal(rows, width)
        s["branch"] = normal(case["splits"], rows, width, std=0.5).to(TYPES[case["branch"]])
        s["bias"] = normal(width, std=0.1) if case["bias"] else None
        s["gamma"] = 1.0 + normal(width, std=0.1)
        s["beta"] = normal(width, std=0.1) if case["kind"] == "layer" else None
        s["sum"] = torch.empty(rows, width, device=dev)
        s["out32"] = torch.empty(rows, width, device=dev) if case["out32"] else None
    else:
        rows, width = case["rows"], case["width"]
        s["x"] = (normal(rows, width) * torch.exp(normal(width, std=0.5))).to(TYPES[case["dtype"]])
    # The program's own buffers for 8-bit rows and for reading them back.
    if case["op"] != "linear" or case["out"] == "e4m3":
        s["codes"] = torch.empty(rows, _padded(width), dtype=torch.uint8, device=dev)
        s["scales"] = torch.empty(rows, _padded(width) // 32, dtype=torch.uint8, device=dev)
        s["values"] = torch.empty(rows, width, dtype=torch.bfloat16, device=dev)
    return s


def _activated(v, act):
    """The activation of fp32 columns; gated ones hold 16 gate columns and their 16 value columns in turn."""
    def gelu(t):
        return 0.5 * t * (1.0 + torch.erf(t * 0.7071067811865476))

    if act == "gelu":
        return gelu(v)
    if act == "relu":
        return torch.relu(v)
    if act in ("geglu", "swiglu"):
        groups = v.view(v.shape[0], -1, 2, 16)
        gate, value = groups[:, :, 0], groups[:, :, 1]
        gated = gelu(gate) if act == "geglu" else gate / (1.0 + torch.exp(-gate))
        return (gated * value).reshape(v.shape[0], -1)
    return v


def _plain(s):
    case = s["case"]
    if case["op"] == "linear":
        x, w = _values(s["x"], s["xs"], case["K"]), _values(s["w"], s["ws"], case["K"])
        v = torch.matmul(x, w.t())
        if s["bias"] is not None:
            v = v + s["bias"]
        v = _activated(v, case["act"])
        if s["residual"] is not None:
            v = v + s["residual"].float()
        if case["out"] == "e4m3":
            return {"values": _values(*_quantized(v), v.shape[1]).to(torch.bfloat16)}
        return {"out": v.to(TYPES[case["out"]])}
    if case["op"] == "quantize":
        return {"values": _values(*_quantized(s["x"].float()), case["width"]).to(torch.bfloat16)}
    branch = s["branch"].float().sum(0)
    if s["bias"] is not None:
        branch = branch + s["bias"]
    total = s["residual"] + branch
    v = total - total.mean(-1, keepdim=True) if case["kind"] == "layer" else total
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["gamma"]
    if s["beta"] is not None:
        v = v + s["beta"]
    got = {"sum": total, "values": _values(*_quantized(v), case["width"]).to(torch.bfloat16)}
    return {**got, "out32": v} if case["out32"] else got


_library = []


def _lib():
    if not _library:
        sys.path.insert(0, os.path.abspath("laya-cuda_amd"))
        from laya_cuda import _lib as binding
        _library.extend([binding.load(), binding.check])
    return _library


def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _own(s):
    lib, check = _lib()
    case, stream = s["case"], s["stream"]
    if case["op"] == "linear":
        eight = case["out"] == "e4m3"
        check(lib.laya_op_linear8(
            _at(s["x"]), _at(s["xs"]), _at(s["w"]), _at(s["ws"]), _at(s["bias"]), _at(s["residual"]),
            CODES[case["residual"] or "f32"], _at(s["codes"] if eight else s["out"]), _at(s["scales"]) if eight else None,
            CODES[case["out"]], ACTIVATIONS[case["act"]], case["M"], case["N"], case["K"], -1, stream))
        if not eight:
            return {"out": s["out"]}
        rows, width = case["M"], _features(case)
    else:
        rows, width = case["rows"], case["width"]
        if case["op"] == "norm":
            check(lib.laya_op_norm8(
                _at(s["residual"]), _at(s["branch"]), CODES[case["branch"]], case["splits"], rows * width, _at(s["bias"]),
                _at(s["gamma"]), _at(s["beta"]), EPS, KINDS[case["kind"]], _at(s["sum"]), _at(s["out32"]), _at(s["codes"]),
                _at(s["scales"]), rows, width, stream))
        else:
            check(lib.laya_op_quantize8(_at(s["x"]), CODES[case["dtype"]], width, _at(s["codes"]), _at(s["scales"]), rows,
                                        width, stream))
    # bf16 holds every code times its scale exactly.
    check(lib.laya_op_dequantize8(_at(s["codes"]), _at(s["scales"]), _at(s["values"]), CODES["bf16"], width, rows, width,
                                  stream))
    got = {"values": s["values"]}
    if case["op"] == "norm":
        got["sum"] = s["sum"]
        if case["out32"]:
            got["out32"] = s["out32"]
    return got


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "linear":
        M, N, K, features = case["M"], case["N"], case["K"], _features(case)
        out = 1 + 1 / 32 if case["out"] == "e4m3" else size[case["out"]]
        per_code = _padded(K) * (1 + 1 / 32)
        return {"bytes": (M + N) * per_code + M * features * (out + (size[case["residual"]] if case["residual"] else 0)),
                "flops": 2 * M * N * K}
    elements = case["rows"] * case["width"]
    if case["op"] == "quantize":  # the values, the codes there and back, the values that they stand for
        return {"bytes": elements * (size[case["dtype"]] + 2 * (1 + 1 / 32) + 2), "flops": 0}
    each = 4 + case["splits"] * size[case["branch"]] + 4 + 4 * case["out32"] + 1 + 1 / 32
    return {"bytes": elements * each + 4 * case["width"] * (1 + case["bias"] + (case["kind"] == "layer")), "flops": 0}


def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)  # pow(2, e) is not exact on every device


def _exact_values(codes, scales, width):
    """64-bit values of 8-bit rows, from the fields of the codes."""
    b = codes.view(torch.uint8).to(torch.int64)
    field, fraction = (b >> 3) & 15, (b & 7).double()
    magnitude = torch.where(field == 0, fraction * 2.0 ** -9, (1 + fraction / 8) * _exact_power(field - 7))
    signed = torch.where(b >= 128, -magnitude, magnitude)
    return (signed * _exact_power(scales.to(torch.int64) - 127).repeat_interleave(32, dim=1))[:, :width]


def _exact_quantized(x):
    """64-bit values rounded to what 8-bit rows can hold: multiples of the spacing at each value, ties to even."""
    rows, width = x.shape
    x = torch.cat([x, x.new_zeros(rows, _padded(width) - width)], 1).view(rows, -1, 32)
    top = x.abs().max(-1, keepdim=True).values
    e = torch.frexp(top).exponent - 9  # 448 * 2^e is at most top * 7 / 4, and over top / 8 * 7
    e = torch.where(top <= LARGEST * _exact_power(e), e, e + 1).clamp(min=-127)
    scale = _exact_power(e)
    y = x / scale
    spacing = _exact_power((torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    return (torch.round(y / spacing) * spacing * scale).view(rows, -1)[:, :width]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":  # nothing is computed before the rounding: the same values in any precision
        return {"values": _exact_quantized(s["x"].double())}
    if case["op"] == "linear":
        if case["out"] == "e4m3":
            # A product that lies at a border of its 8-bit rounding lands a whole step to either side by the last bit
            # of its 32-bit sum: what it is rounded to has no 64-bit value that a 32-bit sum could come near.
            return None
        v = torch.mm(_exact_values(s["x"], s["xs"], case["K"]), _exact_values(s["w"], s["ws"], case["K"]).t().contiguous())
        if case["bias"]:
            v += s["bias"].double()
        act = case["act"]
        if act in ("geglu", "swiglu"):
            columns = torch.arange(case["N"], device=v.device)
            g, v = v[:, columns % 32 < 16], v[:, columns % 32 >= 16]
            v = v * (g * torch.special.ndtr(g) if act == "geglu" else g * torch.sigmoid(g))
        elif act == "gelu":
            v = v * torch.special.ndtr(v)
        elif act == "relu":
            v = v.clamp(min=0)
        if case["residual"]:
            v = v + s["residual"].double()
        return {"out": v}
    total = s["residual"].double() + s["branch"].double().sum(0)
    if case["bias"]:
        total = total + s["bias"].double()
    got = {"sum": total, "values": None}  # rounded to 8 bits after 32-bit arithmetic: as above
    if case["out32"]:
        if case["kind"] == "layer":
            deviation, mean = torch.std_mean(total, -1, keepdim=True, correction=0)
            y = (total - mean) / torch.sqrt(deviation ** 2 + EPS)
        else:
            y = total / torch.sqrt((total ** 2).sum(-1, keepdim=True) / case["width"] + EPS)
        y = y * s["gamma"].double()
        got["out32"] = y + s["beta"].double() if case["kind"] == "layer" else y
    return got

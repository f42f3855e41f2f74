"""The measured work of rotary positions and of attention with masks, capped scores and distance biases.

Rotary positions turn pairs of a head's leading values by an angle, position times frequency; frequencies may be
scaled for contexts longer than the trained one.  Attention works on packed sequences: query i of a sequence of
Q queries and K keys stands at position i + K - Q, sees keys from `before` positions before its own to `after` behind it
(-1: no limit) that are in its document, and the sequence's prefix in any case.  Scores are scaled, capped (cap *
tanh(score / cap)), and get a bias that falls with distance or stands in a table by distance.  Sizes are those of the
repository's encoders (heads of 64, 12 or 16 of them, requests of up to 1,024 tokens, 65,536 rows in a batch) and generic
ones: heads of 32 to 256, fewer key heads than query heads, long caches read by single tokens.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # the library's element types
LAYOUTS = {"half": 0, "interleaved": 1}
TRAINED = 8192  # positions that the scaled frequencies were trained on


def _rotary(name, **values):
    return {"name": name, "op": "rotary", "amplitude": 1.0, "scaling": "none", "direction": 1, "far": 1024, **values}


def _attend(name, **values):
    return {"name": name, "op": "attend", "cap": 0.0, "bias": "none", "span": 0, "before": -1, "after": -1,
            "prefix": False, "documents": 0, "ragged": False, **values}


def listed():
    return [
        # One token's queries and keys on their way into a cache: latency alone.
        _rotary("rotary_1", dtype="f16", rows=1, heads=24, dim=64, rotated=64, layout="half"),
        # An odd number of rows, positions far past the trained ones, the first 32 of each head's 80 values, and the
        # gradient's direction.
        _rotary("rotary_5003_part", dtype="f32", rows=5003, heads=12, dim=80, rotated=32, layout="interleaved",
                scaling="linear", far=1000003, direction=-1),
        # The largest batch, 64 x 1,024 tokens, queries and keys of 16 heads in one call.
        _rotary("rotary_65536", dtype="bf16", rows=65536, heads=32, dim=64, rotated=64, layout="half"),
        # One long context with frequencies scaled by parts.
        _rotary("rotary_131072_parts", dtype="bf16", rows=131072, heads=10, dim=128, rotated=128, layout="half",
                scaling="parts", amplitude=1.139, far=131072),
        # A single token over a short context: latency alone.
        _attend("step_1x500", dtype="f16", seqs=1, queries=1, keys=500, heads=12, kv_heads=12, dim=64, bias="slopes", after=0),
        # A batch of single tokens whose contexts differ, every head with keys of its own.
        _attend("step_48_ragged", dtype="f16", seqs=48, queries=1, keys=4100, ragged=True, heads=16, kv_heads=16, dim=64,
                bias="slopes", after=0),
        # Single tokens over very long caches that four query heads share: the caches' bytes are the time.
        _attend("step_4x131072", dtype="bf16", seqs=4, queries=1, keys=131072, heads=32, kv_heads=8, dim=128, cap=50.0,
                after=0),
        # One 512-token request with capped scores: few rows, every key seen.
        _attend("prompt_512_cap", dtype="f16", seqs=1, queries=512, keys=512, heads=12, kv_heads=12, dim=64, cap=30.0),
        # Ragged requests with a learned bias by distance, 32 of up to 1,024 tokens.
        _attend("prompt_ragged_table", dtype="bf16", seqs=32, queries=1024, keys=1024, ragged=True, heads=12, kv_heads=12,
                dim=64, bias="table", span=128),
        # The largest batch: each sequence holds a shared state and documents that see it and themselves.
        _attend("prompt_65536_documents", dtype="bf16", seqs=64, queries=1024, keys=1024, heads=16, kv_heads=16, dim=64,
                bias="slopes", prefix=True, documents=200),
        # Odd sizes: a later piece of a prompt, heads of 80, a window, capped.
        _attend("prompt_1571_window", dtype="f16", seqs=3, queries=1571, keys=4099, heads=10, kv_heads=5, dim=80, cap=20.0,
                before=700, after=0),
        # One long causal prompt.
        _attend("prompt_16384", dtype="bf16", seqs=1, queries=16384, keys=16384, heads=8, kv_heads=2, dim=128, after=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "step", "prompt", "prompt"])
    if kind == "rotary":
        dim = rng.choice([64, 80, 128, 2 * rng.randint(16, 128)])
        heads = rng.randint(1, 40)
        return _rotary("", dtype=rng.choice(["f32", "f16", "bf16"]), rows=_log(rng, 1, (1 << 27) // (heads * dim)), heads=heads,
                       dim=dim, rotated=rng.choice([dim, 2 * rng.randint(1, dim // 2)]),
                       layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "base", "parts"]),
                       amplitude=rng.choice([1.0, 1.139]), far=_log(rng, 16, 2000000), direction=rng.choice([1, -1]))
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16, rng.randint(1, 16)])
    common = {"dtype": rng.choice(["f16", "bf16"]), "kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 1, 2, 4, 7]),
              "dim": rng.choice([64, 64, 128, 8 * rng.randint(4, 32)]), "cap": rng.choice([0.0, 0.0, 20.0, 50.0]),
              "bias": rng.choice(["none", "slopes", "table"]), "span": rng.choice([32, 128, rng.randint(1, 1000)]),
              "ragged": rng.random() < 0.5}
    width = common["heads"] * common["dim"]
    if kind == "step":
        seqs = _log(rng, 1, 64)
        queries = rng.choice([1, 1, 1, rng.randint(2, 8)])
        keys = _log(rng, queries, max(64, (1 << 28) // (seqs * queries * width)))
        return _attend("", seqs=seqs, queries=queries, keys=keys, after=0, before=rng.choice([-1, -1, _log(rng, 16, 4096)]),
                       prefix=rng.random() < 0.3, **common)
    keys = _log(rng, 1, 6000)
    queries = keys if rng.random() < 0.7 else rng.randint(1, keys)
    seqs = _log(rng, 1, max(1, min(64, (1 << 36) // (queries * keys * width))))
    masked = rng.random() < 0.5
    return _attend("", seqs=seqs, queries=queries, keys=keys, after=rng.choice([-1, 0, 0, rng.randint(0, 200)]),
                   before=rng.choice([-1, -1, _log(rng, 8, 4096)]), prefix=masked,
                   documents=_log(rng, 8, 500) if masked and queries == keys else 0, **common)


def _lengths(case):
    """Queries and keys of each sequence, the same for every seed: spread from a tenth of the largest to it."""
    n = case["seqs"]
    part = 0.1 + 0.9 * (np.arange(1, n + 1) * 0.6180339887 % 1.0) if case["ragged"] else np.ones(n)
    part[0] = 1.0
    keys = np.maximum(1, (part * case["keys"]).astype(np.int64))
    queries = np.maximum(1, (part * case["queries"]).astype(np.int64)) if case["queries"] > 8 else np.full(n, case["queries"])
    return np.minimum(queries, keys), keys


def _documents(case, keys):
    """The document of each key of each sequence [seqs][largest], lengths between half and one and a half of the mean."""
    edges = np.cumsum((case["documents"] * (0.5 + np.arange(1, 4 * case["keys"] // case["documents"] + 8) * 0.7548776662 % 1.0)).astype(np.int64) + 1)
    shift = np.arange(len(keys)) * 37 % case["documents"]
    return np.searchsorted(edges, np.arange(case["keys"])[None, :] + shift[:, None], side="right")


def _prefixes(case, keys):
    return np.maximum(1, keys // 8)


def _frequencies(case):
    """Radians a position, in 64 bits."""
    rotated, base, factor = case["rotated"], 10000.0, 8.0
    if case["scaling"] == "base":  # a larger base: the slowest pair reaches `factor` times as far, the fastest stays
        base *= factor ** (rotated / (rotated - 2.0)) if rotated > 2 else factor
    f = base ** (-np.arange(0, rotated, 2, dtype=np.float64) / rotated)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "parts":  # pairs of more than 32 turns over the trained positions stay, of less than 1 slow down
        kept = np.clip((TRAINED * f / (2 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        f = f * kept + f / factor * (1.0 - kept)
    return f


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * std

    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    kind = TYPES[case["dtype"]]
    if case["op"] == "rotary":
        rows, heads, dim = case["rows"], case["heads"], case["dim"]
        # The values' heads lie behind the queries' and keys' in a row of the projection, and are not turned.
        s["x"] = normal(rows, heads + max(1, heads // 2), dim).to(kind)
        s["positions"] = torch.randint(0, case["far"], (rows,), generator=gen, device=dev, dtype=torch.int32)
        s["turns"] = torch.from_numpy(_frequencies(case) / (2 * math.pi)).to(dev)
        s["out"] = torch.empty(rows, heads, dim, dtype=kind, device=dev)
        return s
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    queries, keys = _lengths(case)
    n, step = len(keys), case["queries"] <= 8 < case["keys"]
    q_rows = int(queries.sum())
    q_starts = np.cumsum(queries) - queries
    if case["queries"] == case["keys"] and not step:  # rows of one projection: queries, keys, values
        packed = normal(q_rows, heads + 2 * kv_heads, dim)
        packed[:, :heads + kv_heads] *= 1.5
        packed = packed.to(kind)
        s["q"], s["k"], s["v"] = packed.split([heads, kv_heads, kv_heads], 1)
        k_starts = q_starts
    else:  # caches with room for the longest context of the batch
        k_starts = np.arange(n) * case["keys"]
        s["q"] = normal(q_rows, heads, dim, std=1.5).to(kind)
        s["k"] = torch.randn(n * case["keys"], kv_heads, dim, generator=gen, device=dev, dtype=kind).mul_(1.5)
        s["v"] = torch.randn(n * case["keys"], kv_heads, dim, generator=gen, device=dev, dtype=kind)
    for name, host in (("q_starts", q_starts), ("q_lengths", queries), ("k_starts", k_starts), ("k_lengths", keys)):
        s[name] = torch.from_numpy(host.astype(np.int32)).to(dev)
    s["prefix"] = torch.from_numpy(_prefixes(case, keys).astype(np.int32)).to(dev) if case["prefix"] else None
    s["documents"] = s["bounds"] = None
    if case["documents"]:
        ids = _documents(case, keys)
        s["documents"] = torch.from_numpy(np.concatenate([ids[i, :keys[i]] for i in range(n)]).astype(np.int32)).to(dev)
        s["bounds"] = torch.empty(q_rows, 2, dtype=torch.int32, device=dev)
    s["slopes"] = s["table"] = None
    if case["bias"] == "slopes":
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device=dev) / heads) * torch.exp(normal(heads, std=0.05))
    if case["bias"] == "table":
        s["table"] = normal(heads, 2 * case["span"] + 1)
    s["out"] = torch.empty(q_rows, heads, dim, dtype=kind, device=dev)
    return s


def _plain_rotary(s):
    case = s["case"]
    heads, r = case["heads"], case["rotated"]
    turn = s["positions"].double()[:, None] * s["turns"]
    angle = (turn - torch.floor(turn)) * (2 * math.pi * case["direction"])
    c, sn = (t.float()[:, None] * case["amplitude"] for t in (torch.cos(angle), torch.sin(angle)))
    x = s["x"][:, :heads].float()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if case["layout"] == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    p, q = a * c - b * sn, a * sn + b * c
    turned = torch.cat([p, q], -1) if case["layout"] == "half" else torch.stack([p, q], -1).flatten(-2)
    return {"out": torch.cat([turned, x[..., r:]], -1).to(TYPES[case["dtype"]])}


def _visible(s, case, position, key):
    """[seqs][queries][keys]: which keys a query at its position sees."""
    lengths = s["k_lengths"].long()[:, None, None]
    see = key < lengths
    near = torch.ones_like(see)
    if case["before"] >= 0:
        near = near & (key >= position - case["before"])
    if case["after"] >= 0:
        near = near & (key <= position + case["after"])
    if s["documents"] is not None:
        row = (s["k_starts"].long()[:, None] + torch.arange(case["keys"], device=see.device)).clamp(max=s["documents"].shape[0] - 1)
        ids = s["documents"][row]
        near = near & (ids[:, :, None] == ids[:, None, :])
    if s["prefix"] is not None:
        near = near | (key < s["prefix"].long()[:, None, None])
    return see & near


def _plain_attend(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, dev = heads // kv_heads, s["q"].device
    n, most_q, most_k = case["seqs"], case["queries"], case["keys"]
    q_lengths, k_lengths = s["q_lengths"].long(), s["k_lengths"].long()
    qi, ki = torch.arange(most_q, device=dev), torch.arange(most_k, device=dev)
    q_row = (s["q_starts"].long()[:, None] + qi).clamp(max=s["q"].shape[0] - 1)
    k_row = (s["k_starts"].long()[:, None] + ki).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][q_row].float().view(n, most_q, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * most_q, dim)
    k = s["k"][k_row].float().permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(n, kv_heads, group, most_q, most_k)
    if case["cap"]:
        scores = torch.tanh(scores.div_(case["cap"])).mul_(case["cap"])
    position = (qi + (k_lengths - q_lengths)[:, None])[:, :, None]  # [seqs][queries][1]
    distance = ki - position
    if s["slopes"] is not None:
        scores -= s["slopes"].view(1, kv_heads, group, 1, 1) * distance.abs()[:, None, None]
    if s["table"] is not None:
        at = distance.clamp(-case["span"], case["span"]) + case["span"]
        scores += s["table"][:, at].view(kv_heads, group, n, most_q, most_k).permute(2, 0, 1, 3, 4)
    scores = scores.masked_fill_(~_visible(s, case, position, ki)[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    weights = scores.div_(torch.where(total == 0, torch.ones_like(total), total)).view(n, kv_heads, group * most_q, most_k)
    v = s["v"][k_row].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(weights, v).view(n, kv_heads, group, most_q, dim).permute(0, 3, 1, 2, 4).reshape(n * most_q, heads, dim)
    row = torch.arange(s["q"].shape[0], device=dev)
    seq = torch.searchsorted(s["q_starts"].long(), row, right=True) - 1
    return {"out": out[seq * most_q + row - s["q_starts"].long()[seq]].to(TYPES[case["dtype"]])}


_library = []


def _lib():
    if not _library:
        sys.path.insert(0, os.path.abspath("laya-cuda_amd"))
        from laya_cuda import _lib as binding
        _library.append(binding)
        binding.load()
    return _library[0]


def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _call(s):
    """The call's description and workspace, which a program keeps as long as its buffers and sizes stay."""
    if "call" not in s:
        case, binding = s["case"], _lib()
        a = binding.LayaAttend(
            struct_bytes=ctypes.sizeof(binding.LayaAttend), dtype=CODES[case["dtype"]], heads=case["heads"],
            kv_heads=case["kv_heads"], dim=case["dim"], n_seq=case["seqs"], max_q=case["queries"], max_k=case["keys"],
            q_rows=s["q"].shape[0], k_rows=s["k"].shape[0], scale=1.0 / math.sqrt(case["dim"]), cap=case["cap"],
            before=case["before"], after=case["after"], span=case["span"] if case["bias"] == "table" else 0)
        for name in ("q", "k", "v", "out"):
            setattr(a, name, s[name].data_ptr())
            setattr(a, name + "_row", s[name].stride(0))
            setattr(a, name + "_head", s[name].stride(1))
        for name in ("q_starts", "q_lengths", "k_starts", "k_lengths", "prefix", "bounds", "slopes", "table"):
            setattr(a, name, _at(s[name]))
        size = binding.load().laya_attend_workspace(ctypes.byref(a))
        s["call"], s["workspace"] = a, torch.empty(max(size, 1), dtype=torch.uint8, device=s["q"].device)
    return s["call"], s["workspace"]


def _own(s):
    binding, case = _lib(), s["case"]
    lib = binding.load()
    if case["op"] == "rotary":
        binding.check(lib.laya_op_rotary(
            _at(s["x"]), s["x"].stride(0), s["x"].stride(1), _at(s["out"]), s["out"].stride(0), s["out"].stride(1),
            CODES[case["dtype"]], _at(s["positions"]), _at(s["turns"]), case["amplitude"], LAYOUTS[case["layout"]],
            case["direction"], case["rows"], case["heads"], case["dim"], case["rotated"], s["stream"]))
        return {"out": s["out"]}
    call, workspace = _call(s)
    if s["documents"] is not None:
        binding.check(lib.laya_op_document_bounds(
            _at(s["documents"]), _at(s["q_starts"]), _at(s["q_lengths"]), case["seqs"], s["q"].shape[0], case["queries"],
            _at(s["bounds"]), s["stream"]))
    binding.check(lib.laya_op_attend(ctypes.byref(call), _at(workspace), workspace.numel(), s["stream"]))
    return {"out": s["out"]}


def run(state):
    if own:
        return _own(state)
    return _plain_rotary(state) if state["case"]["op"] == "rotary" else _plain_attend(state)


def _pairs(case):
    """Query-key pairs that the masks leave, over all sequences."""
    queries, keys = _lengths(case)
    total = 0
    for i, (nq, nk) in enumerate(zip(queries, keys)):
        p = np.arange(nq) + nk - nq
        lo = np.maximum(0, p - case["before"]) if case["before"] >= 0 else np.zeros(nq, np.int64)
        hi = np.minimum(nk, p + case["after"] + 1) if case["after"] >= 0 else np.full(nq, nk)
        if case["documents"]:
            ids = _documents(case, keys)[i, :nk]
            lo = np.maximum(lo, np.searchsorted(ids, ids, side="left"))
            hi = np.minimum(hi, np.searchsorted(ids, ids, side="right"))
        first = _prefixes(case, keys)[i] if case["prefix"] else 0
        total += int(np.minimum(first, nk) * nq + np.maximum(0, hi - np.maximum(lo, first)).sum())
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        elements = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * elements * size + 4 * case["rows"], "flops": 3 * case["rows"] * case["heads"] * case["rotated"]}
    queries, keys = _lengths(case)
    # A window leaves the keys before it unread.
    read = np.minimum(keys, queries + case["before"] + (_prefixes(case, keys) if case["prefix"] else 0)) if case["before"] >= 0 else keys
    return {"bytes": size * case["dim"] * int(2 * case["heads"] * queries.sum() + 2 * case["kv_heads"] * read.sum()),
            "flops": 4 * _pairs(case) * case["heads"] * case["dim"]}


def exact(case, seed):
    """The definition in 64 bits: one sequence and one key head at a time."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        r, x = case["rotated"], s["x"][:, :case["heads"]].double()
        theta = torch.from_numpy(_frequencies(case)).to(x.device) * s["positions"].double().unsqueeze(1) * case["direction"]
        index = torch.arange(r // 2, device=x.device)
        first, second = (index, index + r // 2) if case["layout"] == "half" else (2 * index, 2 * index + 1)
        z = torch.complex(x[:, :, first], x[:, :, second]) * torch.polar(torch.full_like(theta, case["amplitude"]), theta).unsqueeze(1)
        x[:, :, first], x[:, :, second] = z.real, z.imag
        return {"out": x}
    queries, keys = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    q_at = 0
    for i, (nq, nk) in enumerate(zip(queries.tolist(), keys.tolist())):
        k_at = int(s["k_starts"][i])
        j = torch.arange(nk, device=out.device).unsqueeze(0)
        p = torch.arange(nk - nq, nk, device=out.device).unsqueeze(1)
        hidden = torch.zeros(nq, nk, dtype=torch.bool, device=out.device)
        if case["before"] >= 0:
            hidden |= p - j > case["before"]
        if case["after"] >= 0:
            hidden |= j - p > case["after"]
        if case["documents"]:
            ids = s["documents"][k_at:k_at + nk]
            hidden |= ids[nk - nq:].unsqueeze(1) != ids.unsqueeze(0)
        if case["prefix"]:
            hidden[:, :int(s["prefix"][i])] = False
        for h in range(case["heads"]):
            kv = h // group
            t = s["q"][q_at:q_at + nq, h].double() @ s["k"][k_at:k_at + nk, kv].double().t().contiguous() / math.sqrt(case["dim"])
            if case["cap"]:
                t = case["cap"] * torch.tanh(t / case["cap"])
            if case["bias"] == "slopes":
                t -= s["slopes"][h].double() * (j - p).abs()
            if case["bias"] == "table":
                t += s["table"][h].double()[torch.clamp(j - p, -case["span"], case["span"]) + case["span"]]
            t[hidden] = -math.inf
            t = torch.nan_to_num(torch.softmax(t, -1), nan=0.0)
            out[q_at:q_at + nq, h] = t @ s["v"][k_at:k_at + nk, kv].double().contiguous()
        q_at += nq
    return {"out": out}

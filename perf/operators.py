"""Products of many tokens with quantized weights, the same grouped by expert, and the routing around them, as cases that can be
timed and compared: what each case stands for is said at `listed()`; `draw()` gives further cases of the same ranges.

A case is a dict of plain values.  `prepare()` makes what a program holds before the call, `run()` makes one pass: where `own` is
false by elementary torch operations in 32 bits, where it is true by the public entry points of `cubek_amd`.  `exact()` gives
the results in 64 bits.

A weight is the value that dequantize stores for the type of x, F(F(scale) * code): that rounding belongs to what the codes stand for,
in the plain form and in 64 bits alike.
"""
import math

import torch

own = False

_TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
_BYTES = {"F32": 4, "F16": 2, "BF16": 2}
_BITS = {"Q8S": 8, "E4M3": 8, "Q4S": 4, "E2M1": 4, "Q2S": 2}
_MOST = {"Q8S": 127.0, "E4M3": 448.0, "Q4S": 7.0, "E2M1": 6.0, "Q2S": 1.0}


def listed():
    return [
        # one token of decoding: an attention output projection with its residual, the smallest product there is
        dict(name="decode_residual", kind="matmul", tokens=1, rows=4096, cols=4096, elem="BF16", out="BF16", value="Q4S", store="U32",
             param="F32", block=32, block_rows=1, bias=False, activation="identity", gated=False, residual=True),
        # a decode step of 24 sequences over gate and up projections at once, groups of 128 with f16 scales
        dict(name="decode_gated", kind="matmul", tokens=24, rows=14336, cols=4096, elem="F16", out="F16", value="Q4S", store="U32",
             param="F16", block=128, block_rows=1, bias=False, activation="silu", gated=True, residual=False),
        # a ragged prompt through a down projection of fp8 bytes with a scale per 128 x 128 block, bias and residual
        dict(name="prompt_down", kind="matmul", tokens=509, rows=4096, cols=14336, elem="BF16", out="BF16", value="E4M3", store="Native",
             param="F32", block=128, block_rows=128, bias=True, activation="identity", gated=False, residual=True),
        # a long prompt through the largest weight of the benchmark (configuration 5: 4-bit e2m1 codes, blocks of 32)
        dict(name="prompt_largest", kind="matmul", tokens=4096, rows=28672, cols=8192, elem="BF16", out="BF16", value="E2M1", store="U32",
             param="F32", block=32, block_rows=1, bias=True, activation="gelu", gated=False, residual=False),
        # a decode step of 16 sequences through eight experts, two each: gate and up projections
        dict(name="experts_decode", kind="experts", tokens=16, experts=8, chosen=2, gather=True, rows=14336, cols=4096, elem="BF16",
             out="BF16", value="Q4S", store="U32", param="F32", block=32, block_rows=1, bias=False, activation="silu", gated=True),
        # one token through two of eight experts: the down projections, results in 32 bits for the weighted sum that follows
        dict(name="experts_one_token", kind="experts", tokens=1, experts=8, chosen=2, gather=False, rows=4096, cols=14336, elem="BF16",
             out="F32", value="Q4S", store="U32", param="F32", block=32, block_rows=1, bias=False, activation="identity", gated=False),
        # a ragged prompt through many small experts of 8 bits: gate and up projections, some experts with hardly a token
        dict(name="experts_many", kind="experts", tokens=1021, experts=64, chosen=6, gather=True, rows=1408, cols=2048, elem="F16",
             out="F16", value="Q8S", store="U32", param="F16", block=32, block_rows=1, bias=True, activation="silu", gated=True),
        # a long prompt through the down projections of eight experts
        dict(name="experts_prompt", kind="experts", tokens=4096, experts=8, chosen=2, gather=False, rows=4096, cols=14336, elem="BF16",
             out="BF16", value="Q4S", store="U32", param="F32", block=64, block_rows=1, bias=False, activation="identity", gated=False),
        # the choice of two of eight experts for a decode step of 16 sequences
        dict(name="route_decode", kind="route", tokens=16, experts=8, chosen=2, elem="F32", score="softmax", normalize=True),
        # the choice of eight of 128 experts for a long prompt of odd length
        dict(name="route_prompt", kind="route", tokens=16381, experts=128, chosen=8, elem="BF16", score="softmax", normalize=True),
        # the weighted sum of two experts' results for a decode step, with the residual
        dict(name="combine_decode", kind="combine", tokens=16, chosen=2, rows=4096, elem="F32", out="BF16", residual=True),
        # the weighted sum of eight experts' results for a long prompt
        dict(name="combine_prompt", kind="combine", tokens=8191, chosen=8, rows=2048, elem="BF16", out="BF16", residual=True),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    cases = listed()
    flops, moved = max(work(c)["flops"] for c in cases), max(work(c)["bytes"] for c in cases)
    while True:
        case = _draw_one(rng)
        w = work(case)
        if w["flops"] <= flops and w["bytes"] <= moved and 3072 not in case.values():
            return case


def _draw_one(rng):
    kind = rng.choice(["matmul", "matmul", "matmul", "experts", "experts", "experts", "route", "combine"])
    if kind == "route":
        experts = rng.choice([4, 8, 16, 40, 60, 64, 128, 160, 256, 512])
        return dict(kind=kind, tokens=_between(rng, 1, 32768), experts=experts, chosen=rng.randint(1, min(8, experts)),
                    elem=rng.choice(["F32", "BF16", "F16"]), score=rng.choice(["softmax", "softmax", "sigmoid"]), normalize=rng.choice([True, False]))
    if kind == "combine":
        return dict(kind=kind, tokens=_between(rng, 1, 8192), chosen=rng.randint(1, 8), rows=_between(rng, 256, 8192),
                    elem=rng.choice(["F32", "BF16", "F16"]), out=rng.choice(["F32", "BF16", "F16"]), residual=rng.choice([True, False]))
    elem = rng.choice(["BF16", "BF16", "F16"])
    value, store, block, block_rows = rng.choice([
        ("Q4S", "U32", 32, 1), ("Q4S", "U32", 64, 1), ("Q4S", "U32", 128, 1), ("Q8S", "U32", 32, 1), ("Q8S", "Native", 64, 1), ("Q2S", "U32", 64, 1),
        ("E2M1", "U32", 32, 1), ("E2M1", "Native", 32, 1), ("E4M3", "Native", 128, 128), ("Q8S", "U32", 0, 0)])
    unit = max(block, 32)
    gated = rng.choice([True, False, False])
    common = dict(elem=elem, out=rng.choice([elem, elem, "F32"]), value=value, store=store, param=rng.choice(["F32", elem]), block=block,
                  block_rows=block_rows, bias=rng.choice([True, False]), gated=gated,
                  activation=rng.choice(["silu", "gelu"]) if gated else rng.choice(["identity", "identity", "relu", "silu", "gelu"]))
    step = max(1, block_rows)
    if kind == "matmul":
        return dict(kind=kind, tokens=_between(rng, 1, 8192), rows=step * _between(rng, 256 // step, 28672 // step),
                    cols=unit * _between(rng, 512 // unit, 28672 // unit), residual=rng.choice([True, False]), **common)
    experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
    return dict(kind=kind, tokens=_between(rng, 1, 4096), experts=experts, chosen=rng.randint(1, min(8, experts)), gather=rng.choice([True, False]),
                rows=step * _between(rng, 256 // step, 14336 // step), cols=unit * _between(rng, 256 // unit, 14336 // unit), **common)


# ---- inputs ----------------------------------------------------------------------------------------------------------------


def _encode(w, case):
    """The codes and scales of floats [rows, cols], the way a weight is quantized: scale = absmax / most of a block, codes rounded."""
    rows, cols = w.shape
    value, block, high = case["value"], case["block"], max(1, case["block_rows"])
    param = _TORCH[case["param"]]
    if block:
        v = w.view(rows // high, high, cols // block, block)
        scale = (v.abs().amax((1, 3), keepdim=True) / _MOST[value]).clamp_(min=1e-8).to(param)
        q = (v / scale.float()).view(rows, cols)
        scale = scale.view(rows // high, cols // block)
    else:  # one scale, the same for every slice of rows that is encoded
        scale = torch.full((1,), 0.11 / _MOST[value], device=w.device).to(param)
        q = w / scale.float()
    q = q.round_().clamp_(-_MOST[value], _MOST[value])
    if value == "E4M3":
        return q.to(torch.float8_e4m3fn).view(torch.uint8), scale
    if value == "E2M1" and case["store"] == "Native":  # nibbles: 0, 1, 2, 3, 4, 6 are codes 0, 2, 4, 5, 6, 7
        q = torch.where(q.abs() == 5.0, 4.0 * q.sign(), q)
        code = torch.tensor([0, 2, 4, 5, 6, 0, 7], device=w.device)[q.abs().int()] | ((q < 0).int() << 3)
        return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), scale
    if case["store"] == "Native":
        return q.to(torch.int8).view(torch.uint8), scale
    bits = _BITS[value]
    fields = (q.int() & ((1 << bits) - 1)).view(rows, -1, 32 // bits)
    words = fields[..., 0].clone()
    for i in range(1, 32 // bits):
        words |= fields[..., i] << (i * bits)
    return words, scale


def _weights(gen, case, rows):
    """Stored tensors of a weight [rows, cols] of normally distributed floats, quantized some rows at a time."""
    step = max(1, (1 << 26) // case["cols"] // 128) * 128
    parts = [_encode(torch.randn((min(step, rows - r), case["cols"]), generator=gen, device="cuda") * 0.02, case) for r in range(0, rows, step)]
    if len(parts) == 1:
        return parts[0]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]) if case["block"] else parts[0][1]


def _activations(gen, shape, dtype):
    """Normal values, one channel in a hundred six times as large."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.where(torch.rand(shape[-1:], generator=gen, device="cuda") < 0.01, 6.0, 1.0)
    return x.to(dtype)


def _logits(gen, tokens, experts, dtype):
    """A router's logits: some experts are asked for more than others."""
    return (torch.randn((tokens, experts), generator=gen, device="cuda") + 0.7 * torch.randn((experts,), generator=gen, device="cuda")).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, t, s = case["kind"], case["tokens"], {"case": case}
    if kind == "route":
        s["logits"] = _logits(gen, t, case["experts"], _TORCH[case["elem"]])
        return s
    k = case.get("chosen", 1)
    if kind == "combine":
        s["h"] = torch.randn((t * k, case["rows"]), generator=gen, device="cuda").to(_TORCH[case["elem"]])
        s["slots"] = torch.randperm(t * k, generator=gen, device="cuda").view(t, k).int()
        s["weights"] = torch.softmax(torch.randn((t, k), generator=gen, device="cuda"), -1)
        if case["residual"]:
            s["residual"] = torch.randn((t, case["rows"]), generator=gen, device="cuda").to(_TORCH[case["out"]])
        return s
    wide = case["rows"] * (2 if case["gated"] else 1)
    if kind == "matmul":
        s["codes"], s["scales"] = _weights(gen, case, wide)
        s["x"] = _activations(gen, (t, case["cols"]), _TORCH[case["elem"]])
        bias = (wide,)
        if case["residual"]:
            s["residual"] = torch.randn((t, case["rows"]), generator=gen, device="cuda").to(_TORCH[case["out"]])
    else:
        e = case["experts"]
        codes, scales = _weights(gen, case, e * wide)
        s["codes"] = codes.view(e, wide, -1)
        s["scales"] = scales.view(e, -1, scales.shape[-1]) if case["block"] else scales
        picked = _logits(gen, t, e, torch.float32).topk(k, dim=-1).indices.flatten()
        order = torch.argsort(picked, stable=True)  # positions by expert, then by token
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.bincount(picked, minlength=e).cumsum(0)]).int()
        if case["gather"]:
            s["row_of"] = (order // k).int()
        s["x"] = _activations(gen, (t if case["gather"] else t * k, case["cols"]), _TORCH[case["elem"]])
        bias = (e, wide)
    if case["bias"]:
        s["bias"] = (torch.randn(bias, generator=gen, device="cuda") * 0.1).to(_TORCH[case["elem"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    return _hold(s) if own else s


# ---- the framework's calls -------------------------------------------------------------------------------------------------


def _hold(s):
    """What a program keeps beside its tensors: handles, the scheme, result tensors and workspaces."""
    from cubek_amd import (Activation, ComputeClient, ElemType, Epilogue, QuantLevel, QuantParam, QuantScheme, QuantStore, QuantValue, Score,
                           TensorHandleRef, experts, matmul, routing)
    case = s["case"]
    h = TensorHandleRef.from_torch
    client, kind, t = ComputeClient.current(), case["kind"], case["tokens"]
    elem, k = ElemType[case["elem"]], case.get("chosen", 1)
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")
    if kind == "route":
        e = case["experts"]
        out = (empty((t, k), torch.float32), empty((t, k), torch.int32), empty((e + 1,), torch.int32), empty((t * k,), torch.int32), empty((t, k), torch.int32))
        size = routing.workspace_bytes(t, e, k)
        space = empty((max(size, 16),), torch.uint8)
        handles = [h(v) for v in (s["logits"],) + out]
        score = Score.Softmax if case["score"] == "softmax" else Score.Sigmoid
        normalize = case["normalize"]

        def call():
            routing.launch_ref(client, *handles, elem, score, normalize, workspace=space.data_ptr(), workspace_size=size)
            return out
        s["call"] = call
        return s
    y_elem = ElemType[case["out"]]
    residual = h(s["residual"]) if "residual" in s else None
    if kind == "combine":
        y = empty((t, case["rows"]), _TORCH[case["out"]])
        hh, slots, weights, hy = h(s["h"]), h(s["slots"]), h(s["weights"]), h(y)

        def call():
            routing.combine(client, hh, slots, weights, hy, elem, y_elem, residual)
            return y
        s["call"] = call
        return s
    level = QuantLevel.Tensor if not case["block"] else QuantLevel.block([case["block_rows"], case["block"]] if case["block_rows"] > 1 else [case["block"]])
    scheme = (QuantScheme.default().with_value(QuantValue[case["value"]]).with_store(QuantStore[case["store"]]).with_param(QuantParam[case["param"]])
              .with_level(level))
    epilogue = Epilogue(Activation[case["activation"].capitalize()], gated=case["gated"], bias=h(s["bias"]) if "bias" in s else None, residual=residual)
    y = empty((t * k, case["rows"]), _TORCH[case["out"]])
    codes, scales, x, hy = h(s["codes"]), h(s["scales"]), h(s["x"]), h(y)
    if kind == "matmul":
        size = matmul.workspace_bytes(codes, scheme, x, elem, epilogue)
        space = empty((max(size, 16),), torch.uint8)

        def call():
            matmul.launch_ref(client, codes, scales, scheme, x, hy, elem, y_elem, epilogue, workspace=space.data_ptr(), workspace_size=size)
            return y
    else:
        offsets, rows = h(s["offsets"]), h(s["row_of"]) if "row_of" in s else None
        size = experts.workspace_bytes(codes, scheme, hy, elem, epilogue)
        space = empty((max(size, 16),), torch.uint8)

        def call():
            experts.launch_ref(client, codes, scales, scheme, x, offsets, hy, elem, y_elem, rows, epilogue, workspace=space.data_ptr(), workspace_size=size)
            return y
    s["call"] = call
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------------


def _decoded(codes, case):
    """The numbers that a stored tensor [rows, ...] holds, in 32 bits."""
    if case["value"] == "E4M3":
        return codes.view(torch.float8_e4m3fn).float()
    if case["store"] == "Native":
        if case["value"] == "Q8S":
            return codes.view(torch.int8).float()
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        table = torch.cat([table, -table])
        nibbles = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)
        return table[nibbles.int()]
    bits = _BITS[case["value"]]
    shifts = torch.arange(32 - bits, -1, -bits, dtype=torch.int32, device=codes.device)
    return ((codes.unsqueeze(-1) << shifts) >> (32 - bits)).view(codes.shape[0], -1).float()


def _dequantized(codes, scales, case):
    """A weight [rows, cols] as dequantize would store it for the type of x, widened."""
    dtype = _TORCH[case["elem"]]
    q, s = _decoded(codes, case), scales.float().to(dtype).float()
    if case["block"]:
        rows, cols = q.shape
        high = case["block_rows"]
        q = (q.view(rows // high, high, cols // case["block"], case["block"]) * s.view(rows // high, 1, cols // case["block"], 1)).view(rows, cols)
    else:
        q = q * s
    return q.to(dtype).float()


def _activated(v, name):
    if name == "relu":
        return v.clamp(min=0.0)
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v


def _product(x, codes, scales, bias, case):
    """The product of rows of x with one weight, and what comes behind it but the residual, in 32 bits."""
    v = x.float() @ _dequantized(codes, scales, case).t()
    if bias is not None:
        v = v + bias.float()
    if case["gated"]:
        return _activated(v[:, :case["rows"]], case["activation"]) * v[:, case["rows"]:]
    return _activated(v, case["activation"])


def _route(s):
    case = s["case"]
    t, e, k = case["tokens"], case["experts"], case["chosen"]
    logits = s["logits"].float()
    # a stable sort keeps the lower index in front where two are equal
    experts = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    if case["score"] == "softmax":
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    weights = p.gather(-1, experts)
    if case["normalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    flat = experts.flatten()
    order = torch.argsort(flat, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * k, device=order.device)
    counts = (flat.unsqueeze(0) == torch.arange(e, device=flat.device).unsqueeze(1)).sum(-1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=flat.device), counts.cumsum(0)])
    return weights, experts.int(), offsets.int(), (order // k).int(), slots.view(t, k).int()


def run(s):
    if "call" in s:
        return s["call"]()
    case = s["case"]
    kind = case["kind"]
    if kind == "route":
        return _route(s)
    out = _TORCH[case["out"]]
    if kind == "combine":
        y = (s["h"].float()[s["slots"].long()] * s["weights"].unsqueeze(-1)).sum(1)
        return (y + s["residual"].float() if case["residual"] else y).to(out)
    if kind == "matmul":
        v = _product(s["x"], s["codes"], s["scales"], s.get("bias"), case)
        return (v + s["residual"].float() if case["residual"] else v).to(out)
    y = torch.empty((case["tokens"] * case["chosen"], case["rows"]), dtype=out, device="cuda")
    at = s["offsets"].tolist()
    for e in range(case["experts"]):
        a, b = at[e], at[e + 1]
        if a == b:
            continue
        x = s["x"][s["row_of"][a:b].long()] if case["gather"] else s["x"][a:b]
        y[a:b] = _product(x, s["codes"][e], s["scales"][e] if case["block"] else s["scales"], s["bias"][e] if case["bias"] else None, case).to(out)
    return y


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------


def work(case):
    """Bytes and operations of one pass.  Experts: the weights of those that have a token, as many as an even choice would give."""
    kind, t = case["kind"], case["tokens"]
    if kind == "route":
        pairs = t * case["chosen"]
        return {"bytes": t * case["experts"] * _BYTES[case["elem"]] + 16 * pairs + 4 * (case["experts"] + 1), "flops": 5 * t * case["experts"]}
    if kind == "combine":
        pairs = t * case["chosen"]
        return {"bytes": pairs * (case["rows"] * _BYTES[case["elem"]] + 8) + t * case["rows"] * _BYTES[case["out"]] * (2 if case["residual"] else 1),
                "flops": 2 * pairs * case["rows"]}
    wide = case["rows"] * (2 if case["gated"] else 1)
    one = wide * case["cols"] * _BITS[case["value"]] // 8
    if case["block"]:
        one += wide * case["cols"] // (case["block"] * case["block_rows"]) * _BYTES[case["param"]]
    if case["bias"]:
        one += wide * _BYTES[case["elem"]]
    pairs, passed, taken = t, t, 1.0
    if kind == "experts":
        pairs = t * case["chosen"]
        passed = t if case["gather"] else pairs
        taken = case["experts"] * (1.0 - (1.0 - case["chosen"] / case["experts"]) ** t)
    extra = t * case["rows"] * _BYTES[case["out"]] if case.get("residual") else 0
    moved = taken * one + passed * case["cols"] * _BYTES[case["elem"]] + pairs * case["rows"] * _BYTES[case["out"]] + extra
    return {"bytes": int(moved), "flops": 2 * pairs * wide * case["cols"]}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------


def _exact_weights(codes, scales, case):
    """A weight [rows, cols] in 64 bits: each code looked up among the numbers that its bits stand for."""
    bits, device = _BITS[case["value"]], codes.device
    raw = codes.contiguous().view(torch.uint8).view(codes.shape[0], -1)  # little-endian: the first value lies lowest
    if bits < 8:
        raw = torch.stack([(raw >> i) & ((1 << bits) - 1) for i in range(0, 8, bits)], -1).view(codes.shape[0], -1)
    number = torch.arange(1 << bits, dtype=torch.float64, device=device)
    if case["value"] == "E4M3":
        sign, power, rest = 1 - 2 * (number // 128), number % 128 // 8, number % 8
        number = sign * torch.where(power == 0, rest * 2.0 ** -9, (8 + rest) * 2.0 ** (power - 10))
    elif case["value"] == "E2M1" and case["store"] == "Native":
        sign, power, rest = 1 - 2 * (number // 8), number % 8 // 2, number % 2
        number = sign * torch.where(power == 0, rest / 2, (2 + rest) * 2.0 ** (power - 2))
    else:
        number = torch.where(number >= 1 << (bits - 1), number - (1 << bits), number)
    v = number[raw.long()]
    s = scales.double().to(_TORCH[case["elem"]]).double()
    if case["block"]:
        s = s.repeat_interleave(case["block_rows"], 0).repeat_interleave(case["block"], 1)
    return (v * s).to(_TORCH[case["elem"]]).double()  # a code times a scale has at most 19 bits: rounded once


def _exact_product(x, codes, scales, bias, case):
    x, rows = x.double(), case["rows"]

    def part(first, last):
        high = max(1, case["block_rows"])
        first_block, last_block = first // high, (last + high - 1) // high
        w = _exact_weights(codes[first_block * high:last_block * high], scales[first_block:last_block] if case["block"] else scales, case)
        v = torch.mm(x, w[first - first_block * high:last - first_block * high].t().contiguous())
        return v if bias is None else v + bias[first:last].double()

    def act(v):
        if case["activation"] == "relu":
            return torch.relu(v)
        if case["activation"] == "silu":
            return v * torch.sigmoid(v)
        if case["activation"] == "gelu":
            return v * torch.special.ndtr(v)
        return v

    out = []
    for r in range(0, rows, 2048):
        to = min(rows, r + 2048)
        out.append(act(part(r, to)) * part(rows + r, rows + to) if case["gated"] else act(part(r, to)))
    return torch.cat(out, 1)


def exact(case, seed):
    s = _inputs(case, seed)
    kind, t = case["kind"], case["tokens"]
    if kind == "route":
        e, k, logits = case["experts"], case["chosen"], s["logits"].double()
        key = logits - torch.arange(e, device="cuda") * 1e-13  # lower indexes first among equals: logits lie further apart
        experts = key.topk(k, -1).indices
        weights = (logits.log_softmax(-1).exp() if case["score"] == "softmax" else torch.sigmoid(logits)).gather(-1, experts)
        if case["normalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        by = experts.flatten() * (t * k) + torch.arange(t * k, device="cuda")
        order = by.sort().values % (t * k)
        offsets = torch.searchsorted(experts.flatten().sort().values, torch.arange(e + 1, device="cuda"))
        slots = order.sort().indices.view(t, k)
        return weights, experts.int(), offsets.int(), (order // k).int(), slots.int()
    if kind == "combine":
        y = torch.zeros((t, case["rows"]), dtype=torch.float64, device="cuda")
        for j in range(case["chosen"]):
            y += s["weights"][:, j:j + 1].double() * s["h"].index_select(0, s["slots"][:, j].long()).double()
        return y + s["residual"].double() if case["residual"] else y
    if kind == "matmul":
        y = _exact_product(s["x"], s["codes"], s["scales"], s.get("bias"), case)
        return y + s["residual"].double() if case["residual"] else y
    parts, counts = [], s["offsets"].diff().tolist()
    x = s["x"].index_select(0, s["row_of"].long()) if case["gather"] else s["x"]
    for e, rows in enumerate(x.split(counts)):
        parts.append(_exact_product(rows, s["codes"][e], s["scales"][e] if case["block"] else s["scales"], s["bias"][e] if case["bias"] else None, case))
    return torch.cat(parts)

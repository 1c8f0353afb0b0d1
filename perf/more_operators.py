"""A cache of keys and values in pages, quantized or not, with what a model does around it, as cases that can be timed and compared: appending
new tokens (rotary positions and quantization on the way), attention over the pages for single new tokens and for prompts, copying pages.
What each case stands for is said at `listed()`; `draw()` gives further cases of the same ranges.

A case is a dict of plain values.  `prepare()` makes what a program holds before the call, `run()` makes one pass: where `own` is
false by elementary torch operations in 32 bits (in 64 for the angles of far positions and for what is rounded to codes behind them), where it is
true by the public entry points of `cubek_amd`.  `exact()` gives the results in 64 bits.

What a cache holds is scale * code, not rounded again.  Codes are made the way quantize makes them from values of the tensor's type F: scale =
F(2 absmax / (most - least)) of a block, stored in its own type P; code = round(F(x / F(P(scale)))) kept within the range.
"""
import math

import torch

own = False

_TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
_BYTES = {"F32": 4, "F16": 2, "BF16": 2}
_BITS = {"Q8S": 8, "E4M3": 8, "Q4S": 4, "E2M1": 4}
_MOST = {"Q8S": 127.0, "E4M3": 448.0}


def listed():
    return [
        # a decode step of 16 sequences: queries and keys turned by half-split rotary positions, keys and values to 8 bits in blocks of 32 (the
        # smallest calls there are)
        dict(name="append_decode", kind="append", tokens=16, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, far=4096, elem="F16", value="Q8S",
             param="F16", block=32, page=16),
        # a ragged prompt to fp8, one scale a head, positions far out
        dict(name="append_prompt", kind="append", tokens=4093, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, far=131072, elem="BF16",
             value="E4M3", param="F32", block=128, page=64),
        # a chunk of a prompt to a cache that is not quantized, a quarter of each head turned in neighbouring pairs
        dict(name="append_plain", kind="append", tokens=1021, heads=16, kv_heads=16, dim=64, rotary=16, interleaved=True, far=4096, elem="F16", value="",
             param="F16", block=0, page=16),
        # one new token of three short sequences: latency
        dict(name="decode_few", kind="attention", seqs=3, fewest=1, most=1, shortest=130, longest=701, heads=32, kv_heads=8, dim=128, elem="F16", value="Q8S",
             param="F16", block=32, page=16, cap=0.0, window=0, slopes=False, prefix=False),
        # a decode step of 64 sequences of unlike lengths
        dict(name="decode_batch", kind="attention", seqs=64, fewest=1, most=1, shortest=257, longest=8191, heads=32, kv_heads=8, dim=128, elem="BF16",
             value="Q8S", param="F32", block=128, page=64, cap=0.0, window=0, slopes=False, prefix=False),
        # one new token of a single long sequence over a cache of 4 bits
        dict(name="decode_long", kind="attention", seqs=1, fewest=1, most=1, shortest=131071, longest=131071, heads=64, kv_heads=8, dim=128, elem="BF16",
             value="Q4S", param="BF16", block=32, page=64, cap=0.0, window=0, slopes=False, prefix=False),
        # five drafted tokens of eight sequences to be checked at once: large heads, capped scores, a sliding window
        dict(name="decode_draft", kind="attention", seqs=8, fewest=5, most=5, shortest=900, longest=12001, heads=16, kv_heads=8, dim=256, elem="BF16",
             value="E4M3", param="F32", block=128, page=32, cap=50.0, window=4096, slopes=False, prefix=False),
        # a chunk of a prompt behind what the cache holds already, scores with a bias that falls with distance
        dict(name="prompt_chunk", kind="attention", seqs=1, fewest=509, most=509, shortest=8190, longest=8190, heads=32, kv_heads=8, dim=128, elem="BF16",
             value="Q8S", param="F32", block=32, page=16, cap=0.0, window=0, slopes=True, prefix=False),
        # prompts of unlike lengths at once, each with a prefix that all of its tokens see, over a cache that is not quantized
        dict(name="prompt_prefix", kind="attention", seqs=7, fewest=33, most=2047, shortest=2047, longest=2047, heads=16, kv_heads=16, dim=64, elem="F16",
             value="", param="F16", block=0, page=16, cap=0.0, window=0, slopes=False, prefix=True),
        # a long prompt from its start, fp8
        dict(name="prompt_longest", kind="attention", seqs=1, fewest=8191, most=8191, shortest=8191, longest=8191, heads=32, kv_heads=8, dim=128, elem="BF16",
             value="E4M3", param="F32", block=128, page=64, cap=0.0, window=0, slopes=False, prefix=False),
        # a sequence forks: its last page in every layer, for three continuations
        dict(name="copy_fork", kind="copy", layers=4, pages=256, pairs=3, kv_heads=8, dim=128, elem="BF16", value="Q8S", param="F32", block=128, page=16),
        # a pool of pages compacted
        dict(name="copy_compact", kind="copy", layers=8, pages=4096, pairs=1021, kv_heads=8, dim=128, elem="BF16", value="Q8S", param="F32", block=128, page=16),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    cases = listed()
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "copy"])
    like = [c for c in cases if c["name"].startswith(kind)]
    flops, moved, room = max(work(c)["flops"] for c in like), max(work(c)["bytes"] for c in cases), max(_room(c) for c in cases)
    while True:
        case = _draw_one(rng, kind)
        w = work(case)
        if w["flops"] <= flops and w["bytes"] <= moved and _room(case) <= room:
            return case


def _room(case):
    """What has to fit the card: entries of the padded scores and of the padded cache, which the plain form takes, or bytes of the pools."""
    if case["kind"] == "append":
        return 0
    if case["kind"] == "copy":
        return 2 * case["layers"] * case["pages"] * case["kv_heads"] * case["page"] * _row_bytes(case)
    return case["seqs"] * case["longest"] * (case["heads"] * case["most"] + 2 * case["kv_heads"] * case["dim"])


def _draw_one(rng, kind):
    elem = rng.choice(["BF16", "BF16", "F16"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 16), (64, 8), (16, 8), (8, 1), (28, 4), (40, 8), (5, 5)])
    dim, block = rng.choice([(64, 32), (64, 64), (96, 32), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128)])
    value = rng.choice(["Q8S", "Q8S", "E4M3", "Q4S", "E2M1", ""])
    common = dict(dim=dim, block=block if value else 0, value=value, param=rng.choice(["F32", elem]) if value else elem, page=rng.choice([16, 16, 32, 64, 128]), elem=elem)
    if kind == "copy":
        pages = _between(rng, 64, 4096)
        return dict(common, kind=kind, layers=rng.randint(1, 8), pages=pages, pairs=_between(rng, 1, pages // 4), kv_heads=kv_heads)
    if kind == "append":
        if value in ("Q4S", "E2M1"):
            common["value"] = "E4M3"
        return dict(common, kind=kind, tokens=_between(rng, 1, 8192), heads=heads, kv_heads=kv_heads, rotary=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleaved=rng.choice([True, False]), far=_between(rng, 256, 262144))
    extra = dict(cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, 512, 4096]), slopes=rng.choice([True, False, False]))
    if kind == "decode":
        seqs, most = _between(rng, 1, 256), rng.choice([1, 1, 1, 2, 4, 7])
        longest = max(most, _between(rng, 1, 262144 // seqs))
        return dict(common, kind="attention", seqs=seqs, fewest=most, most=most, shortest=max(most, longest // rng.choice([1, 2, 8])), longest=longest, heads=heads,
                    kv_heads=kv_heads, prefix=False, **extra)
    if value:  # prompts of 16 bits by 16 bits of the same range, quantized ones by the wider type
        common["elem"] = "BF16"
        common["param"] = rng.choice(["F32", "BF16"])
    seqs, most = _between(rng, 1, 8), _between(rng, 64, 8191)
    past = rng.choice([0, 0, _between(rng, 1, 8192)])
    return dict(common, kind="attention", seqs=seqs, fewest=max(1, most // rng.choice([1, 1, 2, 16])), most=most, shortest=most + past // 2, longest=most + past, heads=heads,
                kv_heads=kv_heads, prefix=rng.choice([True, False, False]), **extra)


def _spread(low, high, n):
    """n whole numbers evenly from low to high."""
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _sequences(case):
    """(new tokens, length of the cache with them) of each sequence; their order goes by the seed."""
    new = _spread(case["fewest"], case["most"], case["seqs"])
    return [(n, max(n, length)) for n, length in zip(new, _spread(case["shortest"], case["longest"], case["seqs"]))]


# ---- inputs ----------------------------------------------------------------------------------------------------------------


def _codes(gen, case, shape):
    """Stored tensor and scales of random contents [..., dim]: normal values in steps of their scales."""
    value, lead, dim = case["value"], shape[:-1], shape[-1]
    if not value:
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).to(_TORCH[case["elem"]]), None)
    scales = (0.5 + torch.rand(lead + (dim // case["block"],), generator=gen, device="cuda")).mul_({"Q8S": 0.025, "E4M3": 0.006, "Q4S": 0.3, "E2M1": 0.4}[value])
    scales = scales.to(_TORCH[case["param"]])
    if value == "E4M3":
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(150).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scales
    if value == "Q8S":
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(40).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8), scales
    if value == "E2M1":  # pairs of nibbles, any of which is a number
        return torch.randint(0, 256, lead + (dim // 2,), generator=gen, device="cuda", dtype=torch.uint8), scales
    nibbles = torch.randint(-7, 8, lead + (dim // 2, 2), generator=gen, device="cuda", dtype=torch.int8) & 15
    return (nibbles[..., 0] | (nibbles[..., 1] << 4)).view(torch.int32), scales


def _pool(gen, case, pages):
    """The stored tensors of a cache: keys, their scales, values, their scales."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    return _codes(gen, case, shape) + _codes(gen, case, shape)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    dtype, page, dim = _TORCH[case["elem"]], case["page"], case["dim"]
    if case["kind"] == "copy":
        s["pools"] = [_pool(gen, case, case["pages"]) for _ in range(case["layers"])]
        s["pairs"] = torch.randperm(case["pages"], generator=gen, device="cuda")[:2 * case["pairs"]].view(-1, 2).int()  # no page twice
        if case["pairs"] <= 4:  # a fork: one page to several
            s["pairs"][:, 0] = s["pairs"][0, 0]
        return s
    if case["kind"] == "append":
        t, heads, kv_heads = case["tokens"], case["heads"], case["kv_heads"]
        pages = max(-(-t // page) * 2, min(t, 64)) + 8
        s["keys"], s["key_scales"], s["values"], s["value_scales"] = _pool(gen, case, pages)
        x = torch.randn((t, (heads + 2 * kv_heads) * dim), generator=gen, device="cuda")  # what the layer's one projection gives
        x *= torch.where(torch.rand(x.shape[-1:], generator=gen, device="cuda") < 0.02, 8.0, 1.0)  # some channels are larger
        s["x"] = x.to(dtype)
        q, k, v = s["x"].view(t, -1, dim).split([heads, kv_heads, kv_heads], 1)
        s["q"], s["k"], s["v"] = q, k, v
        free = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(t, device="cuda")
        first = torch.randint(0, max(1, case["far"] - t), (), generator=gen, device="cuda")
        if t <= 64:  # a decode step: every token has a page and a position of its own; the batch is padded
            s["slots"] = free[at] * page + torch.randint(0, page, (t,), generator=gen, device="cuda")
            s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda").int()
            s["slots"] = torch.where(at % 8 == 7, -1, s["slots"]).int()
        else:
            s["slots"] = (free[at // page] * page + at % page).int()
            s["positions"] = (first + at).int()
        half = torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda")
        s["frequencies"] = (10000.0 ** (-2.0 * half / case["rotary"])).float()
        return s
    order = torch.randperm(case["seqs"], generator=gen, device="cuda")
    counts, lengths = torch.tensor(_sequences(case), device="cuda")[order].unbind(1)
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)]).int()
    s["lengths"] = lengths.int()
    need = -(-lengths // page)
    width = -(-max(n for _, n in _sequences(case)) // page)
    pages = sum(-(-n // page) for _, n in _sequences(case)) + 5
    s["keys"], s["key_scales"], s["values"], s["value_scales"] = _pool(gen, case, pages)
    at = torch.arange(width, device="cuda")
    free = torch.randperm(pages, generator=gen, device="cuda")
    first = need.cumsum(0) - need
    s["table"] = torch.where(at < need[:, None], free[(first[:, None] + at).clamp_(max=pages - 1)], -1).int()
    tokens = sum(n for n, _ in _sequences(case))
    s["q"] = (torch.randn((tokens, case["heads"], dim), generator=gen, device="cuda") * 1.5).to(dtype)
    if case["slopes"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"])
    if case["prefix"]:
        s["prefix"] = (lengths // 3).int()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    return _hold(s) if own else s


# ---- the framework's calls -------------------------------------------------------------------------------------------------


def _cache_of(s, tensors):
    """The framework's cache over the stored tensors: keys, their scales, values, their scales."""
    from cubek_amd import Cache, QuantLevel, QuantParam, QuantScheme, QuantStore, QuantValue, TensorHandleRef
    case, h = s["case"], lambda t: None if t is None else TensorHandleRef.from_torch(t)
    scheme = None
    if case["value"]:
        store = QuantStore.U32 if case["value"] == "Q4S" else QuantStore.Native
        scheme = (QuantScheme.default().with_value(QuantValue[case["value"]]).with_store(store).with_param(QuantParam[case["param"]])
                  .with_level(QuantLevel.block([case["block"]])))
    keys, key_scales, values, value_scales = (h(t) for t in tensors)
    return Cache(keys, values, scheme, key_scales, value_scales)


def _hold(s):
    """What a program keeps beside its tensors: handles, the scheme, result tensors and workspaces."""
    from cubek_amd import ComputeClient, ElemType, Rotary, Scores, TensorHandleRef, attention, cache
    case, client, h = s["case"], ComputeClient.current(), TensorHandleRef.from_torch
    elem = ElemType[case["elem"]]
    if case["kind"] == "copy":
        tensors, pairs = [h(t) for pool in s["pools"] for t in pool if t is not None], h(s["pairs"])
        s["call"] = lambda: cache.copy_pages(client, tensors, pairs)
        return s
    held = _cache_of(s, (s["keys"], s["key_scales"], s["values"], s["value_scales"]))
    q = h(s["q"])
    if case["kind"] == "append":
        s["q_out"] = torch.empty((case["tokens"], case["heads"], case["dim"]), dtype=s["q"].dtype, device="cuda")
        rotary = Rotary(h(s["frequencies"]), interleaved=case["interleaved"])
        k, v, slots, positions, q_out = (h(s[n]) for n in ("k", "v", "slots", "positions", "q_out"))
        s["call"] = lambda: cache.append(client, held, k, v, slots, elem, q=q, q_out=q_out, positions=positions, rotary=rotary)
        return s
    s["y"] = torch.empty_like(s["q"])
    y, table, offsets, lengths = (h(s[n]) for n in ("y", "table", "offsets", "lengths"))
    scores = Scores(cap=case["cap"], window=case["window"], slopes=h(s["slopes"]) if case["slopes"] else None, prefix=h(s["prefix"]) if case["prefix"] else None)
    size = attention.workspace_bytes(held, q, table, elem)
    s["space"] = torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")
    space = s["space"].data_ptr()
    s["call"] = lambda: attention.launch_ref(client, held, q, y, table, offsets, lengths, elem, scores, workspace=space, workspace_size=size)
    return s


def _shown(codes, case):
    """A stored tensor of 8 bits or of floats by the values that it holds."""
    if not case["value"]:
        return codes
    return codes.view(torch.float8_e4m3fn if case["value"] == "E4M3" else torch.int8)


def _updated(s, q_out):
    case = s["case"]
    out = [q_out, _shown(s["keys"], case), _shown(s["values"], case)]
    return out + [s["key_scales"], s["value_scales"]] if case["value"] else out


def run(s):
    kind = s["case"]["kind"]
    if kind == "copy":
        if "call" in s:
            s["call"]()
        else:
            _copied(s)
        return [t for pool in s["pools"] for t in pool if t is not None]
    if "call" in s:
        s["call"]()
        return _updated(s, s["q_out"]) if kind == "append" else s["y"]
    return _append(s) if kind == "append" else _attention(s)


# ---- the plain form --------------------------------------------------------------------------------------------------------


def _copied(s):
    source, to = s["pairs"].long().unbind(1)
    return [t.index_copy_(0, to, t[source]) for pool in s["pools"] for t in pool if t is not None]


def _turned(x, angles, case):
    """x [tokens, heads, dim] with the first `rotary` entries of each head turned, in 64 bits, rounded once to the type of x."""
    c, w, r = angles.cos()[:, None], angles.sin()[:, None], case["rotary"]
    v = x[..., :r].double()
    if case["interleaved"]:
        a, b = v[..., 0::2], v[..., 1::2]
        turned = torch.stack([a * c - b * w, b * c + a * w], -1).flatten(-2)
    else:
        a, b = v[..., :r // 2], v[..., r // 2:]
        turned = torch.cat([a * c - b * w, b * c + a * w], -1)
    return torch.cat([turned.to(x.dtype), x[..., r:]], -1)


def _quantized(x, case):
    """Codes and scales of x [tokens, heads, dim]."""
    if not case["value"]:
        return x, None
    dtype, most = _TORCH[case["elem"]], _MOST[case["value"]]
    v = x.float().unflatten(-1, (-1, case["block"]))
    scale = (2.0 * v.abs().amax(-1) / (2.0 * most)).to(dtype).to(_TORCH[case["param"]])
    code = (v / scale.to(dtype).float().unsqueeze(-1)).to(dtype).float().round().clamp(-most, most).flatten(-2)
    return (code.to(torch.float8_e4m3fn) if case["value"] == "E4M3" else code.to(torch.int8)).view(torch.uint8), scale


def _stored(pool, slots, rows):
    """Rows [tokens, heads, ...] into their slots of [pages, heads, page, ...]; a slot of -1 takes none."""
    if rows is None:
        return None
    keep = slots >= 0
    at = torch.where(keep, slots, slots.amax()).long()  # what is not kept rewrites what the last slot's own token brings
    rows = torch.where(keep.view(-1, 1, 1), rows, rows[slots.argmax()])
    return pool.transpose(1, 2).index_put_((at // pool.shape[2], at % pool.shape[2]), rows)


def _append(s):
    case = s["case"]
    angles = s["positions"].double()[:, None] * s["frequencies"].double()
    k, k_scales = _quantized(_turned(s["k"], angles, case), case)
    v, v_scales = _quantized(s["v"], case)
    _stored(s["keys"], s["slots"], k), _stored(s["values"], s["slots"], v)
    _stored(s["key_scales"], s["slots"], k_scales), _stored(s["value_scales"], s["slots"], v_scales)
    return _updated(s, _turned(s["q"], angles, case))


def _decoded(codes, case):
    """The numbers that a stored tensor [..., stored] holds, in 32 bits."""
    if case["value"] == "E4M3":
        return codes.view(torch.float8_e4m3fn).float()
    if case["value"] == "Q8S":
        return codes.view(torch.int8).float()
    if not case["value"]:
        return codes.float()
    codes = codes.view(torch.uint8)
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    if case["value"] == "E2M1":
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        return torch.cat([table, -table])[nibbles.int()]
    return (nibbles ^ 8).float() - 8.0


def _gathered(codes, scales, table, case):
    """[seqs, kv_heads, width * page, dim] of the pages of each sequence, in 32 bits."""
    take = lambda t: t[table].transpose(1, 2).flatten(2, 3)  # noqa: E731
    v = _decoded(take(codes), case)
    if scales is None:
        return v
    return (v.unflatten(-1, (-1, case["block"])) * take(scales).float().unsqueeze(-1)).flatten(-2)


def _attention(s):
    case, dim, heads, kv_heads = s["case"], s["case"]["dim"], s["case"]["heads"], s["case"]["kv_heads"]
    table = s["table"].clamp(min=0).long()
    keys = _gathered(s["keys"], s["key_scales"], table, case)
    offsets, lengths = s["offsets"].long(), s["lengths"].long()
    most = case["most"]
    new = torch.arange(most, device="cuda")
    counts = offsets.diff()
    token = (offsets[:-1, None] + new).clamp(max=s["q"].shape[0] - 1)  # [seqs, most]
    q = s["q"].float()[token].view(-1, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seqs, kv_heads, group * most, dim]
    x = torch.matmul(q * dim ** -0.5, keys.transpose(-1, -2).contiguous()).view(-1, kv_heads, heads // kv_heads, most, keys.shape[2])
    del keys
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    j = torch.arange(x.shape[-1], device="cuda")
    i = (lengths - counts)[:, None] + new  # the position of each query
    apart = i[:, :, None] - j  # [seqs, most, keys]
    seen = apart >= 0
    if case["prefix"]:
        seen = seen | (j < s["prefix"].long()[:, None, None])
    seen = seen & (j < lengths[:, None, None])
    if case["window"]:
        seen = seen & (apart < case["window"])
    if case["slopes"]:
        x = x - s["slopes"].view(1, kv_heads, -1, 1, 1) * apart.abs()[:, None, None]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    values = _gathered(s["values"], s["value_scales"], table, case)
    y = torch.matmul(x.flatten(2, 3), values).view(-1, kv_heads, heads // kv_heads, most, dim) / total.clamp(min=1e-30)
    y = y.permute(0, 3, 1, 2, 4).reshape(-1, most, heads, dim)
    t = torch.arange(s["q"].shape[0], device="cuda")
    of = torch.searchsorted(offsets[1:], t, right=True)
    return y[of, t - offsets[of]].to(s["q"].dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------


def _row_bytes(case):
    """Bytes of one head of one token in the cache."""
    if not case["value"]:
        return case["dim"] * _BYTES[case["elem"]]
    return case["dim"] * _BITS[case["value"]] // 8 + case["dim"] // case["block"] * _BYTES[case["param"]]


def work(case):
    """Bytes and operations of one pass.  Attention: keys and values that some query sees, read once; two products for each query and each key it sees."""
    if case["kind"] == "copy":
        once = case["layers"] * 2 * case["kv_heads"] * case["page"] * _row_bytes(case)
        sources = 1 if case["pairs"] <= 4 else case["pairs"]
        return {"bytes": once * (sources + case["pairs"]) + 8 * case["pairs"], "flops": 0}
    size = _BYTES[case["elem"]]
    if case["kind"] == "append":
        t, q, kv = case["tokens"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        stored = 2 * case["kv_heads"] * _row_bytes(case)
        return {"bytes": t * (size * (2 * q + 2 * kv) + stored + 8) + 2 * case["rotary"], "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    pairs = keys = tokens = 0
    for n, length in _sequences(case):
        tokens += n
        window = case["window"] or length
        prefix = length // 3 if case["prefix"] else 0
        first = length - n
        # query i of length - n ... length - 1 sees max(0, i - window + 1) ... i, and the prefix behind it
        below = max(0, min(n, window - 1 - first))  # queries whose window reaches the start
        pairs += below * (2 * first + below + 1) // 2 + (n - below) * window
        ahead = max(0, min(n, prefix - first))
        pairs += ahead * (prefix - first) - ahead * (ahead + 1) // 2
        keys += min(length, window + n - 1)
    moved = 2 * keys * case["kv_heads"] * _row_bytes(case) + 2 * tokens * case["heads"] * case["dim"] * size + 4 * (keys // case["page"] + 2 * case["seqs"])
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------


def _numbers(codes, case):
    """What a stored tensor [..., stored] holds in 64 bits: each code looked up among the numbers that its bits stand for."""
    if not case["value"]:
        return codes.double()
    bits, raw = _BITS[case["value"]], codes.contiguous().view(torch.uint8)
    if bits == 4:
        raw = torch.stack([raw % 16, raw // 16], -1).flatten(-2)
    number = torch.arange(1 << bits, dtype=torch.float64, device=codes.device)
    if case["value"] == "E4M3":
        sign, power, rest = 1 - 2 * (number // 128), number % 128 // 8, number % 8
        number = sign * torch.where(power == 0, rest * 2.0 ** -9, (8 + rest) * 2.0 ** (power - 10))
    elif case["value"] == "E2M1":
        sign, power, rest = 1 - 2 * (number // 8), number % 8 // 2, number % 2
        number = sign * torch.where(power == 0, rest / 2, (2 + rest) * 2.0 ** (power - 2))
    else:
        number = torch.where(number >= 1 << (bits - 1), number - (1 << bits), number)
    return number[raw.long()]


def _exact_append(s):
    case, dtype = s["case"], s["x"].dtype
    angle = torch.outer(s["positions"].double(), s["frequencies"].double())
    z, r = torch.polar(torch.ones_like(angle), angle).unsqueeze(1), case["rotary"]

    def turned(x):
        v = x.double()
        pairs = v[..., :r].unflatten(-1, (-1, 2)) if case["interleaved"] else v[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        return torch.cat([(pairs if case["interleaved"] else pairs.transpose(-1, -2)).flatten(-2), v[..., r:]], -1)

    out = [turned(s["q"])]
    scales = []
    at = s["slots"].long()
    keep = at >= 0
    for name, x in (("keys", turned(s["k"]).to(dtype)), ("values", s["v"])):
        pool, x = s[name], x.double()
        shape = pool.shape[:3] + (case["dim"],)
        now = _numbers(pool, case).transpose(1, 2).flatten(0, 1)
        if case["value"]:
            most, block = _MOST[case["value"]], case["block"]
            top = torch.stack([part.abs().amax(-1) for part in x.split(block, -1)], -1)
            scale = (top / most).to(dtype).to(_TORCH[case["param"]])
            by = scale.to(dtype).double().repeat_interleave(block, -1)
            x = (x / by).to(dtype).double().round().clamp(-most, most)
            if case["value"] == "E4M3":
                x = x.to(torch.float8_e4m3fn).double()
            held = s[name[:-1] + "_scales"].double().transpose(1, 2).flatten(0, 1)
            held[at[keep]] = scale[keep].double()
            scales.append(held.view(shape[0], shape[2], shape[1], -1).transpose(1, 2))
        now[at[keep]] = x[keep]
        now = now.view(shape[0], shape[2], shape[1], -1).transpose(1, 2)
        out.append(now.to(torch.int8) if case["value"] == "Q8S" else now)
    return out + scales


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "copy":
        came_from = torch.arange(case["pages"], device="cuda").scatter_(0, s["pairs"][:, 1].long(), s["pairs"][:, 0].long())
        return [t[came_from].double() if t.is_floating_point() else t[came_from] for pool in s["pools"] for t in pool if t is not None]
    if case["kind"] == "append":
        return _exact_append(s)
    group, page, dim = case["heads"] // case["kv_heads"], case["page"], case["dim"]
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def held(codes, scales, pages, head, length):
        v = _numbers(codes[pages, head], case).flatten(0, 1)[:length]
        return v if scales is None else v * scales[pages, head].double().flatten(0, 1)[:length].repeat_interleave(case["block"], -1)

    for e, length in enumerate(lengths):
        a, b = offsets[e], offsets[e + 1]
        pages = s["table"][e, :-(-length // page)].long()
        i, j = torch.arange(length - (b - a), length, device="cuda")[:, None], torch.arange(length, device="cuda")
        hidden = j > i
        if case["prefix"]:
            hidden &= j >= s["prefix"][e]
        if case["window"]:
            hidden |= i - j >= case["window"]
        for head in range(case["kv_heads"]):
            k = held(s["keys"], s["key_scales"], pages, head, length).t().contiguous()
            v = held(s["values"], s["value_scales"], pages, head, length)
            for g in range(head * group, head * group + group):
                x = torch.mm(s["q"][a:b, g].double(), k) / math.sqrt(dim)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if case["slopes"]:
                    x -= s["slopes"][g].double() * (i - j).abs()
                p = torch.softmax(x.masked_fill_(hidden, -math.inf), -1)
                out[a:b, g] = torch.mm(p, v)
    return out

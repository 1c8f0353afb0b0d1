"""cq_cache_append and cq_cache_copy.  Codes and scales have to be those of the oracle for keys turned in 64 bits and rounded once; turned queries
are the exact ones rounded to F by way of f32: half a step of F, and |v| 2^-24 (1 + 2^-7) for the first rounding of a number v that the second takes
to within 2^-8 of itself."""
import numpy as np
import pytest

from attention_reference import h, laid_out, on_device
from cubek_amd import Cache, ComputeClient, ElemType, QuantStore, QuantValue, Rotary, cache, rotary
from matmul_reference import PARAM, TORCH, random_weight, scheme_of, storage

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
U32, NATIVE = QuantStore.U32, QuantStore.Native
V = QuantValue
SCHEMES = [None, (V.Q8S, NATIVE, 32, 0), (V.Q8F, U32, 64, 1), (V.Q4S, U32, 32, 2), (V.E4M3, NATIVE, 64, 0), (V.E5M2, NATIVE, 32, 2), (V.E2M1, NATIVE, 32, 0),
           (V.E2M1, U32, 16, 1), (V.E2M1_OCP, U32, 64, 0), (V.Q4F, U32, 8, 0)]


def turned(x, positions, frequencies, magnitude, interleaved):
    """[tokens, heads, dim] in 64 bits."""
    n = len(frequencies)
    angle = positions[:, None].astype(np.float64) * frequencies.astype(np.float64)
    c, w = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    y = x.copy()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ya, yb = a * c - b * w, b * c + a * w
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = ya, yb
    else:
        y[..., :n], y[..., n:2 * n] = ya, yb
    return y


def run(oracle, elem, of, tokens, heads, kv_heads, dim, page, turns, interleaved=False, order="heads", seed=0, far=5000, offset=0, magnitude=1.0, in_place=False,
        sizes=1.0, with_q=True):
    import torch

    rng = np.random.default_rng(seed)
    scheme = None if of is None else scheme_of(of[0], [of[2]], of[3], of[1])
    pages = -(-tokens // page) + 2
    shape = (pages, kv_heads, page, dim)
    before = []  # keys, values, their scales
    for _ in range(2):
        if scheme is None:
            before.append((torch.tensor(rng.normal(0, 1, shape)).to(TORCH[elem]).cuda(), None))
        else:
            codes, scales = random_weight(rng, scheme, shape)
            before.append((on_device(codes, scheme), scales.cuda()))
    tensors = [[laid_out(t, order).clone(memory_format=torch.preserve_format) if order == "heads" and t is not None else laid_out(t, order) for t in pair] for pair in before]
    x = torch.zeros((tokens, (heads + 2 * kv_heads) * dim + offset + 8), dtype=TORCH[elem], device="cuda")
    x[:, offset:offset + (heads + 2 * kv_heads) * dim] = torch.tensor(rng.normal(0, 1, (tokens, (heads + 2 * kv_heads) * dim)) * sizes).to(TORCH[elem]).cuda()
    part = x[:, offset:offset + (heads + 2 * kv_heads) * dim].view(tokens, -1, dim)
    q, k, v = part.split([heads, kv_heads, kv_heads], 1)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    skipped = rng.random(tokens) < 0.2
    slots[skipped] = rng.choice([-1, pages * page, 2 ** 31 - 1, -2 ** 31], skipped.sum())
    positions = rng.integers(-far, far, tokens).astype(np.int32)
    frequencies = np.array(rotary.frequencies(turns), np.float32) if turns else np.zeros(0, np.float32)
    host = [t.double().cpu().numpy() for t in (q, k, v)]
    q_out = q if in_place else torch.full((tokens, heads, dim), 8.0, dtype=TORCH[elem], device="cuda")
    f = torch.from_numpy(frequencies).cuda()
    ints = [torch.from_numpy(a).cuda() for a in (slots, positions)]
    (keys, key_scales), (values, value_scales) = [[None if t is None else h(t) for t in pair] for pair in tensors]
    cache.append(ComputeClient.current(), Cache(keys, values, scheme, key_scales, value_scales), h(k), h(v), h(ints[0]), elem, q=h(q) if with_q else None,
                 q_out=h(q_out) if with_q else None, positions=h(ints[1]) if turns else None, rotary=Rotary(h(f), magnitude, interleaved) if turns else None)
    torch.cuda.synchronize()

    if with_q:
        want = turned(host[0], positions, frequencies, magnitude, interleaved) if turns else host[0]
        got = q_out.double().cpu().numpy()
        near = torch.from_numpy(want).to(TORCH[elem]).double().numpy()
        step = np.maximum(np.abs(near), 2.0 ** -14) * torch.finfo(TORCH[elem]).eps
        assert (np.abs(got - want) <= step * 0.5 + np.abs(want) * 2.0 ** -24 * (1 + 2.0 ** -7)).all()
    fresh = turned(host[1], positions, frequencies, magnitude, interleaved) if turns else host[1]
    for name, rows, (old, old_scales), (new, new_scales) in zip(("keys", "values"), (fresh, host[2]), before, tensors):
        rows = torch.from_numpy(rows).to(TORCH[elem])
        expect = old.cpu().clone()
        keep = np.nonzero(~skipped)[0]
        pg, pl = slots[keep] // page, slots[keep] % page
        if scheme is None:
            expect[pg, :, pl] = rows[keep]
            assert torch.equal(expect.view(torch.int16 if elem != F32 else torch.int32), new.cpu().contiguous().view(torch.int16 if elem != F32 else torch.int32)), name
            continue
        stored = storage(rows.float() if elem == F32 else rows)
        s = oracle.compute_scales(stored, elem, rows.shape, scheme)
        codes, s = oracle.quantize(stored, elem, rows.shape, s, scheme)
        codes = torch.from_numpy(codes.view(np.int32) if codes.dtype == np.uint32 else codes)
        param = PARAM[int(scheme.param)]
        s = torch.from_numpy(s) if param == torch.float32 else torch.from_numpy(s.view(np.int16)).view(param)
        expect[pg, :, pl] = codes[keep]
        expect_scales = old_scales.cpu().clone()
        expect_scales[pg, :, pl] = s[keep]
        as_bits = lambda t: t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)  # noqa: E731
        assert torch.equal(as_bits(expect_scales), as_bits(new_scales.cpu())), name
        assert torch.equal(expect, new.cpu()), (name, (expect != new.cpu()).sum())


@pytest.mark.parametrize("of", SCHEMES, ids=str)
@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("interleaved", [False, True])
def test_every_store_and_type(oracle, of, elem, interleaved):
    run(oracle, elem, of, 37, 8, 2, 128, 16, 128, interleaved)


@pytest.mark.parametrize("dim,turns,block", [(64, 64, 32), (64, 16, 64), (64, 8, 16), (96, 48, 32), (96, 96, 96), (128, 30, 32), (80, 80, 16), (80, 20, 40), (100, 100, 20), (256, 128, 128),
                                             (512, 512, 128), (34, 2, 2), (128, 0, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes_of_heads_and_blocks(oracle, dim, turns, block, interleaved):
    for value in (V.Q8S, V.E2M1):
        run(oracle, BF16, (value, NATIVE, block, 0), 21, 6, 3, dim, 8, turns, interleaved)
    run(oracle, F16, None, 21, 6, 3, dim, 8, turns, interleaved)


@pytest.mark.parametrize("tokens", [1, 2, 64, 300, 1021])
@pytest.mark.parametrize("heads,kv_heads,page", [(32, 8, 16), (1, 1, 1), (28, 4, 64), (64, 64, 7)])
def test_numbers_of_tokens_and_heads(oracle, tokens, heads, kv_heads, page):
    run(oracle, F16, (V.Q8S, NATIVE, 32, 1), tokens, heads, kv_heads, 64, page, 64, seed=tokens)


@pytest.mark.parametrize("order", ["slots", "gaps"])
@pytest.mark.parametrize("offset", [0, 1, 3, 4])
@pytest.mark.parametrize("of", [None, (V.Q8S, NATIVE, 32, 0), (V.Q4S, U32, 32, 2)], ids=str)
def test_orders_and_alignment(oracle, order, offset, of):
    for elem in (BF16, F32):
        run(oracle, elem, of, 19, 4, 2, 64, 16, 64, order=order, offset=offset)


def test_in_place_without_queries_and_with_a_magnitude(oracle):
    run(oracle, BF16, (V.E4M3, NATIVE, 64, 0), 40, 8, 2, 64, 16, 64, in_place=True, magnitude=1.3)
    run(oracle, BF16, (V.E4M3, NATIVE, 64, 0), 40, 8, 2, 64, 16, 64, in_place=True, interleaved=True)
    run(oracle, BF16, (V.E4M3, NATIVE, 64, 0), 40, 8, 2, 64, 16, 64, with_q=False)


@pytest.mark.parametrize("far", [1, 1 << 20, (1 << 31) - 1])
def test_far_positions(oracle, far):
    run(oracle, F32, (V.Q8S, NATIVE, 32, 0), 200, 2, 2, 64, 16, 64, far=far)
    run(oracle, BF16, (V.Q8S, NATIVE, 32, 0), 200, 2, 2, 64, 16, 64, far=far)


@pytest.mark.parametrize("sizes", [0.0, 1e-30, 1e30])
def test_sizes_of_values(oracle, sizes):
    run(oracle, BF16, (V.Q8S, NATIVE, 32, 0), 20, 2, 2, 64, 16, 64, sizes=sizes)
    run(oracle, F32, (V.Q4S, U32, 32, 0), 20, 2, 2, 64, 16, 64, sizes=sizes)


@pytest.mark.parametrize("shape", [(9, 2, 16, 64), (40, 3, 5), (7, 1), (5,), (12, 8, 16, 128), (6, 70001)])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_copies_of_pages(shape, count):
    import torch

    rng = np.random.default_rng(len(shape))
    for dtype in (torch.uint8, torch.int32, torch.bfloat16):
        tensors = [torch.from_numpy(rng.integers(0, 100, shape)).to(dtype).cuda() for _ in range(count)]
        tensors[-1] = torch.cat([tensors[-1].view(shape[0], -1)] * 2, 1)[:, :tensors[-1].view(shape[0], -1).shape[1]].view(shape[0], -1)  # pages with gaps
        order = rng.permutation(shape[0])
        half = shape[0] // 2
        pairs = np.stack([order[:half][rng.integers(0, half, half)], order[half:2 * half]], 1).astype(np.int32)
        pairs = np.concatenate([pairs, [[-1, 0], [0, shape[0]], [2 ** 31 - 1, 1], [1, -2 ** 31], [order[0], order[0]]]]).astype(np.int32)
        want = [t.cpu().clone() for t in tensors]
        for t in want:
            t[pairs[:half, 1]] = t[pairs[:half, 0]]
        cache.copy_pages(ComputeClient.current(), [h(t) for t in tensors], h(torch.from_numpy(pairs).cuda()))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.cpu()) for a, b in zip(want, tensors))


def test_copies_of_nothing():
    import torch

    t = torch.ones((4, 8), device="cuda")
    none = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    cache.copy_pages(ComputeClient.current(), [h(t)], h(none))
    cache.copy_pages(ComputeClient.current(), [], h(torch.zeros((1, 2), dtype=torch.int32, device="cuda")))
    cache.copy_pages(ComputeClient.current(), [h(t[:0]), h(t[:, :0])], h(torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    assert (t == 1).all()


def test_append_read_fork_and_read_again(oracle):
    """A step as a program makes it: append, attention, a fork by copying the last page, both continuations; and all of it captured."""
    import torch

    from cubek_amd import attention

    rng = np.random.default_rng(0)
    scheme = scheme_of(V.Q8S, [64], 0, NATIVE)
    pages, kv_heads, page, dim, heads = 12, 2, 16, 64, 4
    keys, values = (torch.zeros((pages, kv_heads, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = [torch.zeros((pages, kv_heads, page, 1), device="cuda") for _ in range(2)]
    held = Cache(h(keys), h(values), scheme, h(scales[0]), h(scales[1]))
    f = torch.tensor(rotary.frequencies(dim), device="cuda")

    def step(x, positions, slots, table, offsets, lengths, y):
        client = ComputeClient.current()
        q, k, v = x.view(x.shape[0], -1, dim).split([heads, kv_heads, kv_heads], 1)
        cache.append(client, held, h(k), h(v), h(slots), BF16, q=h(q), q_out=h(q), positions=h(positions), rotary=Rotary(h(f)))
        attention.launch_ref(client, held, h(q), h(y), h(table), h(offsets), h(lengths), BF16)

    def ints(*a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    prompt = torch.tensor(rng.normal(0, 1, (40, (heads + 2 * kv_heads) * dim))).bfloat16().cuda()
    y = torch.zeros((40, heads, dim), dtype=torch.bfloat16, device="cuda")
    table = ints([3, 7, 1], [3, 7, 9])
    slots = torch.tensor([[3, 7, 1][i // 16] * 16 + i % 16 for i in range(40)], dtype=torch.int32, device="cuda")
    step(prompt.clone(), torch.arange(40, dtype=torch.int32, device="cuda"), slots, table[:1], ints(0, 40), ints(40), y)
    cache.copy_pages(ComputeClient.current(), [h(t) for t in (keys, values, *scales)], h(ints([1, 9])))
    token = torch.tensor(rng.normal(0, 1, (2, (heads + 2 * kv_heads) * dim))).bfloat16().cuda()
    token[1] = token[0]
    both = torch.zeros((2, heads, dim), dtype=torch.bfloat16, device="cuda")
    args = (ints(40, 40), ints(1 * 16 + 8, 9 * 16 + 8), table, ints(0, 1, 2), ints(41, 41), both)
    step(token.clone(), *args)
    torch.cuda.synchronize()
    assert torch.equal(both[0], both[1]) and both.abs().max() > 0
    # the same token as the last of a prompt of 41, read in one go
    again = torch.zeros((41, heads, dim), dtype=torch.bfloat16, device="cuda")
    slots41 = torch.cat([slots, ints(1 * 16 + 8)])
    step(torch.cat([prompt, token[:1]]), torch.arange(41, dtype=torch.int32, device="cuda"), slots41, table[:1], ints(0, 41), ints(41), again)
    torch.cuda.synchronize()
    assert (again[40].float() - both[0].float()).abs().max() <= 2.0 ** -6 * again[40].abs().max()  # another kernel: other roundings of weights to 16 bits
    assert torch.equal(again[:8], y[:8]) or (again[:8].float() - y[:8].float()).abs().max() <= 2.0 ** -6 * y.abs().max()
    x, graph = token.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, *args)
    for _ in range(3):
        x.copy_(token)
        both.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = both.clone()
        x.copy_(token)
        step(x, *args)
        torch.cuda.synchronize()
        assert torch.equal(got, both)

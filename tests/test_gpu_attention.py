"""cq_attention against numpy in 64 bits; tolerances are derived in attention_reference.py."""
import numpy as np
import pytest

from attention_reference import Attention, h
from cubek_amd import ComputeClient, ElemType, QuantStore, QuantValue, Scores, attention
from matmul_reference import TORCH, scheme_of

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
U32, NATIVE = QuantStore.U32, QuantStore.Native
V = QuantValue

# value, store, block, type of the scales
SCHEMES = {
    "floats": None, "q8": (V.Q8S, NATIVE, 32, 0), "q8f_words": (V.Q8F, U32, 64, 1), "q4": (V.Q4S, U32, 32, 2), "q4f": (V.Q4F, U32, 64, 0), "e4m3": (V.E4M3, NATIVE, 64, 0),
    "e5m2": (V.E5M2, NATIVE, 32, 2), "e2m1": (V.E2M1, NATIVE, 32, 0), "e2m1_words": (V.E2M1, U32, 32, 1), "ocp": (V.E2M1_OCP, U32, 64, 0),
}


def scheme(name):
    if SCHEMES[name] is None:
        return None
    value, store, block, param = SCHEMES[name]
    return scheme_of(value, [block], param, store)


@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("name", SCHEMES)
def test_every_store_and_type(oracle, name, elem):
    for seed, sequences in enumerate(([(1, 1), (1, 130), (1, 64)], [(70, 70), (5, 129), (33, 100)])):
        Attention(oracle, seed, sequences, 4, 2, 64, 16, elem, scheme(name)).check((name, sequences))


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("name", ["floats", "q8", "q4", "e4m3"])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_sizes_of_heads(oracle, dim, name, elem):
    value = None if name == "floats" else scheme_of(SCHEMES[name][0], [32], 0, SCHEMES[name][1])
    for seed, sequences in enumerate(([(1, 333), (1, 31)], [(3, 200)], [(150, 190)])):
        Attention(oracle, seed, sequences, 8, 2, dim, 32, elem, value).check((dim, sequences))


@pytest.mark.parametrize("block,dim", [(128, 128), (64, 128), (128, 256), (64, 64), (16, 64), (8, 64), (96, 96), (40, 80), (20, 100), (2, 6)])
@pytest.mark.parametrize("tokens", [1, 40])
def test_sizes_of_blocks(oracle, block, dim, tokens):
    for value in (V.Q8S, V.E2M1):
        Attention(oracle, dim, [(tokens, 77), (tokens, tokens)], 4, 4, dim, 16, BF16, scheme_of(value, [block], 0, NATIVE)).check((block, dim, value))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 17, 48, 64, 128, 1000])
@pytest.mark.parametrize("tokens", [1, 6, 50])
def test_sizes_of_pages(oracle, page, tokens):
    for name in ("q8", "floats"):
        Attention(oracle, page, [(tokens, tokens + extra) for extra in (0, 1, 15, 16, 47, 64, 250)], 4, 2, 64, page, BF16, scheme(name)).check((page, name))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (8, 1), (16, 1), (28, 4), (40, 1), (6, 2)])
@pytest.mark.parametrize("tokens", [1, 3, 7, 20, 130])
def test_groups_of_heads(oracle, heads, kv_heads, tokens):
    for name in ("q8", "floats"):
        Attention(oracle, heads, [(tokens, 140), (tokens, tokens), (1, 65)], heads, kv_heads, 64, 16, F16, scheme(name)).check((name,))


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("name", ["q8", "floats"])
def test_lengths(oracle, length, name):
    sequences = [(1, length), (1, max(length - 1, 0)), (min(length, 2), length), (length, length)]
    Attention(oracle, length, sequences, 4, 2, 64, 16, BF16, scheme(name)).check(sequences)


SCORES = {
    "cap": dict(cap=5.0), "window": dict(window=20), "window of one": dict(window=1), "wide window": dict(window=4294967295), "scale": dict(scale=-0.3),
    "all": dict(cap=3.0, window=70, scale=0.2),
}


@pytest.mark.parametrize("tokens", [1, 4, 37, 150])
@pytest.mark.parametrize("name", ["q8", "floats"])
@pytest.mark.parametrize("kind", list(SCORES) + ["slopes", "prefix", "prefix and window", "everything"])
def test_scores(oracle, tokens, name, kind):
    case = Attention(oracle, tokens, [(tokens, 151), (tokens, tokens), (tokens, 260)], 8, 4, 64, 16, F16, scheme(name))
    scores = dict(SCORES.get(kind, {}))
    if kind in ("slopes", "everything"):
        scores["slopes"] = (2.0 ** -np.arange(1, 9)).astype(np.float32)
    if kind.startswith("prefix") or kind == "everything":
        scores["prefix"] = [150, max(tokens // 2, 1), -4]
    if kind in ("prefix and window", "everything"):
        scores["window"] = 30
    if kind == "everything":
        scores["cap"] = 10.0
    case.check(kind, **scores)


@pytest.mark.parametrize("order", ["slots", "gaps"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("name", SCHEMES)
def test_orders_of_the_cache(oracle, order, tokens, name):
    Attention(oracle, 5, [(tokens, 90), (tokens, 41)], 4, 2, 64, 16, BF16, scheme(name), order).check((order, name))


@pytest.mark.parametrize("tokens", [1, 50])
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_strides_of_queries_and_results(oracle, tokens, offset):
    import torch

    case = Attention(oracle, 9, [(tokens, 90), (tokens, 77)], 4, 2, 64, 16, BF16, scheme("q8"))
    plain = case.call()
    fused = torch.zeros((2 * tokens, 1000), dtype=torch.bfloat16, device="cuda")
    q = fused[:, offset:offset + 256].view(2 * tokens, 4, 64)
    q.copy_(case.q)
    out = torch.full((4, 2 * tokens, 80), -3.0, dtype=torch.bfloat16, device="cuda")
    y = out.transpose(0, 1)[:, :, offset:offset + 64]
    case.call(q=q, y=y)
    want, bound = case.want()
    from matmul_reference import check_rounded

    check_rounded(y.double().cpu().numpy(), want, bound, BF16)
    assert (out[:, :, :offset] == -3).all() and (out[:, :, offset + 64:] == -3).all()
    if offset % 8 == 0:
        assert torch.equal(y, plain)


@pytest.mark.parametrize("tokens", [1, 5, 60])
@pytest.mark.parametrize("name", ["q8", "e5m2", "q4", "floats"])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_what_is_not_seen_may_hold_anything(oracle, tokens, name, elem):
    """Entries behind a sequence's end, behind its window and, for each token, behind itself are infinite or not a number."""
    case = Attention(oracle, 3, [(tokens, 100), (tokens, 61), (tokens, tokens)], 4, 2, 64, 16, elem, scheme(name))
    window = 20
    want, bound = case.want(window=window)  # the first tokens' results hold whatever becomes of what they do not see
    page = case.k.entries.shape[2]
    for pool in (case.k, case.v):
        bad = np.ones(pool.entries.shape[:3], bool)  # [pages, heads, places]
        for s, (n, length) in enumerate(case.sequences):
            for j in range(max(0, length - n - window + 1), length - n + 1):  # what the first of the new tokens sees
                bad[case.table[s, j // page], :, j % page] = False
        spoil(pool, bad, scheme(name))
    got = case.call(window=window).double().cpu().numpy()
    first = case.offsets[:-1]
    assert np.isfinite(got[first]).all()
    from matmul_reference import check_rounded

    check_rounded(got[first], want[first], bound[first], elem)
    # and those behind it see what is not a number, all of them but where the window has passed it by
    for s, (n, length) in enumerate(case.sequences):
        if n > 1:
            assert np.isnan(got[first[s] + 1:case.offsets[s + 1]]).any(-1).all()


def spoil(pool, bad, of):
    """Infinities and NaN in the rows that `bad` names."""
    import torch

    at = torch.from_numpy(bad).cuda()
    if of is None:
        pool.stored[at] = float("nan")
        pool.stored[..., 1::2][at] = float("inf")
    else:
        pool.scales[at] = float("nan")
        if of.value == V.E5M2:
            pool.stored[at] = 0x7c  # infinity


@pytest.mark.parametrize("tokens", [1, 30])
def test_rows_of_nobody_stay(oracle, tokens):
    case = Attention(oracle, 4, [(tokens, 50), (0, 20), (tokens, 33)], 4, 2, 64, 16, BF16, scheme("q8"))
    import torch

    extra = 5
    q = torch.zeros((case.tokens + extra, 4, 64), dtype=torch.bfloat16, device="cuda")
    q[2:2 + case.tokens] = case.q.cuda()
    y = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    plain = case.call()
    case.offsets = case.offsets + 2
    case.call(q=q, y=y)
    assert torch.equal(y[2:2 + case.tokens], plain)
    assert (y[:2] == 9).all() and (y[2 + case.tokens:] == 9).all()


def test_more_tokens_than_keys_and_numbers_outside_of_everything(oracle):
    import torch

    case = Attention(oracle, 4, [(4, 4), (6, 20), (3, 32)], 4, 2, 64, 16, BF16, scheme("q8"))
    whole = case.call()
    case.lengths[:] = [2, 20, 2 ** 31 - 1]  # four tokens for two keys; a length past the table's row
    y = case.call()
    assert (y[:2] == 0).all() and torch.equal(y[4:], whole[4:])
    case.lengths[:] = [-5, 0, -2 ** 31]
    assert (case.call() == 0).all()
    case.lengths[:] = [4, 20, 32]
    case.offsets[:] = [-9, 4, 10, 2 ** 31 - 1]
    assert torch.equal(case.call(), whole)
    case.offsets[:] = [0, 10, 4, 13]  # falls: only that nothing is written out of place is asked for
    case.call()
    case.offsets[:] = [0, 4, 10, 13]
    case.table[case.table < 0] = 2 ** 31 - 1
    assert torch.equal(case.call(), whole)
    case.table[:] = -2 ** 31
    assert torch.isfinite(case.call()).all()


@pytest.mark.parametrize("tokens,length", [(1, 3000), (1, 20011), (3, 9000), (40, 6000), (700, 2500)])
@pytest.mark.parametrize("name", ["q8", "q4", "floats"])
def test_long_sequences_with_a_workspace_and_without(oracle, tokens, length, name):
    case = Attention(oracle, 8, [(tokens, length), (tokens, length // 3)], 4, 1, 128, 64, BF16, scheme(name))
    case.check("with")
    case.check("without", workspace=False)
    case.check("window", window=length // 2)


def test_many_short_sequences(oracle):
    rng = np.random.default_rng(0)
    sequences = [(int(n), int(n) + int(m)) for n, m in zip(rng.integers(0, 4, 300), rng.integers(0, 40, 300))]
    Attention(oracle, 0, sequences, 4, 2, 64, 16, F16, scheme("q8")).check()
    Attention(oracle, 0, [(1, 1 + int(m)) for m in rng.integers(0, 40, 5000)], 2, 1, 64, 16, F16, scheme("q8")).check()


@pytest.mark.parametrize("size", [1e-18, 1e-5, 1e4, 1e18])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("name", ["q8", "q4", "e4m3", "floats"])
def test_entries_far_from_one(oracle, size, tokens, name):
    """bf16's range: entries of the cache of any size, queries of the inverse size."""
    case = Attention(oracle, 6, [(tokens, 200), (tokens, 64)], 4, 2, 64, 16, BF16, scheme_of(*[SCHEMES[name][0], [32], 2, SCHEMES[name][1]]) if SCHEMES[name] else None)
    for pool in (case.k, case.v):
        where = pool.stored if pool.scales is None else pool.scales
        scaled = (where.double() * size).to(where.dtype)
        ratio = (scaled.double() / where.double()).nan_to_num(1.0).cpu().numpy()
        where.copy_(scaled)
        pool.entries *= ratio if pool.scales is None else ratio.repeat(32, -1)
    case.q = (case.q.double() / size).to(case.q.dtype)
    case.check(size)


def test_large_scores(oracle):
    case = Attention(oracle, 2, [(1, 300), (70, 300)], 4, 2, 64, 16, BF16, scheme("q8"), spread=100.0)
    case.check("one key takes all")


@pytest.mark.parametrize("tokens", [1, 40])
def test_captured_and_replayed_beside_eager_calls(oracle, tokens):
    import torch

    case = Attention(oracle, 1, [(tokens, 700), (tokens, 2000), (tokens, 130)], 8, 2, 128, 16, BF16, scheme("q8"))
    ints = [torch.from_numpy(a).cuda() for a in (case.table, case.offsets, case.lengths)]
    q, y = case.q.cuda(), torch.zeros(tuple(case.q.shape), dtype=case.q.dtype, device="cuda")
    size = attention.workspace_bytes(case.cache, h(q), h(ints[0]), BF16)
    space = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")

    def run():
        attention.launch_ref(ComputeClient.current(), case.cache, h(q), h(y), *(h(t) for t in ints), BF16, workspace=space.data_ptr(), workspace_size=size)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:  # both with the same workspace
        with torch.cuda.graph(graph):
            run()
    for it in range(4):
        ints[2].copy_(torch.tensor([tokens + 100 * it, 2000 - 300 * it, 130 - 20 * it], dtype=torch.int32))
        q.mul_(1.1)
        for graph in graphs:
            y.fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            y.fill_(6.0)
            run()
            torch.cuda.synchronize()
            assert torch.equal(got, y), it


def test_two_streams_with_workspaces_of_their_own(oracle):
    import torch

    cases = [Attention(oracle, seed, [(1, 5000)] * 3, 8, 1, 128, 64, BF16, scheme("q8")) for seed in (1, 2)]
    alone = [c.call() for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    held = []
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                ints = [torch.from_numpy(a).cuda() for a in (c.table, c.offsets, c.lengths)]
                q, y = c.q.cuda(), torch.empty_like(c.q, device="cuda")
                size = attention.workspace_bytes(c.cache, h(q), h(ints[0]), BF16)
                space = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
                held.append((ints, q, y, space))
                attention.launch_ref(ComputeClient.current(), c.cache, h(q), h(y), *(h(t) for t in ints), BF16, Scores(), space.data_ptr(), size)
    torch.cuda.synchronize()
    for i, (_, _, y, _) in enumerate(held):
        assert torch.equal(y, alone[i % 2])


def test_a_cache_beyond_4_gib(oracle):
    """Pages whose bytes start past 2^32, with a query whose keys all lie there."""
    import torch
    from cubek_amd import Cache, TensorHandleRef

    case = Attention(oracle, 2, [(1, 64), (40, 64)], 2, 1, 64, 16, BF16, scheme("q8"))
    page_bytes, pages = 16 * 64, (5 << 30) // (16 * 64)
    big = torch.zeros((pages, 1, 16, 64), dtype=torch.uint8, device="cuda")
    first = pages - case.k.stored.shape[0]
    stored = []
    for t in (case.k.stored, case.v.stored):
        big_t = big if not stored else torch.zeros_like(big)
        big_t[first:] = t
        stored.append(big_t)
    scales = [torch.zeros((pages, 1, 16, 2), dtype=torch.float32, device="cuda") for _ in range(2)]
    for t, own in zip(scales, (case.k.scales, case.v.scales)):
        t[first:] = own
    plain = case.call()
    case.cache = Cache(h(stored[0]), h(stored[1]), case.cache.scheme, h(scales[0]), h(scales[1]))
    case.table = np.where(case.table < 0, case.table, case.table + first).astype(np.int32)
    assert torch.equal(case.call(), plain)

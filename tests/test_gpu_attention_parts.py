"""cq_attention where keys are shared out: parts of unlike sequences, tiles of one part beside tiles of several, workspaces of any size, the same bits in every call."""
import numpy as np
import pytest

from attention_reference import Attention, h
from cubek_amd import ComputeClient, ElemType, QuantStore, QuantValue, Scores, attention
from matmul_reference import check_rounded, scheme_of

pytestmark = pytest.mark.gpu
F16, BF16 = ElemType.F16, ElemType.BF16
V, U32, NATIVE = QuantValue, QuantStore.U32, QuantStore.Native
CODES = {"q8": (V.Q8S, NATIVE), "q4": (V.Q4S, U32), "e4m3": (V.E4M3, NATIVE), "e5m2": (V.E5M2, NATIVE), "e2m1": (V.E2M1, NATIVE), "floats": None}


def scheme(name, block, param=0):
    return None if CODES[name] is None else scheme_of(CODES[name][0], [block], param, CODES[name][1])


@pytest.mark.parametrize("name", ["q8", "q4", "floats"])
@pytest.mark.parametrize("tokens", [1, 3])
def test_many_sequences_of_unlike_lengths(oracle, name, tokens):
    """More parts than the GPU holds at once, the later ones smaller."""
    sequences = [(tokens, tokens + 80 * i) for i in range(70)]
    Attention(oracle, 1, sequences, 8, 8, 32, 16, BF16, scheme(name, 32)).check()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("name", ["q8", "e2m1", "floats"])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_prompts_of_one_part_beside_prompts_of_several(oracle, dim, name, elem):
    case = Attention(oracle, 2, [(140, 3300), (90, 90), (0, 500), (200, 1100), (1, 2500)], 4, 2, dim, 64, elem, scheme(name, 64))
    case.check()
    case.check("window", window=1500, cap=20.0)


@pytest.mark.parametrize("tokens,lengths", [(1, (9000, 700, 30)), (50, (4000, 3000, 50))])
def test_rows_of_nobody_stay_where_keys_are_shared_out(oracle, tokens, lengths):
    import torch

    case = Attention(oracle, 4, [(tokens, n) for n in lengths], 4, 2, 64, 16, BF16, scheme("q8", 64))
    q = torch.zeros((case.tokens + 9, 4, 64), dtype=torch.bfloat16, device="cuda")
    q[4:4 + case.tokens] = case.q.cuda()
    y = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    want, bound = case.want()
    case.offsets = case.offsets + 4
    case.call(q=q, y=y)
    check_rounded(y[4:4 + case.tokens].double().cpu().numpy(), want, bound, BF16)
    assert (y[:4] == 9).all() and (y[4 + case.tokens:] == 9).all()


@pytest.mark.parametrize("tokens", [1, 8, 120])
def test_workspaces_smaller_than_asked_for(oracle, tokens):
    import torch

    case = Attention(oracle, 5, [(tokens, 6000), (tokens, 2000)], 8, 2, 64, 16, BF16, scheme("q8", 32))
    want, bound = case.want()
    q, ints = case.q.cuda(), [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (case.table, case.offsets, case.lengths)]
    size = attention.workspace_bytes(case.cache, h(q), h(ints[0]), BF16)
    assert size > 0
    for part in (1.0, 0.6, 0.3, 0.1, 0.01):
        room = int(size * part) // 16 * 16
        space = torch.full((size + 4096,), 255, dtype=torch.uint8, device="cuda")
        y = torch.full(q.shape, 77.0, dtype=q.dtype, device="cuda")
        attention.launch_ref(ComputeClient.current(), case.cache, h(q), h(y), *(h(t) for t in ints), BF16, Scores(), workspace=space.data_ptr(), workspace_size=room)
        torch.cuda.synchronize()
        check_rounded(y.double().cpu().numpy(), want, bound, BF16, part)
        assert (space[room:] == 255).all(), part  # nothing is written behind it


@pytest.mark.parametrize("dim,block", [(64, 32), (64, 64), (128, 32), (128, 128), (224, 32), (256, 64)])
@pytest.mark.parametrize("name", [n for n in CODES if n != "floats"])
@pytest.mark.parametrize("tokens", [1, 7, 80])
def test_results_of_f16_over_codes(oracle, dim, block, name, tokens):
    """Codes are exact in f16 and so are queries of f16: between them and a result stand the rounding of a weight with its scale (2^-11 of each
    product), sums in f32 and the result's own rounding."""
    case = Attention(oracle, 3, [(tokens, 300), (tokens, tokens + 64)], 4, 1, dim, 16, F16, scheme(name, block))
    case.u = 0.0
    want, bound = case.want()
    entries, case.v.entries = case.v.entries, np.abs(case.v.entries)
    size, _ = case.want()
    case.v.entries = entries
    check_rounded(case.call().double().cpu().numpy(), want, bound + size * 2.0 ** -11 * (1 + 2.0 ** -10), F16, (name, block))


@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_same_bits_in_every_call(oracle, dim, name, elem):
    import torch

    for sequences in ([(1, 1), (1, 130), (1, 64), (1, 1900)], [(5, 35), (7, 300), (1, 64), (9, 1400)], [(150, 150), (1, 2100), (70, 900)]):
        case = Attention(oracle, 0, sequences, 4, 2, dim, 16, elem, scheme(name, 32))
        first = case.call()
        for _ in range(6):
            assert torch.equal(case.call().view(torch.int16), first.view(torch.int16)), sequences


@pytest.mark.parametrize("length", [33, 700])
@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_slopes_on_either_side_of_the_position(oracle, length, tokens):
    """Keys of a prefix stand before and behind the position; a bias of both signs."""
    slopes = np.array([0.5, -0.01, 2.0 ** -8, 0.0], np.float32)
    n = min(tokens, length)
    case = Attention(oracle, 7, [(n, length), (n, length + 40)], 4, 2, 128, 16, F16, scheme("q8", 32))
    case.check("prefix", slopes=slopes, prefix=[length, 5])
    case.check("causal", slopes=slopes)
    case.check("capped", slopes=slopes, prefix=[length, length], cap=4.0, window=25)


@pytest.mark.parametrize("tokens", [2, 12, 200])
@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_a_last_key_that_is_not_a_number(oracle, tokens, name, elem):
    """The last token sees it, the ones in front of it do not, in a sequence of several parts and in one of one."""
    case = Attention(oracle, 6, [(tokens, 3000), (tokens, tokens + 40)], 4, 2, 128, 16, elem, scheme(name, 32))
    want, bound = case.want()
    for s, (_, length) in enumerate(case.sequences):
        for pool in (case.k, case.v):
            at = (int(case.table[s, (length - 1) // 16]), slice(None), (length - 1) % 16)
            if pool.scales is None:
                pool.stored[at] = float("nan")
            else:
                pool.scales[at] = float("nan")
    got = case.call().double().cpu().numpy()
    for s in range(2):
        a, b = case.offsets[s], case.offsets[s + 1] - 1
        check_rounded(got[a:b], want[a:b], bound[a:b], elem, s)
        assert np.isnan(got[b]).all()

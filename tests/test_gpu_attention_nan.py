"""cq_attention of queries, keys and values that are not numbers, in parts of the keys that hold nothing else: a token whose sum is not a number gets no number,
however its keys are shared out."""
import numpy as np
import pytest

from attention_reference import Attention
from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import check_rounded, scheme_of

pytestmark = pytest.mark.gpu
F16, BF16 = ElemType.F16, ElemType.BF16
NATIVE, U32 = QuantStore.Native, QuantStore.U32
SCHEMES = {"floats": None, "q8": scheme_of(QuantValue.Q8S, [32], 0, NATIVE), "q4": scheme_of(QuantValue.Q4S, [32], 0, U32), "e4m3": scheme_of(QuantValue.E4M3, [64], 0, NATIVE)}

# new tokens and keys: one part, two and about 64 of attention_few_kernel, one, two and several of attention_many_kernel
LENGTHS = [(1, 100), (1, 600), (1, 20011), (3, 9000), (90, 120), (90, 2000), (90, 9000)]


@pytest.mark.parametrize("tokens,length", LENGTHS)
@pytest.mark.parametrize("name", SCHEMES)
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_queries_that_are_not_numbers(oracle, tokens, length, name, elem):
    """A query with one entry that is not a number sees no score that is one; the other heads' queries are as they were."""
    case = Attention(oracle, 3, [(tokens, length), (tokens, tokens + 30)], 4, 1, 64, 16, elem, SCHEMES[name])
    want, bound = case.want()
    odd = [(0, 1), (tokens - 1, 2), (tokens, 0)]  # (token, head); the second sequence has one part
    for token, head in odd:
        case.q[token, head, 5] = float("nan")
        want[token, head] = np.nan
    for workspace in (True, False):
        check_rounded(case.call(workspace).double().cpu().numpy(), want, bound, elem, workspace)


@pytest.mark.parametrize("tokens,length", [(1, 600), (1, 20011), (3, 9000), (90, 9000)])
@pytest.mark.parametrize("first,last", [(0.0, 0.5), (0.45, 0.9), (0.0, 1.0)])
@pytest.mark.parametrize("name", SCHEMES)
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_parts_whose_keys_are_not_numbers(oracle, tokens, length, first, last, name, elem):
    """All tokens see half of their keys, or all of them, as not numbers, whole parts among them; another sequence's are numbers."""
    case = Attention(oracle, 4, [(tokens, length), (tokens, 700)], 4, 2, 64, 16, elem, SCHEMES[name])
    want, bound = case.want()
    keys = np.arange(int(first * length), int(last * length))
    at = (case.table[0, keys // 16], slice(None), keys % 16)
    held = case.k.stored if case.k.scales is None else case.k.scales
    held[at] = float("nan")
    want[:tokens] = np.nan
    for row in range(tokens):  # of a prompt, those in front of these keys do not see them
        if length - tokens + row < keys[0]:
            want[row] = case.want()[0][row]
    for workspace in (True, False):
        check_rounded(case.call(workspace).double().cpu().numpy(), want, bound, elem, workspace)


@pytest.mark.parametrize("tokens,length", [(1, 600), (1, 20011), (90, 9000)])
@pytest.mark.parametrize("name", ["floats", "q8"])
def test_the_first_parts_alone_are_not_numbers(oracle, tokens, length, name):
    """Wherever the parts' ends are: one part, or some, that hold nothing else beside parts of numbers."""
    for last in (64, 192, 256, 320, 512, 1024, 2048):
        case = Attention(oracle, 6, [(tokens, length)], 2, 1, 64, 16, BF16, SCHEMES[name])
        keys = np.arange(min(last, length))
        at = (case.table[0, keys // 16], slice(None), keys % 16)
        held = case.k.stored if case.k.scales is None else case.k.scales
        held[at] = float("nan")
        assert np.isnan(case.call().double().cpu().numpy()).all(), last


@pytest.mark.parametrize("tokens,length", [(1, 20011), (90, 9000)])
def test_what_is_not_a_number_is_one_for_every_workspace(oracle, tokens, length):
    """The same answer in one part and in as many as there is room for, and zeros only of tokens that see nothing."""
    case = Attention(oracle, 5, [(tokens, length), (2, 2)], 2, 1, 64, 16, BF16, SCHEMES["q8"])
    case.q[:tokens] = float("nan")
    case.lengths[1] = 0
    for workspace in (True, False):
        got = case.call(workspace).double().cpu().numpy()
        assert np.isnan(got[:tokens]).all() and (got[tokens:] == 0).all(), workspace

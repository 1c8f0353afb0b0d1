"""cq_attention where numbers in device memory and the fields of cq_scores take their lowest and highest values."""
import numpy as np
import pytest

from attention_reference import Attention
from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import check_rounded, scheme_of

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
Q8 = scheme_of(QuantValue.Q8S, [32], 0, QuantStore.Native)


@pytest.mark.parametrize("elem", [BF16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("scheme", [Q8, None], ids=["q8", "floats"])
def test_prefixes_outside_of_the_sequence(oracle, elem, tokens, scheme):
    """The lowest numbers are no prefix, the highest the whole sequence; without a window and within one."""
    case = Attention(oracle, 1, [(tokens, 200), (tokens, 200), (tokens, 170), (tokens, tokens + 1), (tokens, 190)], 4, 2, 64, 16, elem, scheme)
    given = [-2 ** 31, 2 ** 31 - 1, -2 ** 31 + 1, -1, 0]
    for window in (0, 30):
        want, bound = case.want(prefix=[0, 200, 0, 0, 0], window=window)
        got = case.call(prefix=given, window=window).double().cpu().numpy()
        check_rounded(got, want, bound, elem, window)


@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("scheme", [Q8, None], ids=["q8", "floats"])
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e10, 1e30, 3e38])
def test_large_caps(oracle, elem, tokens, scheme, cap):
    """Caps far above the scores: they keep the scores' own bits.  tanh of x is off by 2^-20 of itself: 2^-19 of the score with the roundings around it, instead of the bound's
    2^-20 of the cap; weights go by e^(cap tanh(t / cap)) and not e^t, which makes no difference to the bound's weights where |t| < 30: t^3 / (3 cap^2) < 0.01."""
    case = Attention(oracle, 2, [(tokens, 200), (tokens, tokens)], 4, 2, 64, 16, elem, scheme, spread=2.0)
    held, case.v.entries = case.v.entries, np.abs(case.v.entries)
    size, _ = case.want(cap=cap)
    case.v.entries = held
    want, _ = case.want(cap=cap)
    _, bound = case.want()
    most = 64 ** -0.5 * case.q.double().abs().sum(-1).numpy()[..., None] * np.abs(case.k.entries).max()
    got = case.call(cap=cap).double().cpu().numpy()
    check_rounded(got, want, 1.02 * bound + 2 * size * 2.0 ** -19 * np.minimum(most, 30.0), elem)


@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("scheme", [Q8, None], ids=["q8", "floats"])
def test_caps_of_the_scores_size_and_of_all_sizes(oracle, tokens, scheme):
    """Scores on both sides of a quarter of the cap, and caps down to f32's lowest numbers, which leave all weights alike."""
    for elem in (BF16, F16, F32):
        case = Attention(oracle, 3, [(tokens, 200), (tokens, tokens)], 4, 2, 64, 16, elem, scheme, spread=30.0)
        for cap in (64.0, 65.0, 150.0, 1000.0):
            case.check(cap, cap=cap)
        for cap in (1e-3, 1e-30, 1.2e-38, 1e-42, 2.0 ** -149):
            case.check(cap, cap=cap)
            case.check((cap, "no scale"), cap=cap, scale=0.0)

"""cq_attention where numbers in device memory and the fields of cq_scores take their lowest and highest values."""
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

"""What cq_attention rounds to 16 bits on its way to a result of bf16.

A result's own rounding is off by 2^-9 of it at most, and by 2^-9 / 1.18 of its norm where mantissas are spread evenly (the mean square over a binade: 1/12 of a step squared, over 1 to 2).
What is left of 2^-9 of the norm, in squares, is 2^-9 (1 - 1 / 1.39)^(1/2) = 2^-9.9 for all that is in front."""
import numpy as np
import pytest

from attention_reference import Attention
from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import check_rounded, scheme_of

pytestmark = pytest.mark.gpu
BF16 = ElemType.BF16


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_keys_scale_is_not_rounded_by_itself(oracle, dim):
    """Scores of a normal distribution, 1.5 wide, of keys whose scales have 24 bits.  A key's entries, rounded each for itself to 2^-11 (2^-12.5 in the mean square, evenly spread), move
    its score by dim^(-1/2) of that many parts of it, at most 2^-12.5 * 4 or so, where weights are; its scale, rounded, by 2^-12.3 times the score, which for the keys that have most weight
    lies around 2 * 1.5^2 and with that alone past 2^-9.9 of the norm."""
    case = Attention(oracle, 1, [(300, 2048)], 4, 1, dim, 16, BF16, scheme_of(QuantValue.E4M3, [dim // 2 if dim == 256 else dim], 0, QuantStore.Native))
    codes = np.random.default_rng(2).normal(0, 150, case.k.entries.shape).clip(-440, 440)
    import torch

    stored = torch.from_numpy(codes).to(torch.float8_e4m3fn)
    for pool in (case.k, case.v):
        pool.stored.copy_(stored.view(torch.uint8).cuda())
        pool.scales.copy_(torch.tensor(np.random.default_rng(3).uniform(0.5, 1.5, tuple(pool.scales.shape)) / 150, dtype=torch.float32))
        pool.entries = stored.double().numpy() * pool.scales.double().cpu().repeat_interleave(dim // pool.scales.shape[-1], -1).numpy()
    case.q = (case.q.double() * 1.5 / 1.04).to(case.q.dtype)  # of keys 1.04 wide
    want, _ = case.want()
    got = case.call().double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2.0 ** -9 * np.linalg.norm(want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,length", [(1, 400), (1, 3000), (9, 700), (30, 500)])
def test_weights_over_a_cache_of_bf16_have_16_bits(oracle, dim, tokens, length):
    """Products of bf16 are exact in f32; a weight is two numbers of bf16, off by 2^-18 of it: what the second leaves of what the first leaves."""
    case = Attention(oracle, 2, [(tokens, length), (tokens, tokens + 5)], 2, 1, dim, 16, BF16, None)
    case.u = 0.0
    want, bound = case.want()
    held, case.v.entries = case.v.entries, np.abs(case.v.entries)
    size, _ = case.want()
    case.v.entries = held
    check_rounded(case.call().double().cpu().numpy(), want, bound + size * 2.0 ** -17, BF16)

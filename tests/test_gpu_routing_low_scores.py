"""Routing by the sigmoid where the scores are small: finite logits far below 0 keep their quotients, masked experts weigh nothing.  The checks are those
of test_gpu_routing.py, in 64 bits."""
import numpy as np
import pytest
import torch

from cubek_amd import ElemType, Score
from matmul_reference import TORCH
from test_gpu_routing import check, route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("tokens,num,chosen", [(9, 8, 3), (300, 100, 7), (40, 256, 20)])
def test_finite_logits_far_below_zero(tokens, num, chosen, normalize):
    rng = np.random.default_rng(num)
    for elem in (ElemType.F32, ElemType.BF16, ElemType.F16):
        for middle, spread in ((-80.0, 3.0), (-90.0, 0.0), (-95.0, 8.0), (-200.0, 40.0), (-690.0, 6.0), (-1.0, 2.0)):
            x = torch.tensor(middle + spread * rng.uniform(-1, 1, (tokens, num)), dtype=torch.float32).to(TORCH[elem])
            got = route(x.cuda(), chosen, elem, Score.Sigmoid, normalize)
            check(x.double().numpy(), chosen, Score.Sigmoid, normalize, got)
            if normalize:  # nobody loses its experts: the weights of a token are a whole
                assert np.abs(got[0].sum(1) - 1.0).max() < 2.0 ** -13


@pytest.mark.parametrize("tokens", [6, 300])
def test_masked_experts_weigh_nothing(tokens):
    """Masks of a type's lowest value do as those of -infinity, beside logits that are small themselves, and where nothing else is left."""
    rng = np.random.default_rng(1)
    for elem in (ElemType.F32, ElemType.BF16, ElemType.F16):
        lowest = torch.finfo(TORCH[elem]).min
        x = torch.tensor(rng.uniform(-130, -90, (tokens, 16)), dtype=torch.float32).to(TORCH[elem])
        x[:, 3:] = lowest
        x[1] = lowest
        x[2, 3:] = float("-inf")
        weights = route(x.cuda(), 5, elem, Score.Sigmoid, True)[0]
        assert (weights[1] == 0.0).all() and (weights[:, 3:] == 0.0).all()
        rest = np.delete(np.arange(tokens), 1)
        p = np.exp(-np.sort(-x.double().numpy()[rest, :3], 1))
        want = p / p.sum(1, keepdims=True)
        assert np.abs(weights[rest][:, :3] - want).max() < 2.0 ** -13

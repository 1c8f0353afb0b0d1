"""cq_attention at drawn sizes, codes, scores and orders against numpy in 64 bits (CQ_RANDOM_ATTENTION: how many)."""
import os
import random

import numpy as np
import pytest

from attention_reference import Attention
from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import scheme_of

pytestmark = pytest.mark.gpu
V, U32, NATIVE = QuantValue, QuantStore.U32, QuantStore.Native
CODES = [None, None, (V.Q8S, NATIVE), (V.Q8F, U32), (V.Q4S, U32), (V.E4M3, NATIVE), (V.E5M2, NATIVE), (V.E2M1, NATIVE), (V.E2M1, U32), (V.E2M1_OCP, U32)]


def drawn(seed):
    rng = random.Random(seed)
    code = rng.choice(CODES)
    dim, block = rng.choice([(32, 32), (64, 32), (64, 64), (96, 32), (128, 32), (128, 64), (128, 128), (160, 32), (192, 64), (224, 32), (256, 64), (256, 128), (80, 40), (48, 16), (136, 8)])
    kv_heads, group = rng.choice([(1, 1), (2, 1), (1, 3), (2, 4), (1, 8), (3, 5), (1, 16), (2, 7)])
    kind = rng.choice(["single", "draft", "prompt", "mixed"])
    new = {"single": (1, 1), "draft": (2, 9), "prompt": (30, 200), "mixed": (0, 60)}[kind]
    past = rng.choice([0, 30, 400, 3000])
    sequences = []
    for _ in range(rng.choice([1, 1, 2, 3, 5, 9, 70 if kind == "single" else 4])):
        n = rng.randint(*new)
        sequences.append((n, n + rng.randint(0, past)))
    if sum(n for n, _ in sequences) == 0:
        sequences[0] = (3, 3 + sequences[0][1])
    scores = {}
    if rng.random() < 0.3:
        scores["cap"] = rng.choice([2.0, 30.0, 64.0, 100.0])
    if rng.random() < 0.3:
        scores["window"] = rng.choice([1, 7, 64, 300, 2 ** 32 - 1])
    if rng.random() < 0.3:
        scores["slopes"] = np.array([rng.choice([0.0, 0.5, 2.0 ** -8, -0.01]) for _ in range(kv_heads * group)], np.float32)
    if rng.random() < 0.3:
        scores["prefix"] = [rng.choice([-2 ** 31, -1, 0, length // 2, length]) for _, length in sequences]
    if rng.random() < 0.2:
        scores["scale"] = rng.choice([0.0, -0.2, 0.01, 1.0])
    elem = rng.choice([ElemType.BF16, ElemType.BF16, ElemType.F16, ElemType.F16, ElemType.F32])
    scheme = None if code is None else scheme_of(code[0], [block], rng.choice([0, 1, 2]), code[1])
    return dict(sequences=sequences, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 16, 32, 64, 128, 1, 8, 24]), elem=elem, scheme=scheme,
                order=rng.choice(["heads", "slots", "gaps"])), scores, rng.random() < 0.7


@pytest.mark.parametrize("seed", range(int(os.environ.get("CQ_RANDOM_ATTENTION", 60))))
def test_drawn_calls(oracle, seed):
    case, scores, workspace = drawn(seed)
    Attention(oracle, seed, **case).check((case, scores), workspace, **scores)

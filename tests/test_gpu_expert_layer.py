"""examples/expert_layer.py, stage by stage: each stage's inputs as the GPU left them, its results against 64 bits within the bounds of
matmul_reference.py, eagerly and from a graph that is replayed on other inputs."""
import os
import sys

import numpy as np
import pytest

from cubek_amd import Activation, ElemType
from matmul_reference import Product, check_rounded, dequantized

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
pytestmark = pytest.mark.gpu
BF16, F32 = ElemType.BF16, ElemType.F32


def wide(t):
    return t.double().cpu().numpy()


def check_layer(oracle, layer, x, b):
    def weights(w):
        codes = w.codes.cpu().numpy().view(np.uint32)
        shape = codes.shape[:-1] + (codes.shape[-1] * w.scheme.num_quants(),)
        return dequantized(oracle, codes, w.scales.cpu(), shape, BF16, w.scheme)
    tokens, chosen = b["experts"].shape
    logits, weight, slots = wide(b["logits"]), wide(b["weights"]), b["slots"].cpu().numpy()
    Product(wide(x), weights(layer.router)).check(logits)
    order = np.argsort(-logits, axis=1, kind="stable")[:, :chosen]
    chose, at, rows = b["experts"].cpu().numpy(), b["offsets"].cpu().numpy(), b["rows"].cpu().numpy()
    assert np.array_equal(chose, order)
    best = np.take_along_axis(logits, order, 1)
    soft = np.exp(best - best[:, :1])
    assert np.abs(weight - soft / soft.sum(1, keepdims=True)).max() < 2.0 ** -19  # a dozen f32 operations on numbers up to 1
    assert sorted(slots.reshape(-1)) == list(range(tokens * chosen)) and np.array_equal(rows[slots], np.repeat(np.arange(tokens)[:, None], chosen, 1))
    assert np.array_equal(np.searchsorted(at, slots, side="right") - 1, chose)
    gate_up, down, inner, out = weights(layer.gate_up), weights(layer.down), wide(b["inner"]), wide(b["out"])
    for e in range(layer.num_experts):
        part = slice(at[e], at[e + 1])
        if at[e] < at[e + 1]:
            Product(wide(x)[rows[part]], gate_up[e], Activation.Silu, True, y_elem=BF16).check(inner[part], e)
            Product(inner[part], down[e], y_elem=BF16).check(out[part], e)
    terms = weight[:, :, None] * out[slots]
    want = wide(x) + terms.sum(1)
    check_rounded(wide(b["y"]), want, (chosen + 2) * 2.0 ** -24 * (np.abs(wide(x)) + np.abs(terms).sum(1)), BF16)


@pytest.mark.parametrize("tokens", [1, 16, 70, 400])
def test_layer(oracle, tokens):
    import torch

    from expert_layer import ExpertLayer

    layer = ExpertLayer(hidden=256, inner=160, num_experts=12, chosen=3)
    buffers = layer.buffers(tokens)
    x = torch.randn((tokens, 256), generator=torch.Generator("cuda").manual_seed(tokens), device="cuda").to(torch.bfloat16)
    layer(x, buffers)
    torch.cuda.synchronize()
    check_layer(oracle, layer, x, buffers[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, buffers)
    for k in range(3):
        x.copy_(torch.randn((tokens, 256), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        check_layer(oracle, layer, x, buffers[0])

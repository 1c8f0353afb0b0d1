"""Products of more than 2^22 workgroups of the smallest tile, where a launch of the larger ones still holds all: every result is written, tokens
from all over against 64 bits."""
import numpy as np
import pytest
import torch

from cubek_amd import ComputeClient, ElemType, Epilogue, QuantValue, TensorHandleRef, experts
from matmul_reference import Product, dequantized, random_weight, scheme_of
from test_gpu_matmul import floats, offsets_of, on_gpu, run_matmul, wide

pytestmark = pytest.mark.gpu
BF16, F32 = ElemType.BF16, ElemType.F32
h = TensorHandleRef.from_torch


@pytest.mark.parametrize("tokens", [16000, 17000])
def test_long_prompt_through_a_head(oracle, tokens):
    rng = np.random.default_rng(tokens)
    rows, cols = 128256, 64
    scheme = scheme_of(QuantValue.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (rows, cols))
    x, bias = floats(rng, (tokens, cols), BF16), floats(rng, (rows,), F32)
    gb, y = bias.cuda(), torch.full((tokens, rows), float("nan"), dtype=torch.bfloat16, device="cuda")
    run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), BF16, BF16, Epilogue(bias=h(gb)), y)
    assert not y.isnan().any()
    w = dequantized(oracle, codes, scales, (rows, cols), BF16, scheme)
    for part in (slice(0, 9), slice(tokens // 2, tokens // 2 + 9), slice(tokens - 9, tokens)):
        Product(wide(x)[part], w, bias=wide(bias), y_elem=BF16).check(wide(y[part].cpu()), part)


def test_long_prompt_through_experts(oracle):
    rng = np.random.default_rng(0)
    sizes, rows, cols = [100, 0, 30000, 9871], 60000, 64
    scheme = scheme_of(QuantValue.Q8S, [32])
    codes, scales = random_weight(rng, scheme, (len(sizes), rows, cols))
    x, at = floats(rng, (sum(sizes), cols), BF16), offsets_of(sizes)
    gc, gs, gx, go = on_gpu(codes), scales.cuda(), x.cuda(), torch.from_numpy(at).cuda()
    y = torch.full((sum(sizes), rows), float("nan"), dtype=torch.bfloat16, device="cuda")
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), BF16, BF16)
    assert not y.isnan().any()
    w = dequantized(oracle, codes, scales, (len(sizes), rows, cols), BF16, scheme)
    for e, p in ((0, 0), (0, 91), (2, 100), (2, 15000), (2, 30091), (3, 30100), (3, 39962)):
        part = slice(p, p + 9)
        Product(wide(x)[part], w[e], y_elem=BF16).check(wide(y[part].cpu()), p)

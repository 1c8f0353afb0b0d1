"""The stride of a dimension of one entry counts nothing: one token, one row of a weight or of its scales, one expert, whatever their strides say,
take the kernel that contiguous tensors take, so that the results have the same bits."""
import numpy as np
import pytest
import torch

from cubek_amd import ComputeClient, ElemType, QuantValue, TensorHandleRef, experts
from matmul_reference import random_weight, scheme_of
from test_gpu_matmul import floats, on_gpu, run_matmul

pytestmark = pytest.mark.gpu
BF16, F32 = ElemType.BF16, ElemType.F32
h = TensorHandleRef.from_torch


def with_stride(t, stride):
    """`t` with another stride of its first dimension of one entry."""
    assert t.shape[0] == 1
    return t.as_strided(t.shape, (stride,) + t.stride()[1:])


@pytest.mark.parametrize("rows", [1, 500])
def test_one_token_or_row(rows):
    rng = np.random.default_rng(rows)
    scheme = scheme_of(QuantValue.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (rows, 2048))
    x = floats(rng, (1, 2048), BF16).cuda()
    gc, gs = on_gpu(codes), scales.cuda()
    want = run_matmul(gc, gs, scheme, x, BF16, F32)
    for stride in (1, 3, 1 << 40):
        assert torch.equal(want, run_matmul(gc, gs, scheme, with_stride(x, stride), BF16, F32)), stride
        if rows == 1:
            assert torch.equal(want, run_matmul(with_stride(gc, stride), with_stride(gs, stride), scheme, x, BF16, F32)), stride


@pytest.mark.parametrize("tokens", [1, 40])
def test_one_expert(tokens):
    rng = np.random.default_rng(tokens)
    scheme = scheme_of(QuantValue.Q8S, [32])
    codes, scales = random_weight(rng, scheme, (1, 200, 1024))
    x, offsets = floats(rng, (tokens, 1024), BF16).cuda(), torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    gc, gs = on_gpu(codes), scales.cuda()

    def run(c, s):
        y = torch.full((tokens, 200), 9.0, device="cuda")
        experts.launch_ref(ComputeClient.current(), h(c), h(s), scheme, h(x), h(offsets), h(y), BF16, F32)
        return y
    want = run(gc, gs)
    for stride in (1, 3, 1 << 40):
        assert torch.equal(want, run(with_stride(gc, stride), with_stride(gs, stride))), stride

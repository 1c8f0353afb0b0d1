"""A weight of more rows than one launch of the general kernel has threads for, in f32: rows on both sides of that, and the last one."""
import pytest
import torch

from cubek_amd import ComputeClient, ElemType, QuantScheme, QuantStore, QuantValue, TensorHandleRef, matmul

pytestmark = pytest.mark.gpu
h = TensorHandleRef.from_torch


def test_rows_beyond_a_launch():
    rows, cols = (1 << 28) + 77, 8
    scheme = QuantScheme.default().with_value(QuantValue.Q8S).with_store(QuantStore.Native)
    codes = torch.randint(-100, 100, (rows, cols), dtype=torch.int8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    scale = torch.full((1,), 0.5, device="cuda")
    x = torch.arange(1, 9, dtype=torch.float32, device="cuda")[None]
    y = torch.full((1, rows), float("nan"), device="cuda")
    matmul.launch_ref(ComputeClient.current(), h(codes.view(torch.uint8)), h(scale), scheme, h(x), h(y), ElemType.F32, ElemType.F32)
    for first in range(0, rows, 1 << 24):  # whole numbers and halves: exact in f32
        part = slice(first, min(rows, first + (1 << 24)))
        assert torch.equal(y[0, part], (codes[part].float() * x).sum(1) * 0.5)

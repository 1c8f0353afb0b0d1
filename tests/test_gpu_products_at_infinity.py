"""What stands behind a product of an infinite x, of an infinite bias and of a sum that leaves the range of f32: the values that the formulas
of include/cubek_matmul.h have there, infinities and NaN exactly, by every kernel and for every activation."""
import numpy as np
import pytest
import torch

from cubek_amd import Activation, ElemType, Epilogue, QuantStore, QuantValue, TensorHandleRef
from matmul_reference import TORCH, Product, dequantized, random_weight, scheme_of
from test_gpu_matmul import floats, on_gpu, run_matmul, wide

pytestmark = pytest.mark.gpu
F32, BF16 = ElemType.F32, ElemType.BF16
h = TensorHandleRef.from_torch


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", list(Activation), ids=lambda a: a.name)
def test_infinite_x_and_bias(oracle, activation, gated):
    """One, 16 and 40 tokens, 300 and 4 in f32: the kernels of a decode step, the tiles with and without shared columns, the general one."""
    scheme = scheme_of(QuantValue.Q4S, [32], 0, QuantStore.U32)
    n, cols = 72, 544
    rows = 2 * n if gated else n
    for tokens, elem, y_elem in ((1, BF16, F32), (16, BF16, BF16), (40, BF16, F32), (300, BF16, BF16), (4, F32, F32)):
        rng = np.random.default_rng(tokens)
        codes, scales = random_weight(rng, scheme, (rows, cols))
        x, bias = floats(rng, (tokens, cols), elem), floats(rng, (rows,), F32)
        x[0, cols - 1] = float("inf")
        x[tokens - 1, 3] = float("-inf")  # one token: +inf and -inf meet
        bias[5], bias[6], bias[rows - 2], bias[rows - 1] = float("inf"), float("-inf"), float("inf"), float("-inf")
        gb = bias.cuda()
        y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, y_elem, Epilogue(activation, gated, bias=h(gb)))
        want = Product(wide(x), dequantized(oracle, codes, scales, (rows, cols), elem, scheme), activation, gated, wide(bias), y_elem=y_elem)
        assert np.isinf(want.y).any() and np.isnan(want.y).any()
        want.check(wide(y.cpu()), (tokens, elem.name))


@pytest.mark.parametrize("activation", list(Activation), ids=lambda a: a.name)
def test_sums_out_of_range(activation):
    """Sums of 64 products of 2^126: infinite in f32, and an activation of infinity behind them."""
    scheme = scheme_of(QuantValue.Q8S, None)
    codes = torch.full((32, 16), 0x01010101, dtype=torch.int32)  # ones
    codes[16:] = -1  # minus one in every field
    for tokens, elem in ((1, BF16), (40, BF16), (200, BF16), (2, F32)):
        x = torch.full((tokens, 64), 2.0 ** 126, dtype=TORCH[elem])
        y = run_matmul(codes.cuda(), torch.ones((1,), device="cuda"), scheme, x.cuda(), elem, F32, Epilogue(activation)).cpu()
        assert (y[:, :16] == float("inf")).all(), (tokens, elem.name)
        low = y[:, 16:]
        if activation == Activation.Identity:
            assert (low == float("-inf")).all()
        elif activation == Activation.Relu:
            assert (low == 0.0).all()
        else:  # -inf times the 0 that the gate has there
            assert low.isnan().all()

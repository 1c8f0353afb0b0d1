"""Weights that are not ordinary numbers: scales that are infinite, NaN, denormal, -0 or beyond the range of the type of x, every code there is, e4m3 and
e5m2 infinities and NaN included.  Each enters as the value that dequantize stores, by every kernel."""
import numpy as np
import pytest
import torch

from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import PARAM, Product, dequantized, scheme_of
from test_gpu_matmul import floats, on_gpu, run_matmul, wide

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
U32, NATIVE = QuantStore.U32, QuantStore.Native
V = QuantValue
SPECIAL = [float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e-40, -3e-8, 7e4, 1e30, -2.0 ** -126, 2.0 ** -14]
SCHEMES = [(V.Q2S, [64], U32), (V.Q2F, None, U32), (V.Q4S, [32], U32), (V.Q4F, [16], U32), (V.Q8S, [32], U32), (V.Q8F, [64], NATIVE), (V.E2M1, [32], U32), (V.E2M1, [32], NATIVE),
           (V.E2M1_OCP, [64], U32), (V.E4M3, [32], NATIVE), (V.E5M2, [32], NATIVE), (V.E5M2, [16], NATIVE), (V.E4M3, [32], U32), (V.E5M2, [32], U32)]


@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("which", range(len(SCHEMES)))
def test_special_scales_and_codes(oracle, which, elem):
    value, block, store = SCHEMES[which]
    for param in (0, 1, 2):
        scheme = scheme_of(value, block, param, store)
        rows, cols = 3 * len(SPECIAL), 256
        rng = np.random.default_rng(which)
        stored = scheme.packed_shape((rows, cols))
        codes = rng.integers(0, 1 << 32, stored, dtype=np.uint64).astype(np.uint32) if store == U32 else rng.integers(0, 256, stored, dtype=np.uint64).astype(np.uint8)
        scales = torch.tensor(rng.uniform(0.25, 1.0, scheme.scales_shape((rows, cols))) * 2.0 ** -7, dtype=torch.float32)
        if block is None:
            variants = [torch.full_like(scales, s) for s in SPECIAL]
        else:  # row 3 k + 1 has the k-th in one block
            for k, s in enumerate(SPECIAL):
                scales[3 * k + 1, k % scales.shape[1]] = s
            variants = [scales]
        for scale in variants:
            scale = scale.to(PARAM[param])
            w = dequantized(oracle, codes, scale, (rows, cols), elem, scheme)
            for tokens in (1, 20, 70):
                x = floats(rng, (tokens, cols), elem)
                y = run_matmul(on_gpu(codes), scale.cuda(), scheme, x.cuda(), elem, F32)
                with np.errstate(invalid="ignore"):
                    Product(wide(x), w).check(wide(y.cpu()), (value.name, store.name, param, tokens))

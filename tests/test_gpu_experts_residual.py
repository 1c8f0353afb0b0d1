"""Products grouped by expert with a residual: apart from y and y itself, positions of nobody left as they are, by every kernel and with shared columns."""
import numpy as np
import pytest
import torch

from cubek_amd import Activation, ComputeClient, ElemType, Epilogue, QuantValue, TensorHandleRef, experts
from matmul_reference import Product, dequantized, random_weight, scheme_of
from test_gpu_matmul import floats, offsets_of, on_gpu, pitched, wide

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
h = TensorHandleRef.from_torch

# sizes of the experts, rows of y, columns, type of x and of y: a decode step, ragged tiles, long rows whose columns are shared, f32
CASES = [([1, 0, 3, 2], 100, 192, BF16, BF16), ([40, 0, 129, 7, 64], 131, 256, F16, F32), ([50, 20], 64, 6144, BF16, BF16), ([3, 30], 50, 96, F32, F32)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("which", range(len(CASES)))
def test_residual(oracle, which, gated, in_place):
    sizes, n, cols, elem, y_elem = CASES[which]
    rng = np.random.default_rng(which)
    scheme = scheme_of(QuantValue.Q4S, [32])
    e, positions, rows = len(sizes), sum(sizes) + 2, n * (2 if gated else 1)  # the last two are nobody's
    codes, scales = random_weight(rng, scheme, (e, rows, cols))
    x, residual = floats(rng, (positions, cols), elem), floats(rng, (positions, n), y_elem)
    at = offsets_of(sizes)
    gc, gs, gx, go = on_gpu(codes), scales.cuda(), x.cuda(), torch.from_numpy(at).cuda()
    y = pitched(residual.cuda(), 5) if in_place else torch.full((positions, n), 9.0, dtype=residual.dtype, device="cuda")
    before = y.clone()
    gr = y if in_place else pitched(residual.cuda(), 3)
    epi = Epilogue(Activation.Gelu, gated, residual=h(gr))
    size = experts.workspace_bytes(h(gc), scheme, h(y), elem, epi)
    space = torch.full((max(16, size),), 255, dtype=torch.uint8, device="cuda")
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), elem, y_elem, None, epi, workspace=space.data_ptr(), workspace_size=size)
    w, got = dequantized(oracle, codes, scales, (e, rows, cols), elem, scheme), wide(y.cpu())
    assert torch.equal(y[sum(sizes):], before[sum(sizes):])
    for i in range(e):
        part = slice(at[i], at[i + 1])
        if sizes[i]:
            Product(wide(x)[part], w[i], Activation.Gelu, gated, residual=wide(residual)[part], y_elem=y_elem).check(got[part], i)

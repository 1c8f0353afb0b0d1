"""cq_matmul_quantized and cq_experts_quantized against products of the oracle's dequantized weights in 64 bits; the tolerance is
derived in matmul_reference.py."""
import numpy as np
import pytest

from cubek_amd import Activation, ComputeClient, ElemType, Epilogue, QuantStore, QuantValue, TensorHandleRef, experts, matmul
from matmul_reference import TORCH, Product, dequantized, random_weight, scheme_of

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
U32, NATIVE = QuantStore.U32, QuantStore.Native
V = QuantValue
h = TensorHandleRef.from_torch


def floats(rng, shape, elem, scale=1.0):
    import torch

    return torch.tensor(rng.normal(0, scale, shape), dtype=torch.float32).to(TORCH[elem])


def wide(t):
    return t.double().numpy()


def on_gpu(codes):
    import torch

    return torch.from_numpy(codes.view(np.int32) if codes.dtype == np.uint32 else codes).cuda()


def pitched(t, pad, fill=float("nan")):
    """A view of the same values whose rows lie `pad` elements further apart, NaN between them."""
    import torch

    whole = torch.full(tuple(t.shape[:-1]) + (t.shape[-1] + pad,), fill, dtype=t.dtype, device="cuda")
    view = whole[..., :t.shape[-1]]
    view.copy_(t)
    return view


def run_matmul(codes, scales, scheme, x, elem, y_elem, epi=None, y=None, with_workspace=True):
    import torch

    epi = epi or Epilogue()
    n = codes.shape[0] // (2 if epi.gated else 1)
    if y is None:
        y = torch.full((x.shape[0], n), 77.0, dtype=TORCH[y_elem], device="cuda")
    size = matmul.workspace_bytes(h(codes), scheme, h(x), elem, epi) if with_workspace else 0
    space = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    matmul.launch_ref(ComputeClient.current(), h(codes), h(scales), scheme, h(x), h(y), elem, y_elem, epi,
                      workspace=space.data_ptr() if size else 0, workspace_size=size)
    return y


SCHEMES = [  # value, block, scales' type, store
    (V.Q4S, [32], 0, U32), (V.Q4F, [64], 1, U32), (V.Q4S, [128], 2, U32), (V.Q8S, [32], 0, U32), (V.Q8F, None, 1, U32), (V.Q8S, [64], 2, NATIVE),
    (V.Q2S, [64], 0, U32), (V.Q2F, [128], 2, U32), (V.E2M1, [32], 0, U32), (V.E2M1, [32], 1, NATIVE), (V.E2M1_OCP, [32], 0, U32),
    (V.E4M3, [16, 32], 0, NATIVE), (V.E5M2, [64], 0, NATIVE), (V.Q4S, [2, 16], 0, U32), (V.Q8S, [8], 0, U32),
]
# tokens, rows of y, columns in units of 128: around the tiles of 16, 32, 64, 128 and 256
SIZES = [(1, 64, 1), (3, 48, 4), (16, 130, 2), (17, 64, 3), (33, 300, 1), (64, 256, 2), (65, 96, 5), (130, 272, 1), (257, 512, 2)]


@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("which", range(len(SCHEMES)))
def test_product_of_every_scheme(oracle, which, elem):
    value, block, param, store = SCHEMES[which]
    scheme = scheme_of(value, block, param, store)
    for i, (tokens, rows, units) in enumerate(SIZES):
        rng = np.random.default_rng(100 * which + i)
        cols, rows = 128 * units, (rows + 15) // 16 * 16 if block and len(block) > 1 else rows
        codes, scales = random_weight(rng, scheme, (rows, cols))
        x = floats(rng, (tokens, cols), elem)
        y_elem = (elem, F32)[i % 2]
        y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, y_elem)
        Product(wide(x), dequantized(oracle, codes, scales, (rows, cols), elem, scheme), y_elem=y_elem).check(wide(y.cpu()), (tokens, rows, cols))


# columns that end inside a stage, a unit or a line; rows that end inside a tile, odd ones
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
@pytest.mark.parametrize("tokens,rows,cols", [(1, 1, 32), (1, 17, 96), (5, 33, 160), (16, 250, 416), (20, 255, 288), (40, 257, 352), (70, 129, 608), (129, 385, 32),
                                              (300, 131, 1120), (2, 5, 8), (37, 70, 24), (31, 513, 4128), (8, 1000, 2080), (600, 300, 736)])
def test_ragged_sizes(oracle, tokens, rows, cols, elem):
    rng = np.random.default_rng(tokens * 1000 + cols)
    for value, store in ((V.Q4S, U32), (V.Q8S, U32), (V.E4M3, NATIVE)):
        scheme = scheme_of(value, [8] if cols % 32 else [32], 0, store)
        codes, scales = random_weight(rng, scheme, (rows, cols))
        x = floats(rng, (tokens, cols), elem)
        y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, elem)
        Product(wide(x), dequantized(oracle, codes, scales, (rows, cols), elem, scheme), y_elem=elem).check(wide(y.cpu()))


@pytest.mark.parametrize("value,block", [(V.Q4S, [32]), (V.Q8S, [32]), (V.Q2F, [64])])
def test_negative_zero_and_large_scales(oracle, value, block):
    for elem in (BF16, F16):
        for tokens in (2, 40, 200):
            rng = np.random.default_rng(tokens)
            scheme = scheme_of(value, block)
            codes, scales = random_weight(rng, scheme, (96, 512), odd_scales=True)
            x = floats(rng, (tokens, 512), elem, 0.1)
            y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, F32)
            Product(wide(x), dequantized(oracle, codes, scales, (96, 512), elem, scheme)).check(wide(y.cpu()))


EPILOGUES = [(Activation.Identity, False, True, True), (Activation.Relu, False, True, False), (Activation.Silu, False, False, True), (Activation.Gelu, False, True, True),
             (Activation.GeluTanh, False, True, False), (Activation.Silu, True, True, True), (Activation.Gelu, True, False, False),
             (Activation.GeluTanh, True, True, False), (Activation.Identity, True, False, True), (Activation.Relu, True, True, True)]


@pytest.mark.parametrize("elem", [BF16, F16, F32], ids=lambda e: e.name)
@pytest.mark.parametrize("which", range(len(EPILOGUES)))
def test_epilogues(oracle, which, elem):
    activation, gated, with_bias, with_residual = EPILOGUES[which]
    scheme = scheme_of(V.Q4S, [32])
    for tokens, n, cols in ((1, 65, 256), (16, 64, 512), (48, 131, 96), (200, 260, 320)):
        rng = np.random.default_rng(which * 10 + tokens)
        rows = n * (2 if gated else 1)
        codes, scales = random_weight(rng, scheme, (rows, cols))
        x = floats(rng, (tokens, cols), elem)
        y_elem = F32 if which % 3 == 0 else elem
        bias = floats(rng, (rows,), (elem, F32)[tokens % 2]) if with_bias else None
        residual = floats(rng, (tokens, n), y_elem) if with_residual else None
        want = Product(wide(x), dequantized(oracle, codes, scales, (rows, cols), elem, scheme), activation, gated, None if bias is None else wide(bias),
                       None if residual is None else wide(residual), y_elem)
        gpu_bias = None if bias is None else bias.cuda()
        y = residual.cuda() if with_residual and tokens == 16 else None  # the residual may be y itself
        gpu_residual = None if residual is None else (y if y is not None else residual.cuda())
        epi = Epilogue(activation, gated, None if bias is None else h(gpu_bias), None if residual is None else h(gpu_residual))
        got = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, y_elem, epi, y, with_workspace=tokens != 48)
        want.check(wide(got.cpu()), tokens)


@pytest.mark.parametrize("tokens", [1, 9, 50, 300])
@pytest.mark.parametrize("pad", [8, 16, 3])
def test_strided_tensors(oracle, tokens, pad):
    """Pitched rows of every tensor, NaN between them and a guard behind y; strided bias and scales."""
    import torch

    rng = np.random.default_rng(pad)
    scheme = scheme_of(V.Q4S, [32])
    rows, cols = 140, 192
    codes, scales = random_weight(rng, scheme, (rows, cols))
    x, residual, bias = floats(rng, (tokens, cols), BF16), floats(rng, (tokens, rows), BF16), floats(rng, (rows,), BF16)
    gx, gr = pitched(x.cuda(), pad), pitched(residual.cuda(), pad)
    gc = pitched(on_gpu(codes), pad, -1)
    gs = scales.cuda().t().contiguous().t()  # stored column by column
    gb = torch.stack([bias, torch.full_like(bias, float("nan"))], 1).cuda()[:, 0]
    whole = torch.full((tokens + 1, rows + pad), 5.0, dtype=torch.bfloat16, device="cuda")
    y = whole[:tokens, :rows]
    run_matmul(gc, gs, scheme, gx, BF16, BF16, Epilogue(Activation.Silu, bias=h(gb), residual=h(gr)), y)
    Product(wide(x), dequantized(oracle, codes, scales, (rows, cols), BF16, scheme), Activation.Silu, False, wide(bias), wide(residual), BF16).check(wide(y.cpu()))
    assert (whole[tokens:] == 5.0).all() and (whole[:, rows:] == 5.0).all()


@pytest.mark.parametrize("tokens", [1, 16, 40, 300])
def test_infinities_and_nan_stay_in_their_token(oracle, tokens):
    """An infinite value of x in the last columns of a row that ends inside a stage, a NaN, and values outside the view."""
    scheme = scheme_of(V.Q4S, [32])
    for cols in (96, 224, 544):
        rng = np.random.default_rng(cols)
        codes, scales = random_weight(rng, scheme, (80, cols))
        x = floats(rng, (tokens, cols), BF16)
        x[0, cols - 1] = float("inf")
        if tokens > 2:
            x[2, 1] = float("nan")
            x[tokens - 1, cols - 9] = float("-inf")
        w = dequantized(oracle, codes, scales, (80, cols), BF16, scheme)
        y = run_matmul(on_gpu(codes), scales.cuda(), scheme, pitched(x.cuda(), 8, float("inf")), BF16, F32)
        with np.errstate(invalid="ignore"):
            Product(wide(x), w).check(wide(y.cpu()), cols)


# tokens, rows of W, columns, with a workspace: few tokens by shares of a row; each shape of tile whole, and with its columns shared out
LARGER = [(12, 260, 2112, True), (30, 400, 1056, True), (31, 972, 7008, True), (44, 70, 96, True), (88, 34, 3584, True), (61, 40, 4416, True),
          (300, 700, 4128, True), (700, 1000, 2848, True), (668, 4564, 96, True), (1100, 1040, 1024, False), (4275, 928, 1984, False)]


@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
@pytest.mark.parametrize("which", range(len(LARGER)))
def test_larger_products(oracle, which, elem):
    tokens, rows, cols, with_workspace = LARGER[which]
    value, store, block = [(V.Q4S, U32, [32]), (V.Q8S, U32, [32]), (V.E4M3, NATIVE, None), (V.Q2S, U32, [32])][(which + (elem == F16)) % 4]
    rng, gated = np.random.default_rng(which), which % 3 == 1
    scheme = scheme_of(value, block, 0, store)
    codes, scales = random_weight(rng, scheme, (rows, cols))
    x, bias = floats(rng, (tokens, cols), elem), floats(rng, (rows,), elem)
    gb = bias.cuda()
    y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), elem, elem, Epilogue(Activation.Silu, gated, bias=h(gb)), with_workspace=with_workspace)
    w = dequantized(oracle, codes, scales, (rows, cols), elem, scheme)
    Product(wide(x), w, Activation.Silu, gated, wide(bias), y_elem=elem).check(wide(y.cpu()))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes,rows", [([0, 1, 64, 65, 128, 129, 0, 300, 32, 33, 96, 500, 7, 200, 256, 189], 2050), ([100, 0, 40] * 13 + [400], 1300)])
def test_groups_of_larger_tiles(oracle, sizes, rows, gated):
    """Tiles that are full, at most half full and hardly begun, on grids of more workgroups than run at once."""
    import torch

    rng = np.random.default_rng(rows)
    scheme = scheme_of(V.Q8S if gated else V.Q4S, [32])
    e, cols, positions, elem = len(sizes), 96, sum(sizes), F16 if gated else BF16
    n = rows // 2 if gated else rows
    codes, scales = random_weight(rng, scheme, (e, rows, cols))
    x = floats(rng, (positions, cols), elem)
    at = offsets_of(sizes)
    gc, gs, gx, go = on_gpu(codes), scales.cuda(), x.cuda(), torch.from_numpy(at).cuda()
    y = torch.full((positions, n), 9.0, device="cuda")
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), elem, F32, epilogue=Epilogue(Activation.Relu, gated))
    w, got = dequantized(oracle, codes, scales, (e, rows, cols), elem, scheme), wide(y.cpu())
    for i in range(e):
        if sizes[i]:
            Product(wide(x)[at[i]:at[i + 1]], w[i], Activation.Relu, gated).check(got[at[i]:at[i + 1]], i)


def test_no_tokens_and_no_columns(oracle):
    import torch

    scheme = scheme_of(V.Q4S, [32])
    codes, scales = random_weight(np.random.default_rng(0), scheme, (64, 64))
    empty = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert run_matmul(on_gpu(codes), scales.cuda(), scheme, empty, BF16, BF16).shape == (0, 64)
    none = torch.empty((64, 0), dtype=torch.int32, device="cuda")
    bias = torch.arange(64, dtype=torch.float32, device="cuda")
    for tokens in (3, 100):
        y = run_matmul(none, torch.empty((64, 0), device="cuda"), scheme, torch.empty((tokens, 0), dtype=torch.bfloat16, device="cuda"), BF16, F32,
                       Epilogue(bias=h(bias)))
        assert torch.equal(y, bias.expand(tokens, 64))


def test_one_token_without_its_dimension(oracle):
    import torch

    rng = np.random.default_rng(5)
    scheme = scheme_of(V.Q8S, [32])
    codes, scales = random_weight(rng, scheme, (100, 256))
    x, y = floats(rng, (256,), F16), torch.empty((100,), device="cuda")
    gc, gs, gx = on_gpu(codes), scales.cuda(), x.cuda()
    matmul.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(y), F16, F32)
    Product(wide(x)[None], dequantized(oracle, codes, scales, (100, 256), F16, scheme)).check(wide(y.cpu())[None])


def offsets_of(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


GROUPS = [[5], [0, 0, 3], [1, 0, 16, 17, 0, 64], [33, 200, 0, 7], [0] * 70 + [9] + [0] * 60 + [300, 1], [2] * 130, [128, 129, 127], [700, 0, 40]]


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("which", range(len(GROUPS)))
def test_groups_of_any_size(oracle, which, gather):
    import torch

    sizes = GROUPS[which]
    rng = np.random.default_rng(which)
    value, store, block, elem = [(V.Q4S, U32, [32], BF16), (V.Q8S, U32, [64], F16), (V.E4M3, NATIVE, [16, 32], BF16), (V.Q2S, U32, [64], F16)][which % 4]
    gated = which % 2 == 1
    scheme = scheme_of(value, block, 0, store)
    e, n, cols, positions = len(sizes), 80, 192, sum(sizes)
    rows = n * (2 if gated else 1)
    codes, scales = random_weight(rng, scheme, (e, rows, cols))
    tokens = positions // 2 + 1 if gather else positions
    row_of = rng.integers(0, tokens, positions).astype(np.int32) if gather else np.arange(positions)
    x, bias = floats(rng, (tokens, cols), elem), floats(rng, (e, rows), elem)
    at = offsets_of(sizes)
    y = torch.full((positions, n), 9.0, device="cuda")
    gc, gb, gs, gx, go, gr = on_gpu(codes), bias.cuda(), scales.cuda(), x.cuda(), torch.from_numpy(at).cuda(), torch.from_numpy(row_of.astype(np.int32)).cuda()
    epi = Epilogue(Activation.Silu, gated, bias=h(gb))
    size = experts.workspace_bytes(h(gc), scheme, h(y), elem, epi)
    space = torch.full((max(16, size),), 255, dtype=torch.uint8, device="cuda")
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), elem, F32, h(gr) if gather else None, epi,
                       workspace=space.data_ptr(), workspace_size=size)
    w = dequantized(oracle, codes, scales, (e, rows, cols), elem, scheme)
    got = wide(y.cpu())
    for i in range(e):
        if sizes[i]:
            Product(wide(x)[row_of[at[i]:at[i + 1]]], w[i], Activation.Silu, gated, wide(bias)[i]).check(got[at[i]:at[i + 1]], i)


@pytest.mark.parametrize("positions", [12, 150])
def test_offsets_and_rows_outside_are_taken_inside(oracle, positions):
    """What the device holds is not known to the host: nothing outside of the tensors is read or written."""
    import torch

    rng = np.random.default_rng(3)
    scheme = scheme_of(V.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (4, 48, 128))
    x = floats(rng, (7, 128), BF16)
    whole = torch.full((positions + 2, 48), 9.0, device="cuda")
    y = whole[1:positions + 1]
    row_of = rng.integers(-3, 12, positions).astype(np.int32)
    row_of[0], row_of[1] = -2 ** 31, 2 ** 31 - 1
    at = np.array([2, 6, 4, 8, 10 ** 9], np.int32)  # two positions of nobody in front, a range that runs backwards, one past the end
    gc, gs, gx, go, gr = on_gpu(codes), scales.cuda(), x.cuda(), torch.from_numpy(at).cuda(), torch.from_numpy(row_of).cuda()
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), BF16, F32, h(gr))
    w, got = dequantized(oracle, codes, scales, (4, 48, 128), BF16, scheme), wide(whole.cpu())
    assert (got[[0, positions + 1]] == 9.0).all() and (got[1:3] == 9.0).all()
    taken = wide(x)[np.clip(row_of, 0, 6)]
    Product(taken[8:], w[3]).check(got[9:positions + 1])
    Product(taken[2:4], w[0]).check(got[3:5])  # 4 .. 5 belong to two experts; 6, 7 to the third
    Product(taken[6:8], w[2]).check(got[7:9])


@pytest.mark.parametrize("tokens", [4, 100])
def test_experts_that_lie_apart(oracle, tokens):
    """Strides of the experts' dimension: every second expert of a larger tensor."""
    import torch

    rng = np.random.default_rng(8)
    scheme = scheme_of(V.Q8S, [32])
    codes, scales = random_weight(rng, scheme, (6, 64, 256))
    x = floats(rng, (2 * tokens, 256), BF16)
    gc, gs, gx = on_gpu(codes)[::2], scales.cuda()[::2], x.cuda()
    go, y = torch.tensor([0, tokens, tokens, 2 * tokens], dtype=torch.int32, device="cuda"), torch.empty((2 * tokens, 64), device="cuda")
    experts.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(gx), h(go), h(y), BF16, F32)
    w, got = dequantized(oracle, codes, scales, (6, 64, 256), BF16, scheme), wide(y.cpu())
    Product(wide(x)[:tokens], w[0]).check(got[:tokens])
    Product(wide(x)[tokens:], w[4]).check(got[tokens:])


def test_same_bits_again():
    """No order of summation changes from call to call, with and between other work on the GPU."""
    import torch

    rng = np.random.default_rng(2)
    scheme = scheme_of(V.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (512, 2048))
    for tokens in (1, 16, 60, 500):
        x = floats(rng, (tokens, 2048), BF16)
        gc, gs, gx = on_gpu(codes), scales.cuda(), x.cuda()
        first = run_matmul(gc, gs, scheme, gx, BF16, F32).clone()
        for _ in range(5):
            torch.randn((1 << 20,), device="cuda").sort()
            assert torch.equal(first, run_matmul(gc, gs, scheme, gx, BF16, F32))


@pytest.mark.parametrize("tokens", [3, 40, 400])
def test_captured_on_another_stream(oracle, tokens):
    """A captured launch, replayed on changing inputs with eager work in between."""
    import torch

    rng = np.random.default_rng(tokens)
    scheme = scheme_of(V.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (256, 1024))
    gc, gs = on_gpu(codes), scales.cuda()
    x, y = torch.zeros((tokens, 1024), dtype=torch.bfloat16, device="cuda"), torch.zeros((tokens, 256), device="cuda")
    size = matmul.workspace_bytes(h(gc), scheme, h(x), BF16)
    space = torch.empty((max(16, size),), dtype=torch.uint8, device="cuda")

    def call():
        matmul.launch_ref(ComputeClient.current(), h(gc), h(gs), scheme, h(x), h(y), BF16, F32, workspace=space.data_ptr(), workspace_size=size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    w = dequantized(oracle, codes, scales, (256, 1024), BF16, scheme)
    for _ in range(4):
        new = floats(rng, (tokens, 1024), BF16)
        x.copy_(new)
        graph.replay()
        replayed = y.clone()
        torch.cuda.synchronize()
        call()
        assert torch.equal(replayed, y)
        Product(wide(new), w).check(wide(y.cpu()))


def test_weights_and_results_beyond_32_bits_of_offset(oracle):
    """The last of six experts of 0.9 GiB each, and results of more than 2^32 bytes."""
    import torch

    rng = np.random.default_rng(1)
    scheme = scheme_of(V.E4M3, [64], 0, NATIVE)
    rows, cols = 30000, 32000
    codes = torch.zeros((6, rows, cols), dtype=torch.uint8, device="cuda")
    scales = torch.full((6, rows, cols // 64), 2.0 ** -12, device="cuda")
    last = torch.from_numpy(rng.integers(0, 0x70, (rows, cols), dtype=np.uint8))
    codes[5].copy_(last)
    for tokens in (3, 80):
        x = floats(rng, (tokens, cols), BF16)
        go = torch.tensor([0, 0, 0, 0, 0, 0, tokens], dtype=torch.int32, device="cuda")
        y = torch.empty((tokens, rows), device="cuda")
        gx = x.cuda()
        experts.launch_ref(ComputeClient.current(), h(codes), h(scales), scheme, h(gx), h(go), h(y), BF16, F32)
        w = codes[5, -40:].cpu().view(torch.float8_e4m3fn).double().numpy() * 2.0 ** -12
        Product(wide(x), w).check(wide(y[:, -40:].cpu()))
    del codes, scales
    scheme = scheme_of(V.Q4S, [32])
    codes, scales = random_weight(rng, scheme, (40000, 32))
    x = floats(rng, (30000, 32), BF16)
    y = run_matmul(on_gpu(codes), scales.cuda(), scheme, x.cuda(), BF16, F32)
    w = dequantized(oracle, codes, scales, (40000, 32), BF16, scheme)
    for part in (slice(0, 50), slice(29950, 30000)):
        Product(wide(x)[part], w).check(wide(y[part].cpu()))

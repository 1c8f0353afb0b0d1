"""cq_route and cq_combine against numpy in 64 bits.  Whole numbers have to be equal.  A weight is a quotient of sums of at most
1024 exponentials in f32, each within 2 units in the last place: within (1024 + 8) 2^-24 < 2^-13 of itself in the worst case; a softmax's exponent
l - max is rounded once, which moves it by 2^-24 |l - max|."""
import numpy as np
import pytest

from cubek_amd import ComputeClient, ElemType, Score, TensorHandleRef, routing
from matmul_reference import TORCH, check_rounded

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ElemType.F32, ElemType.F16, ElemType.BF16
h = TensorHandleRef.from_torch


def route(logits, chosen, elem, score, normalize):
    import torch

    t, e = logits.shape
    outs = [torch.full((t, chosen), 7.0, device="cuda")] + [torch.full(s, -5, dtype=torch.int32, device="cuda") for s in ((t, chosen), (e + 1,), (t * chosen,), (t, chosen))]
    size = routing.workspace_bytes(t, e, chosen)
    space = torch.full((max(16, size),), 255, dtype=torch.uint8, device="cuda")
    routing.launch_ref(ComputeClient.current(), h(logits), *(h(o) for o in outs), elem, score, normalize, workspace=space.data_ptr(), workspace_size=size)
    return [o.cpu().numpy() for o in outs]


def check(logits, chosen, score, normalize, got):
    """`logits` in 64 bits, NaN taken as -infinity."""
    weights, chosen_experts, offsets, rows, slots = got
    t, e = logits.shape
    logits = np.where(np.isnan(logits), -np.inf, logits) + 0.0
    want = np.argsort(-logits, axis=1, kind="stable")[:, :chosen]
    assert np.array_equal(chosen_experts, want)
    flat = want.reshape(-1)
    order = np.argsort(flat, kind="stable")
    assert np.array_equal(offsets, np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e))]))
    assert np.array_equal(rows, order // chosen)
    place = np.empty(t * chosen, np.int64)
    place[order] = np.arange(t * chosen)
    assert np.array_equal(slots, place.reshape(t, chosen))
    with np.errstate(invalid="ignore", over="ignore"):
        top = logits.max(1, keepdims=True) if e else logits
        gap = np.where(logits == top, 0.0, logits - top)
        s = np.where(np.isneginf(logits), 0.0, np.exp(gap) if score == Score.Softmax else 1.0 / (1.0 + np.exp(-logits)))
        w = np.take_along_axis(s, want, 1)
        total = w.sum(1, keepdims=True) if normalize else (s.sum(1, keepdims=True) if score == Score.Softmax else np.ones((t, 1)))
        w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
    spread = np.where(np.isfinite(gap), np.abs(gap), 0.0).max() if gap.size else 0.0
    assert (np.abs(weights - w) <= (2.0 ** -13 + 2.0 ** -22 * spread) * w + 2.0 ** -126).all()


@pytest.mark.parametrize("score", [Score.Softmax, Score.Sigmoid], ids=lambda s: s.name)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("tokens,num,chosen", [(1, 1, 1), (1, 8, 2), (16, 8, 8), (63, 60, 4), (64, 64, 6), (65, 65, 3), (256, 128, 8), (257, 128, 8), (1000, 160, 6),
                                               (1021, 257, 5), (2500, 512, 10), (300, 1024, 64), (20000, 16, 2), (9, 70, 64)])
def test_choice_and_positions(tokens, num, chosen, score, normalize):
    import torch

    rng = np.random.default_rng(tokens + num)
    for elem in (F32, BF16, F16):
        # 16-bit logits have many ties
        logits = torch.tensor(rng.normal(0, 2, (tokens, num)), dtype=torch.float32).to(TORCH[elem])
        check(logits.double().numpy(), chosen, score, normalize, route(logits.cuda(), chosen, elem, score, normalize))


@pytest.mark.parametrize("score", [Score.Softmax, Score.Sigmoid], ids=lambda s: s.name)
@pytest.mark.parametrize("tokens", [7, 600])
def test_ties_masks_and_rows_without_anything(tokens, score):
    import torch

    rng = np.random.default_rng(0)
    x = rng.integers(-2, 3, (tokens, 96)).astype(np.float32)  # nothing but ties
    x[0] = 0.0
    x[0, ::2] = -0.0
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 5:] = -np.inf
    x[4] = -3.4028235e38
    x[5, 40] = np.inf
    x[6, 3:50] = np.nan
    for normalize in (True, False):
        got = route(torch.from_numpy(x).cuda(), 7, F32, score, normalize)
        if score == Score.Softmax:  # beside an infinite logit everything else counts nothing
            assert got[0][5].tolist() == [1.0] + [0.0] * 6
        assert (got[0][1:3] == 0.0).all()
        check(x.astype(np.float64), 7, score, normalize, got)


def test_strided_logits():
    import torch

    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (50, 300)).astype(np.float32)
    gpu = torch.from_numpy(x).cuda()
    check(x.T[:, 3:43].astype(np.float64), 4, Score.Softmax, True, route(gpu.t()[:, 3:43], 4, F32, Score.Softmax, True))
    check(x[:, ::3].astype(np.float64), 4, Score.Softmax, True, route(gpu[:, ::3], 4, F32, Score.Softmax, True))


def test_no_tokens():
    import torch

    got = route(torch.empty((0, 40), device="cuda"), 4, F32, Score.Softmax, True)
    assert got[2].tolist() == [0] * 41


@pytest.mark.parametrize("tokens", [5, 400])
def test_captured(tokens):
    import torch

    rng = np.random.default_rng(4)
    x = torch.zeros((tokens, 128), device="cuda")
    outs = [torch.zeros((tokens, 6), device="cuda")] + [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((tokens, 6), (129,), (tokens * 6,), (tokens, 6))]
    size = routing.workspace_bytes(tokens, 128, 6)
    space = torch.full((max(16, size),), 255, dtype=torch.uint8, device="cuda")

    def call():
        routing.launch_ref(ComputeClient.current(), h(x), *(h(o) for o in outs), F32, workspace=space.data_ptr(), workspace_size=size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        new = rng.normal(0, 1, (tokens, 128)).astype(np.float32)
        x.copy_(torch.from_numpy(new))
        graph.replay()
        torch.cuda.synchronize()
        check(new.astype(np.float64), 6, Score.Softmax, True, [o.cpu().numpy() for o in outs])


@pytest.mark.parametrize("elem,y_elem", [(F32, BF16), (BF16, BF16), (F16, F32), (F32, F32), (BF16, F16)])
@pytest.mark.parametrize("tokens,chosen,cols,pad", [(1, 2, 4096, 0), (5, 1, 7, 0), (33, 8, 258, 0), (100, 6, 1024, 8), (17, 3, 100, 3), (2000, 9, 64, 0), (3, 0, 40, 0)])
def test_weighted_sum(tokens, chosen, cols, pad, elem, y_elem):
    """k FMAs and one addition in f32: within (k + 2) 2^-24 of the sum of sizes in front of the rounding."""
    import torch

    rng = np.random.default_rng(tokens + cols)
    positions = tokens * max(chosen, 1)
    hs = torch.tensor(rng.normal(0, 1, (positions, cols)), dtype=torch.float32).to(TORCH[elem])
    slots = rng.permutation(positions)[:tokens * chosen].reshape(tokens, chosen).astype(np.int32)
    weights = rng.uniform(-1, 1, (tokens, chosen)).astype(np.float32)
    if chosen > 2:  # slots of nobody add nothing, whatever their weight
        slots[0, 1], slots[-1, 0] = -1, positions
        weights[0, 1] = np.inf
    residual = torch.tensor(rng.normal(0, 1, (tokens, cols)), dtype=torch.float32).to(TORCH[y_elem])

    def rows_apart(t):
        whole = torch.full((t.shape[0], cols + pad), float("nan"), dtype=t.dtype, device="cuda")
        whole[:, :cols] = t.cuda()
        return whole[:, :cols]
    gh, gs, gw = rows_apart(hs), torch.from_numpy(slots).cuda(), torch.from_numpy(weights).cuda()
    for with_residual in (False, True):
        y = rows_apart(residual)
        routing.combine(ComputeClient.current(), h(gh), h(gs), h(gw), h(y), elem, y_elem, h(y) if with_residual else None)
        there = (slots >= 0) & (slots < positions)
        w = np.where(there, weights, 0.0).astype(np.float64)
        terms = hs.double().numpy()[np.where(there, slots, 0)] * w[:, :, None]
        want, size = terms.sum(1), np.abs(terms).sum(1)
        if with_residual:
            want, size = want + residual.double().numpy(), size + np.abs(residual.double().numpy())
        check_rounded(y.double().cpu().numpy(), want, (chosen + 2) * 2.0 ** -24 * size, y_elem)

"""cq_cache_append of rows that hold infinities, NaN, zeros and denormals: codes and scales are those of cq_quantize_dynamic, bit for bit."""
import pytest

from attention_reference import h
from cubek_amd import Cache, ComputeClient, ElemType, QuantStore, QuantValue, cache, quantize
from matmul_reference import PARAM, TORCH, scheme_of

pytestmark = pytest.mark.gpu
V, U32, NATIVE = QuantValue, QuantStore.U32, QuantStore.Native
SCHEMES = [(V.Q8S, NATIVE, 32, 0), (V.Q8F, U32, 64, 1), (V.Q4S, U32, 32, 2), (V.E4M3, NATIVE, 64, 0), (V.E5M2, NATIVE, 32, 2), (V.E2M1, NATIVE, 32, 0), (V.E2M1, U32, 16, 1),
           (V.E2M1_OCP, U32, 64, 0), (V.Q4F, U32, 8, 0)]


@pytest.mark.parametrize("of", SCHEMES, ids=str)
@pytest.mark.parametrize("elem", [ElemType.BF16, ElemType.F16, ElemType.F32], ids=lambda e: e.name)
@pytest.mark.parametrize("offset", [0, 1])
def test_odd_values(of, elem, offset):
    """Rows on 16-byte boundaries, and off them: both ways that rows are read."""
    import torch

    scheme = scheme_of(of[0], [of[2]], of[3], of[1])
    tokens, heads, dim = 64, 2, 128
    x = torch.randn((tokens, heads, dim), generator=torch.Generator().manual_seed(1))
    nan, inf = float("nan"), float("inf")
    x[0, 0, 3], x[1, 0, 5], x[2, 0, 7], x[3, 0, 9], x[3, 0, 10] = nan, inf, -inf, nan, inf
    x[4], x[5], x[8], x[10] = 0.0, -0.0, nan, inf
    x[6] *= 1e-38
    x[7] *= 1e-41
    x[9] *= 3e37
    x[11, :, ::2] = 6e4
    x[12] *= 6e-8
    x = x.to(TORCH[elem])
    wide = torch.zeros((tokens, heads * dim + 8), dtype=TORCH[elem], device="cuda")
    wide[:, offset:offset + heads * dim] = x.view(tokens, -1).cuda()
    rows = wide[:, offset:offset + heads * dim].view(tokens, heads, dim)
    plain, stored = x.cuda(), scheme.packed_shape((tokens, heads, dim))
    codes = torch.zeros(stored, dtype=torch.int32 if of[1] == U32 else torch.uint8, device="cuda")
    scales = torch.zeros(scheme.scales_shape((tokens, heads, dim)), dtype=PARAM[of[3]], device="cuda")
    client = ComputeClient.current()
    quantize.launch_dynamic(client, h(plain), h(codes), h(scales), scheme, elem)
    keys, values = (torch.zeros((tokens, heads, 1, stored[-1]), dtype=codes.dtype, device="cuda") for _ in range(2))  # a page a token
    key_scales, value_scales = (torch.zeros((tokens, heads, 1, scales.shape[-1]), dtype=scales.dtype, device="cuda") for _ in range(2))
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
    cache.append(client, Cache(h(keys), h(values), scheme, h(key_scales), h(value_scales)), h(rows), h(rows), h(slots), elem)
    torch.cuda.synchronize()

    def bits(t):
        return t.contiguous().view({4: torch.int32, 2: torch.int16, 1: torch.uint8}[t.element_size()]).view(tokens, heads, -1)

    for got, got_scales in ((keys, key_scales), (values, value_scales)):
        assert torch.equal(bits(got), bits(codes)) and torch.equal(bits(got_scales), bits(scales))

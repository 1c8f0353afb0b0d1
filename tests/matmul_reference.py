"""Products with quantized weights in 64 bits, for the tests: random codes and scales, the oracle's dequantized weights, numpy sums.

Tolerance, derived once (`Product.bound`).  v = sum_k x w + b in f32: at most cols + 2 additions in any order, products of 16-bit factors
exact, products of f32 factors rounded once: |dv| <= (cols + 4) 2^-24 m with m = sum |x w| + |b| (2^-23 where matrix instructions may
round towards zero).  An activation has a slope of at most 1.13 (silu 1.1, gelu 1.13) and is computed within 2^-20 of |act(v)| + 2^-20 |v|
(a handful of f32 operations, the tails of the error function and the exponential cancelling at |v|'s scale).  A gate multiplies two such values.
The result is rounded once, which keeps the order of numbers: it lies between the roundings of both ends of what is allowed in front of it."""
import math

import numpy as np
import torch

from cubek_amd import Activation, ElemType, QuantLevel, QuantScheme, QuantStore, QuantValue

TORCH = {ElemType.F32: torch.float32, ElemType.F16: torch.float16, ElemType.BF16: torch.bfloat16}
PARAM = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}


def scheme_of(value, block=None, param=0, store=QuantStore.U32):
    from cubek_amd import QuantParam

    level = QuantLevel.Tensor if block is None else QuantLevel.block(block)
    return QuantScheme.default().with_value(value).with_level(level).with_param(QuantParam(param)).with_store(store)


def random_weight(rng, scheme, shape, odd_scales=False):
    """Codes (numpy storage), scales (torch, typed scheme.param) of a random weight, no code an infinity or NaN."""
    stored = scheme.packed_shape(shape)
    if scheme.store == QuantStore.U32:
        codes = rng.integers(0, 1 << 32, stored, dtype=np.uint64).astype(np.uint32)
    else:
        codes = rng.integers(0, 256, stored, dtype=np.uint64).astype(np.uint8)
        if scheme.value == QuantValue.E4M3:
            codes[(codes & 0x7F) == 0x7F] = 0x35
        elif scheme.value == QuantValue.E5M2:
            codes[(codes & 0x7C) >= 0x74] = 0x35  # large ones out as well: f16 weights stay finite
    top = 2.0 ** -10 if scheme.store == QuantStore.Native else 2.0 ** -7
    scales = rng.uniform(0.25, 1.0, scheme.scales_shape(shape)) * top
    if odd_scales:  # negative, zero and large ones
        flat = scales.reshape(-1)
        flat[::3] *= -1.0
        flat[::7] = 0.0
        flat[5::11] *= 300.0
    return codes, torch.tensor(scales, dtype=torch.float32).to(PARAM[int(scheme.param)])


def storage(t):
    """numpy bits of a torch tensor, as the oracle takes them."""
    return t.view(torch.int16).numpy().view(np.uint16) if t.element_size() == 2 else t.numpy()


def dequantized(oracle, codes, scales, shape, elem, scheme):
    return oracle.from_bits(oracle.dequantize(codes, shape, storage(scales), elem, scheme), elem).astype(np.float64).reshape(shape)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activated(v, activation):
    with np.errstate(over="ignore", invalid="ignore"):
        if activation == Activation.Relu:
            return np.where(v < 0, 0.0, v)
        if activation == Activation.Silu:
            return v / (1.0 + np.exp(-v))
        if activation == Activation.Gelu:
            return 0.5 * v * (1.0 + _erf(v / math.sqrt(2.0)))
        if activation == Activation.GeluTanh:
            return 0.5 * v * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def rounded(y, elem):
    return torch.from_numpy(np.ascontiguousarray(y)).to(TORCH[elem]).double().numpy()


def check_rounded(got, y, bound, elem, what=""):
    """`got` is a number within `bound` of `y`, rounded once to `elem`; infinities and NaN of `y` are themselves."""
    got, plain = np.asarray(got, dtype=np.float64), np.isfinite(y) & np.isfinite(bound)
    assert np.array_equal(np.isnan(got), np.isnan(y)), what
    assert np.array_equal(got[np.isinf(y)], y[np.isinf(y)]), what
    with np.errstate(invalid="ignore"):
        wrong = plain & ((got < rounded(y - bound, elem)) | (got > rounded(y + bound, elem)))
    if wrong.any():
        at = tuple(i[0] for i in np.nonzero(wrong))
        raise AssertionError(f"{what}: {wrong.sum()} of {wrong.size}, first at {at}: {got[at]} for {y[at]}, allowed {bound[at]}")


class Product:
    """epilogue(x w^T) of arrays in 64 bits, and how far it may be off in front of its rounding to the type of y."""

    def __init__(self, x, w, activation=Activation.Identity, gated=False, bias=None, residual=None, y_elem=ElemType.F32):
        with np.errstate(invalid="ignore", over="ignore"):
            v = x @ w.T
            m = np.abs(x) @ np.abs(w).T
            if bias is not None:
                v, m = v + bias, m + np.abs(bias)
            dv = (x.shape[1] + 4) * 2.0 ** -23 * m
            n = w.shape[0] // 2 if gated else w.shape[0]
            y = activated(v[:, :n], activation)
            dy = dv[:, :n]
            if activation != Activation.Identity:
                dy = 1.13 * dy + 2.0 ** -20 * (np.abs(y) + np.abs(v[:, :n]))
            if gated:
                dy = dy * (np.abs(v[:, n:]) + dv[:, n:]) + np.abs(y) * dv[:, n:] + 2.0 ** -23 * np.abs(y * v[:, n:])
                y = y * v[:, n:]
            if residual is not None:
                y = y + residual
                dy = dy + 2.0 ** -23 * np.abs(y)
            self.y, self.bound, self.elem = y, dy, y_elem

    def check(self, got, what=""):
        check_rounded(got, self.y, self.bound, self.elem, what)
